// Logits in front of the choice of a token: penalties for repeated tokens, biases, and a mask of the tokens that a grammar allows.
//   seen (the token is among the row's tokens[0 .. token_len)):  l <- l > 0 ? l / repetition : l * repetition
//   c times among the generated ones (from prompt_len on):       l <- l - (presence [c > 0] + frequency c)
//   l <- l + sum of the token's biases;   not allowed: l <- -infinity;   all in f32, rounded once
// A workgroup takes C columns of a row: it counts the row's tokens that fall on them in LDS (integers, so their order is nothing to the result) while its
// logits are on the way, then reads the counts beside them.  HBM bounds many rows (every logit once in, once out), the two dependent loads (length, tokens)
// one row.  Every workgroup of a row reads all of its tokens, so wide ones read less and narrow ones are more: 256 rows of 128256 bf16 logits behind 6000
// tokens take 34 to 36 us (3.9 TB/s) with C = 8192, 40 where their tensors are new to the caches, 45 with 4096, 109 with 1024; 16 rows 6.5, 6.1 and 9.9; one row 6.0, 5.1 and 4.9.  Before units with nothing
// to change were left alone, 16384 columns, which leave a CU two workgroups whose loads do not cover their counting, took 43 us, and the workgroups of a row on all XCDs, where its tokens
// come from HBM eight times, 65.  Vector issue bounds long histories (69 % of the cycles): nearly every wavefront's columns hold a token of the row, and all of them go through the penalties.
#include <hip/hip_runtime.h>

#include "kernel_args.h"

using namespace cutile;

namespace {

constexpr int kThreads = 512, kMostBiases = 1024, kRowsByXcd = 64;
constexpr uint32_t kPrompt = 0x80000000u, kBiased = 0x40000000u;   // beside the count of generated tokens

struct LogitsArgs {
  const void* in;
  void* out;
  int64_t in_row, out_row;                           // elements
  const int32_t *tokens, *prompt_lens, *token_lens;  // tokens [rows, most]
  int64_t tokens_row;
  const float *repetition, *presence, *frequency;
  const int32_t* bias_ids;
  const float* bias_values;
  int64_t ids_row, values_row;
  const uint32_t* allowed;                           // bit t % 32 of word t / 32
  int64_t allowed_row;
  int32_t vocab, most, biases, blocks;               // blocks: workgroups of a row
  int32_t rows, pad;
};

template <typename T, int C>
__device__ __forceinline__ void adjust(const LogitsArgs& a) {
  constexpr int kUnits = C / 8 / kThreads > 0 ? C / 8 / kThreads : 1;
  __shared__ __attribute__((aligned(16))) uint32_t words[C];
  __shared__ uint16_t ids[kMostBiases];   // columns: four workgroups of the widest fit a CU
  __shared__ float values[kMostBiases];
  __shared__ int32_t biases;
  struct Unit {   // (loads and stores of 16 bytes need no more than the alignment of their elements: rows of odd lengths are no different)
    T v[8];
  };
  const int tid = threadIdx.x;
  int32_t row = blockIdx.x / a.blocks, block = blockIdx.x % a.blocks;
  if (a.rows >= kRowsByXcd) {   // a row's workgroups on one XCD: its tokens are fetched into one L2
    const int32_t slot = blockIdx.x / 8;
    row = slot / a.blocks * 8 + blockIdx.x % 8, block = slot % a.blocks;
    if (row >= a.rows) return;
  }
  const int32_t col0 = block * C, cols = min(C, a.vocab - col0);
  const T* in = (const T*)a.in + (int64_t)row * a.in_row + col0;
  T* out = (T*)a.out + (int64_t)row * a.out_row + col0;

  Unit held[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int c = (tid + i * kThreads) * 8;
    if (c + 8 <= cols) {
      held[i] = *reinterpret_cast<const Unit*>(in + c);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) held[i].v[e] = c + e < cols ? in[c + e] : (T)0.0f;
    }
  }
  int32_t n = 0, prompt = 0;
  if (a.tokens) {
    n = a.token_lens ? min(max(a.token_lens[row], 0), a.most) : a.most;
    prompt = a.prompt_lens ? min(max(a.prompt_lens[row], 0), n) : 0;
  }
  const float repetition = a.repetition ? a.repetition[row] : 1.0f, presence = a.presence ? a.presence[row] : 0.0f, frequency = a.frequency ? a.frequency[row] : 0.0f;
  for (int i = tid; i < C / 4; i += kThreads) reinterpret_cast<uint4*>(words)[i] = uint4{0, 0, 0, 0};
  __syncthreads();
  if (a.biases > 0 && tid < 64) {   // the entries that fall here, in their order
    int32_t found = 0;
    for (int32_t i = 0; i < a.biases; i += 64) {
      const int32_t id = i + tid < a.biases ? a.bias_ids[(int64_t)row * a.ids_row + i + tid] : -1, c = id - col0;
      const bool here = id >= 0 && c >= 0 && c < cols;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(here);
      if (here) {
        const int32_t at = found + __builtin_popcountll(mask & ((1ull << tid) - 1));
        ids[at] = (uint16_t)c, values[at] = a.bias_values[(int64_t)row * a.values_row + i + tid];
        atomicOr(&words[c], kBiased);
      }
      found += __builtin_popcountll(mask);
    }
    if (tid == 0) biases = found;
  }
  const int32_t* tokens = a.tokens + (int64_t)row * a.tokens_row;
  auto count = [&](int32_t i, int32_t t) {
    const uint32_t c = (uint32_t)t - (uint32_t)col0;
    if (c < (uint32_t)cols) {
      if (i < prompt) atomicOr(&words[c], kPrompt);
      else atomicAdd(&words[c], 1u);
    }
  };
  struct Four {
    int32_t t[4];
  };
  constexpr int kAhead = 4, kStep = kThreads * 4;   // loads under way together
#pragma unroll 1
  for (int32_t i = tid * 4; i < (n & ~3); i += kAhead * kStep) {
    Four four[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) four[k] = i + k * kStep < (n & ~3) ? *reinterpret_cast<const Four*>(tokens + i + k * kStep) : Four{{-1, -1, -1, -1}};
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) count(i + k * kStep + e, four[k].t[e]);
  }
  if (tid < (n & 3)) count((n & ~3) + tid, tokens[(n & ~3) + tid]);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int c = (tid + i * kThreads) * 8;
    if (c >= cols) continue;
    uint32_t word[8], allowed = 0xffu;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint4 w = reinterpret_cast<const uint4*>(words)[c / 4 + b];
      word[b * 4] = w.x, word[b * 4 + 1] = w.y, word[b * 4 + 2] = w.z, word[b * 4 + 3] = w.w;
    }
    if (a.allowed) allowed = a.allowed[(int64_t)row * a.allowed_row + (col0 + c) / 32] >> ((col0 + c) & 31);
    float l[8];
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) l[e] = (float)held[i].v[e], any |= word[e];
    if (any) {   // (most units have nothing to change: 256 rows behind 50 tokens 27 us, 29 without this)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t count = word[e] & (kBiased - 1);
        if ((word[e] & ~kBiased) != 0) l[e] = l[e] > 0.0f ? l[e] / repetition : l[e] * repetition;
        if (count) l[e] -= presence + frequency * (float)count;
        if (word[e] & kBiased) {
          float sum = 0.0f;
          for (int32_t k = 0; k < biases; ++k)
            if (ids[k] == c + e) sum += values[k];
          l[e] += sum;
        }
      }
    }
    Unit u;
#pragma unroll
    for (int e = 0; e < 8; ++e) u.v[e] = allowed >> e & 1 ? (T)l[e] : (T)-INFINITY;
    if (c + 8 <= cols) {
      *reinterpret_cast<Unit*>(out + c) = u;
    } else {
      for (int e = 0; e < 8 && c + e < cols; ++e) out[c + e] = u.v[e];
    }
  }
}

}  // namespace

#define LOGITS(TYPE, T, C) \
  extern "C" __global__ void __launch_bounds__(kThreads) adjust_logits_entry__##TYPE##_##C(LogitsArgs a) { adjust<T, C>(a); }
#define LOGITS_C(TYPE, T) LOGITS(TYPE, T, 1024) LOGITS(TYPE, T, 4096) LOGITS(TYPE, T, 8192)
LOGITS_C(f16, _Float16)
LOGITS_C(bf16, __bf16)
LOGITS_C(f32, float)
