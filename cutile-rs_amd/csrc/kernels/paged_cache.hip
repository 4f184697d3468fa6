// New tokens' keys and values into the pages of a cache, and back.
//
//   write   cache[page, p % page_size, h, :] = new[row, h, :]            mxfp8: in blocks of 32 along D (block_scale.h)
//   read    out[row, h, :] = cache[page, p % page_size, h, :]            mxfp8: rounded once
// with row, p and page as in paged.h.  Nothing is computed: 2 T H D values go in and out once, and HBM bounds a prompt, the chain of dependent loads
// (starts, length, page, row) a single token.  A wavefront takes a token, which makes that chain its own and the search for the token's sequence one load of
// 64 starts; its lanes take 8 values of K and of V at a time.  Short tokens go several to a wavefront, which then finds them side by side: up to 8192 tokens of
// 16 sequences out of mxfp8, one head of 64 values, 11.6 us with 16 to a wavefront and 27.8 with one; one head of 128, 16.7 and 28.9; eight, one to each, 95
// (4.8 TB/s, two thirds of it stores).  4 x 4096 tokens of eight heads into 16 bits 22 us (4.7 TB/s).
#include <hip/hip_runtime.h>

#include "block_scale.h"
#include "kernel_args.h"
#include "paged.h"

using namespace cutile;

namespace {

constexpr int kWaves = 4;

struct Rows {   // new_k, new_v or out: [tokens, heads, D]
  unsigned char *k, *v;
  int64_t k_token, k_head, v_token, v_head;   // bytes
  int32_t per_wave, pad;                      // tokens to a wavefront, up to 16
};

// Where the lane's units are: `u` of the 2 * per_token units (K's first) of a token.
struct Place {
  bool is_v;
  int32_t head, unit;
};
__device__ __forceinline__ Place place(int32_t u, int32_t per_token, int32_t per_row) {
  Place p;
  p.is_v = u >= per_token;
  const int32_t w = p.is_v ? u - per_token : u;
  p.head = w / per_row, p.unit = w % per_row;
  return p;
}

template <typename T>
__device__ __forceinline__ void to_f32(const uint4& raw, float (&v)[8]) {
  const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
}

// A token's page and row; page < 0 where there is none to write to or read from.
struct Found {
  int32_t page, row;
  bool any;   // the token belongs to a sequence
};
__device__ __forceinline__ Found found(const PagedCache& c, int32_t b, int32_t token) {
  Found f{-1, 0, false};
  const paged::Sequence s = paged::sequence(c, b);
  if (token < s.first || token >= s.first + s.count) return f;
  f.any = true;
  const int32_t position = s.position(token - s.first);
  if (position < 0 || position >= s.held) return f;
  f.page = paged::page_or_none(c.table[(int64_t)b * c.table_row + position / c.page_size], c.pages);
  f.row = position % c.page_size;
  return f;
}
__device__ __forceinline__ int32_t of_lane(int32_t v, int lane) { return __builtin_amdgcn_ds_bpermute(lane * 4, v); }
// Of the tokens from `token` on, `n` of them, lane i's is token + i; one: every lane's.
__device__ __forceinline__ Found find(const PagedCache& c, int32_t token, int32_t n) {
  const int32_t lane = threadIdx.x & 63;
  int32_t b = paged::find_sequence(c.batch, token, [&](int32_t i) { return (int64_t)c.starts[i]; });
  if (n == 1) return found(c, b, token);
  const int32_t mine = token + min(lane, n - 1), start = b + lane < c.batch ? c.starts[b + lane] : INT32_MAX;
  int32_t k = 0;   // sequences from b on that start at or in front of the lane's token, by bisection among 64
#pragma unroll
  for (int step = 32; step > 0; step /= 2) k += of_lane(start, k + step - 1) <= mine ? step : 0;
  if (of_lane(start, 63) <= mine) k = 64;
  b += max(k, 1) - 1;
  while (k == 64 && b + 1 < c.batch && c.starts[b + 1] <= mine) ++b;   // (64 sequences and more without tokens)
  return found(c, b, mine);
}

// The wavefront's tokens, unit by unit: move(token, place, page or -1, row).
template <int D, typename F>
__device__ __forceinline__ void each_unit(const PagedCache& c, const Rows& rows, F&& move) {
  constexpr int kRow = D / 8;   // units of a row
  const int32_t first = (blockIdx.x * kWaves + (threadIdx.x >> 6)) * rows.per_wave, lane = threadIdx.x & 63;
  if (first >= c.tokens) return;
  const int32_t n = min(rows.per_wave, c.tokens - first), per_token = c.heads * kRow;
  const Found f = find(c, first, n);
  if (n == 1) {
    if (!f.any) return;
    for (int32_t u = lane; u < 2 * per_token; u += 64) move(first, place(u, per_token, kRow), f.page, f.row);   // (blocks of 4 lanes stay together: kRow is a multiple of 8)
    return;
  }
#pragma unroll 1
  for (int32_t u0 = 0; u0 < n * 2 * per_token; u0 += 64) {
    const int32_t u = u0 + lane, i = min(u / (2 * per_token), n - 1), page = of_lane(f.page, i), row = of_lane(f.row, i), any = of_lane(f.any, i);
    if (any && u < n * 2 * per_token) move(first + i, place(u - i * 2 * per_token, per_token, kRow), page, row);
  }
}

template <typename T, bool MX, int D>
__device__ __forceinline__ void write(const PagedCache& c, const Rows& rows) {
  each_unit<D>(c, rows, [&](int32_t token, const Place& p, int32_t page, int32_t row) {
    if (page < 0) return;
    const unsigned char* from = (p.is_v ? rows.v + (int64_t)token * rows.v_token + (int64_t)p.head * rows.v_head : rows.k + (int64_t)token * rows.k_token + (int64_t)p.head * rows.k_head) + p.unit * 16;
    const uint4 raw = *reinterpret_cast<const uint4*>(from);
    unsigned char* to = (unsigned char*)(p.is_v ? c.v : c.k) + (int64_t)page * c.page_bytes + (int64_t)row * c.row_bytes + (int64_t)p.head * c.head_bytes + p.unit * (MX ? 8 : 16);
    if constexpr (MX) {
      float v[8];
      to_f32<T>(raw, v);
      blocks::quantize_unit<blocks::kMxfp8>(v, blocks::TensorScale{1.0f, 0.0f}, to,
                                            (uint8_t*)(p.is_v ? c.vs : c.ks) + (int64_t)page * c.s_page + (int64_t)row * c.s_row + (int64_t)p.head * c.s_head + p.unit / 4);
    } else {
      *reinterpret_cast<uint4*>(to) = raw;
    }
  });
}

template <typename T, bool MX, int D>
__device__ __forceinline__ void read(const PagedCache& c, const Rows& rows) {
  each_unit<D>(c, rows, [&](int32_t token, const Place& p, int32_t page, int32_t row) {
    unsigned char* to = (p.is_v ? rows.v + (int64_t)token * rows.v_token + (int64_t)p.head * rows.v_head : rows.k + (int64_t)token * rows.k_token + (int64_t)p.head * rows.k_head) + p.unit * 16;
    uint4 raw = {0, 0, 0, 0};
    if (page >= 0) {
      const unsigned char* from = (const unsigned char*)(p.is_v ? c.v : c.k) + (int64_t)page * c.page_bytes + (int64_t)row * c.row_bytes + (int64_t)p.head * c.head_bytes + p.unit * (MX ? 8 : 16);
      if constexpr (MX) {
        const uint2 data = *reinterpret_cast<const uint2*>(from);
        float v[8];
        blocks::unpack_unit<blocks::kMxfp8>(data.x, data.y, (p.is_v ? c.vs : c.ks)[(int64_t)page * c.s_page + (int64_t)row * c.s_row + (int64_t)p.head * c.s_head + p.unit / 4], 1.0f, v);
        T* t = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
      } else {
        raw = *reinterpret_cast<const uint4*>(from);
      }
    }
    *reinterpret_cast<uint4*>(to) = raw;
  });
}

}  // namespace

#define CACHE_KERNELS(NAME, T, MX, D)                                                                                                                      \
  extern "C" __global__ void __launch_bounds__(kWaves * 64) paged_cache_write_entry__##NAME##_d##D(PagedCache c, Rows rows) { write<T, MX, D>(c, rows); } \
  extern "C" __global__ void __launch_bounds__(kWaves * 64) paged_cache_read_entry__##NAME##_d##D(PagedCache c, Rows rows) { read<T, MX, D>(c, rows); }
#define CACHE_KERNELS_D(NAME, T, MX) CACHE_KERNELS(NAME, T, MX, 64) CACHE_KERNELS(NAME, T, MX, 128) CACHE_KERNELS(NAME, T, MX, 256)
CACHE_KERNELS_D(f16, _Float16, false)
CACHE_KERNELS_D(bf16, __bf16, false)
CACHE_KERNELS_D(f16_mxfp8, _Float16, true)
CACHE_KERNELS_D(bf16_mxfp8, __bf16, true)
