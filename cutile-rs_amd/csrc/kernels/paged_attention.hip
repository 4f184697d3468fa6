// Attention of the new tokens of a batch of sequences over a paged cache (paged.h), from one token a sequence to whole prompts:
//   out[i, h, :] = sum_j softmax_j(scale q[i, h, :] . k_j) v_j      over the keys j of the sequence's KV head h / group with p - window < j <= p,
// p the position of token i; no key: zeros.
//
// The rows of a tile are pairs (token, query head of one KV head), token by token: group heads share every key that is read, and a decode step of 8 heads or a
// chunk of 4 tokens fill the columns of a matrix instruction.  S^T = K Q^T and O^T = V^T P^T, so that a lane owns one row and what it holds of P^T is its operand
// of the second product; the softmax keeps a running reference point and sum of each row, in 32 bits.
//  * Tiles of up to 32 rows (decode, drafts): every wavefront has all rows, 16 or 32, and keys of its own, 32 at a time, through registers into LDS that
//    no other wavefront reads: no barrier in the loop.  HBM's rate bounds it: 1 x 131072 tokens, 8 KV heads, bf16, 92 us (5.8 TB/s).  A launch that has no other tiles
//    runs a kernel of four wavefronts (two workgroups on a CU; one at D = 256, whose LDS holds no more), others have eight.  Drafts of 8 tokens of 4 heads behind 64 x 8192 mxfp8 tokens
//    take 174 us so, and 321 where the wavefronts share their keys and a barrier a step.  D = 256 does this for up to 16 rows and only where there are no other tiles: eight wavefronts have no
//    room for keys of their own, so that 17 to 32 rows, and any small tile beside larger ones, go like the larger ones, two wavefronts to 16 rows (the same drafts 604 us, of 4 tokens 309).
//  * Larger tiles: R wavefronts side by side hold kRows rows each, W / R share the keys of a step, which all of them fetch together.  Tiles of all W hold their next
//    scores while the exponentials of the last are made (pipelined_keys).  A prompt of 8192 tokens, 32 heads over 8, D = 128, bf16: 576 us, 954 TFLOP/s of what the
//    rows see; where it was 570, the loop in the order scores, softmax, product took 596, and with a branch around the product, which copied O, 669.
// At the end the partial outputs go through LDS, and where the keys of a tile are dealt to several workgroups through the launch's workspace: the one that
// arrives last adds them up in the order of the keys, so that the order of arrival is nothing to the result.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "fmha_common.h"
#include "kernel_args.h"
#include "paged.h"
#include "split_k.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
constexpr uint32_t kOob = 0x80000000u;

__device__ u32x4 paged_zeros;   // what a key that is not there reads; never written

// 16 e4m3 values of one block as 16-bit ones.
template <typename T>
__device__ __forceinline__ void widen(const u32x4& raw, uint32_t scale_byte, u32x4& lo, u32x4& hi) {
  const float s = __builtin_bit_cast(float, scale_byte << 23);   // the conversion takes the scale by its exponent: byte 0 is 2^-127, 255 NaN
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a, b;
    if constexpr (std::is_same<T, _Float16>::value) {
      a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[i], s, false));
      b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[i], s, true));
    } else {
      a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[i], s, false));
      b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[i], s, true));
    }
    u32x4& to = i < 2 ? lo : hi;
    to[i * 2 % 4] = a, to[i * 2 % 4 + 1] = b;
  }
}

// sum + both 16-bit values of `pair`.
template <typename T>
__device__ __forceinline__ float add_pair(uint32_t pair, float sum) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  if constexpr (std::is_same<T, _Float16>::value) return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), f16x2{1, 1}, sum, false);
  else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), bf16x2{1.0f, 1.0f}, sum, false);
}

// How a wavefront holds X rows (32 or 16) of a tile: S^T and O^T have a row to a column of the matrix instruction, X columns wide, so that lane l has row l % X and, of
// 32 keys, the S values of its group g = l / X; what a lane holds of P^T are then its operands of O^T += V^T P^T, the keys taken in that order.
template <typename T, int D, int X>
struct Shape;
template <typename T, int D>
struct Shape<T, D, 32> {
  using vec8 = typename Elem<T>::vec8;
  using Acc = f32x16;
  static constexpr int kScores = 16, kSteps = 2;            // of 32 keys: values of S a lane holds, matrix products of P
  static constexpr int kInner = 16, kOuter = 32;            // values of D to a product of S, to one of O
  __device__ static __forceinline__ Acc mfma(vec8 a, vec8 b, Acc c) { return Elem<T>::mfma(a, b, c); }
  __device__ static __forceinline__ int key_of(int e, int g) { return (e >> 2) * 8 + g * 4 + (e & 3); }
  __device__ static __forceinline__ int col_of(int e, int g) { return (e >> 2) * 8 + g * 4 + (e & 3); }   // of O^T's rows
  __device__ static __forceinline__ float most(float v) { return max_across_halves(v); }
  __device__ static __forceinline__ float sum(float v) { return sum_across_halves(v); }
};
template <typename T, int D>
struct Shape<T, D, 16> {
  using vec8 = typename Elem<T>::vec8;
  using Acc = f32x4;
  static constexpr int kScores = 8, kSteps = 1;
  static constexpr int kInner = 32, kOuter = 16;
  __device__ static __forceinline__ Acc mfma(vec8 a, vec8 b, Acc c) {
    if constexpr (std::is_same<T, _Float16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ int key_of(int e, int g) { return (e >> 2) * 16 + g * 4 + (e & 3); }
  __device__ static __forceinline__ int col_of(int e, int g) { return g * 4 + e; }
  __device__ static __forceinline__ float most(float v) { return max_across_rows(v); }
  __device__ static __forceinline__ float sum(float v) { return sum_across_rows(v); }
};

// What a workgroup works on: the rows of a tile and its share of their keys.
struct Tile {
  int32_t head;            // KV head
  int32_t row0, rows;      // first packed row of the sequence, number of rows
  int32_t first;           // row of q and out of the sequence's first token
  int32_t pos0;            // position of that token
  int32_t k0, k1;          // keys [k0, k1)
  int32_t all_lo, all_hi;  // keys that all of its rows see, of those that there are
  // Some rows see only a part of keys [key, key + n).
  __device__ __forceinline__ bool partly(int32_t key, int32_t n) const { return key + n - 1 > all_hi || key < all_lo; }
  uint32_t share, shares;
  uint32_t slot;           // of the workspace's counters
  const int32_t* pages;    // the sequence's pages
};

template <typename T, bool MX, int D, int W>
struct Paged {
  using E = Elem<T>;
  using vec8 = typename E::vec8;
  static constexpr int kRows = D == 256 ? 16 : 32;                 // of a larger tile that a wavefront holds: 32 of D = 256 would not fit its registers
  static constexpr int kThreads = W * 64, BM = W * kRows;
  static constexpr int DB = D / 32, KS = D / 16, kUnits = D / 8;   // 16-byte units of a 16-bit row
  // Rows of K and V in LDS are padded so that the lanes of a read meet different banks: 16 bytes for reads of a row a lane, 32 for the transposing ones of
  // four rows.  (Swizzled units, as in fmha.hip, take a register for every address; here they are one address and constants.)
  static constexpr int kRowK = D * 2 + 16, kRowV = D * 2 + 32;
  static constexpr int kOwnBytes = 32 * (kRowK + kRowV);           // 32 keys of a wavefront
  static constexpr int kOwners = D == 256 ? 4 : W;                 // wavefronts that can have keys of their own: what LDS holds
  static constexpr int kLdsBytes = kOwners * kOwnBytes, kBandBytes = kLdsBytes / W;
  static_assert(kBandBytes % 16 == 0 && kBandBytes >= kRows * D * 4 && W % kOwners == 0, "a wavefront's partial output lies where keys were");
  static constexpr int kMostMissed = 2 * (BM / 32 + 2);            // steps that hold a border of what the rows see, at either end
  // Key blocks of a step: short rows leave a load for every thread, long ones the registers that the operands need.
  static constexpr int kStep = D == 64 ? 2 : 1, kWideStep = D == 64 ? 4 : D == 128 ? 2 : 1;
  static constexpr int kLoadUnits = D * (MX ? 1 : 2) / 16;         // 16-byte loads of a row of the cache

  __device__ static __forceinline__ int k_off(int r, int u) { return r * kRowK + u * 16; }
  __device__ static __forceinline__ int v_off(int r, int u) { return r * kRowV + u * 16; }

  // Takes values that are no finite numbers out of 16-bit ones; true if there were some.
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  static constexpr uint16_t kInfinite = std::is_same<T, _Float16>::value ? 0x7c00 : 0x7f80;
  __device__ static __forceinline__ bool clean(u32x4& v) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bad = __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu) >= kInfinite);
      v[i] &= ~bad, any |= bad;
    }
    return any != 0;
  }
  // 16 bytes of K and of V of row r into LDS.  `look`: values of V that are no finite numbers stay out (keys()); true if there were some.
  __device__ static __forceinline__ bool put(unsigned char* sk, unsigned char* sv, int r, int unit, const u32x4& k, u32x4 v, uint32_t ks, uint32_t vs, bool look) {
    bool found = false;
    if constexpr (MX) {
      u32x4 lo, hi;
      widen<T>(k, ks, lo, hi);
      *reinterpret_cast<u32x4*>(sk + k_off(r, unit * 2)) = lo;
      *reinterpret_cast<u32x4*>(sk + k_off(r, unit * 2 + 1)) = hi;
      widen<T>(v, vs, lo, hi);
      if (look) found = clean(lo), found |= clean(hi);
      *reinterpret_cast<u32x4*>(sv + v_off(r, unit * 2)) = lo;
      *reinterpret_cast<u32x4*>(sv + v_off(r, unit * 2 + 1)) = hi;
    } else {
      if (look) found = clean(v);
      *reinterpret_cast<u32x4*>(sk + k_off(r, unit)) = k;
      *reinterpret_cast<u32x4*>(sv + v_off(r, unit)) = v;
    }
    return found;
  }

  // The cache rows of N keys on their way to LDS, by THREADS threads: key r of a step is key `at + r`.
  template <int N, int THREADS>
  struct Loader {
    static constexpr int kLoads = N * kLoadUnits / THREADS, kRowsApart = THREADS / kLoadUnits;
    static_assert(N * kLoadUnits % THREADS == 0 && THREADS % kLoadUnits == 0, "equal shares");
    const PagedCache& c;
    const Tile& t;
    int unit;
    int32_t page_at[kLoads], row_at[kLoads];   // of the next step to be asked for
    int32_t entry[kLoads];                     // its entries of the page table
    int32_t key[kLoads], step;
    u32x4 k[kLoads], v[kLoads];
    uint32_t ks[MX ? kLoads : 1], vs[MX ? kLoads : 1];

    __device__ __forceinline__ Loader(const PagedCache& cache, const Tile& tile, int tid, int32_t start, int32_t by) : c(cache), t(tile), step(by) {
      unit = tid % kLoadUnits;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        key[i] = start + tid / kLoadUnits + i * kRowsApart;
        page_at[i] = key[i] / c.page_size;
        row_at[i] = key[i] % c.page_size;
      }
      ask();
    }
    __device__ __forceinline__ void ask() {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) entry[i] = key[i] < t.k1 ? t.pages[page_at[i]] : -1;
    }
    // Asks for the step's rows, and for the page-table entries of the next.
    __device__ __forceinline__ void load() {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const bool there = (uint32_t)entry[i] < (uint32_t)c.pages;
        const int64_t off = (int64_t)entry[i] * c.page_bytes + (int64_t)row_at[i] * c.row_bytes + (int64_t)t.head * c.head_bytes + unit * 16;
        k[i] = *(there ? (const u32x4*)((const unsigned char*)c.k + off) : &paged_zeros);
        v[i] = *(there ? (const u32x4*)((const unsigned char*)c.v + off) : &paged_zeros);
        if constexpr (MX) {
          const int64_t s = (int64_t)entry[i] * c.s_page + (int64_t)row_at[i] * c.s_row + (int64_t)t.head * c.s_head + unit / 2;
          ks[i] = *(there ? c.ks + s : (const uint8_t*)&paged_zeros);
          vs[i] = *(there ? c.vs + s : (const uint8_t*)&paged_zeros);
        }
        key[i] += step;
        page_at[i] += step / c.page_size;
        row_at[i] += step % c.page_size;
        if (row_at[i] >= c.page_size) row_at[i] -= c.page_size, ++page_at[i];
      }
      ask();
    }
    // True in a lane that kept a value of V back.
    __device__ __forceinline__ bool store(unsigned char* sk, unsigned char* sv, int tid, bool look) {
      bool found = false;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) found |= put(sk, sv, tid / kLoadUnits + i * kRowsApart, unit, k[i], v[i], ks[MX ? i : 0], vs[MX ? i : 0], look);
      return found;
    }
  };

  // The same of 32 keys by one wavefront.  Lane r looks key r up, and the lanes that fetch its row have the place from there; of mxfp8 keys lane r holds the scales of K and lane
  // 32 + r those of V.  (What counts is how often the first-level cache is asked: a load of 64 bytes of each of 16 rows, as the operands of K lie, or a scale byte for
  // every lane cost as much as one of whole rows: 64 x 8192 mxfp8 189 us that way.)
  struct OwnKeys {
    static constexpr int kLoads = 32 * kLoadUnits / 64, kRowsAtOnce = 64 / kLoadUnits, kScaleWords = D == 256 ? 2 : 1;
    typedef uint32_t Scales __attribute__((ext_vector_type(kScaleWords)));
    const PagedCache& c;
    const Tile& t;
    const int lane, step;
    int32_t key, page_at, row_at, entry;
    u32x4 k[kLoads], v[kLoads];
    Scales scales;

    __device__ __forceinline__ OwnKeys(const PagedCache& cache, const Tile& tile, int32_t start, int32_t by) : c(cache), t(tile), lane(threadIdx.x & 63), step(by) {
      key = start + (lane & 31);
      page_at = key / c.page_size, row_at = key % c.page_size;
      ask();
    }
    __device__ __forceinline__ void ask() { entry = key < t.k1 ? t.pages[page_at] : -1; }
    // `word` of lane `from`.
    __device__ __forceinline__ static uint32_t of_lane(uint32_t word, int from) { return __builtin_amdgcn_ds_bpermute(from * 4, (int)word); }
    // Asks for the next 32 keys, and for the page-table entries of those behind them.
    __device__ __forceinline__ void load() {
      const int unit = lane % kLoadUnits;
      const bool there = (uint32_t)entry < (uint32_t)c.pages;
      const int64_t off = there ? (int64_t)entry * c.page_bytes + (int64_t)row_at * c.row_bytes : -1;
      if constexpr (MX) {
        const uint8_t* from = (lane < 32 ? c.ks : c.vs) + (int64_t)entry * c.s_page + (int64_t)row_at * c.s_row + (int64_t)t.head * c.s_head;
        if (!there) from = (const uint8_t*)&paged_zeros;
        if constexpr (D == 64) scales[0] = *(const uint16_t*)from;
        else scales = *(const Scales*)from;
      }
      const unsigned char *kb = (const unsigned char*)c.k + (int64_t)t.head * c.head_bytes + unit * 16, *vb = (const unsigned char*)c.v + (int64_t)t.head * c.head_bytes + unit * 16;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = lane / kLoadUnits + i * kRowsAtOnce;
        const int64_t at = (int64_t)((uint64_t)of_lane((uint32_t)(off >> 32), r) << 32 | of_lane((uint32_t)off, r));
        k[i] = __builtin_nontemporal_load(at >= 0 ? (const u32x4*)(kb + at) : &paged_zeros);
        v[i] = __builtin_nontemporal_load(at >= 0 ? (const u32x4*)(vb + at) : &paged_zeros);
      }
      key += step;
      page_at += step / c.page_size;
      row_at += step % c.page_size;
      if (row_at >= c.page_size) row_at -= c.page_size, ++page_at;
      ask();
    }
    // The scale byte of block `block` of row r; `first`: lane of row 0.
    __device__ __forceinline__ uint32_t scale_of(int first, int r, int block) const {
      uint32_t word = of_lane(scales[0], first + r);
      if constexpr (kScaleWords == 2) {
        const uint32_t second = of_lane(scales[kScaleWords - 1], first + r);
        word = block >= 4 ? second : word;
      }
      return word >> (block % 4 * 8) & 0xff;
    }
    __device__ __forceinline__ bool store(unsigned char* sk, unsigned char* sv, bool look) {
      const int unit = lane % kLoadUnits;
      bool found = false;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = lane / kLoadUnits + i * kRowsAtOnce;
        if constexpr (MX) found |= put(sk, sv, r, unit, k[i], v[i], scale_of(0, r, unit / 2), scale_of(32, r, unit / 2), look);
        else found |= put(sk, sv, r, unit, k[i], v[i], 0, 0, look);
      }
      return found;
    }
  };

  // X rows of a tile as a wavefront holds them.
  template <int X>
  struct Rows {
    using H = Shape<T, D, X>;
    vec8 q[D / H::kInner];
    typename H::Acc o[D / H::kOuter];
    float m, l;               // of the lane's row; l of the lane's share of the keys
    float limit;              // of the row's scores: m moves where one is above it
    int32_t lo, hi;           // keys the lane's row sees
    int32_t all_lo, all_hi;   // that every row of the wavefront sees
    int32_t any_lo, any_hi;   // that one of them sees
    bool used;
    int missed;               // steps of whose V values were kept back
  };

  template <int X>
  __device__ static __forceinline__ void begin(Rows<X>& w, const Tile& t, const TensorArg<3>& q, const PagedPlan& p, int row_block) {
    using H = Shape<T, D, X>;
    const int lane = threadIdx.x & 63;
    const int32_t r0 = row_block * X, n = min(X, t.rows - r0);
    w.used = n > 0;
    const int32_t r = t.row0 + r0 + min(lane % X, max(n, 1) - 1), token = r / p.group, head = r % p.group;   // (lanes beyond the last row repeat it)
    const T* from = (const T*)q.ptr + (int64_t)(t.first + token) * q.strides[0] + (int64_t)(t.head * p.group + head) * q.strides[1];
#pragma unroll
    for (auto& part : w.q) part = vec8{};
    if (w.used) {
#pragma unroll
      for (int ks = 0; ks < D / H::kInner; ++ks) w.q[ks] = __builtin_bit_cast(vec8, (*reinterpret_cast<const u32x4*>(from + ks * H::kInner + lane / X * 8) & p.q_and) ^ p.q_xor);
    }
    auto low = [&](int32_t pos) { return p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0; };
    const int32_t pos = t.pos0 + token, first = t.pos0 + (t.row0 + r0) / p.group, last = t.pos0 + (t.row0 + r0 + max(n, 1) - 1) / p.group;
    w.lo = low(pos), w.hi = min(pos, t.k1 - 1);
    w.any_lo = low(first), w.all_lo = low(last);
    w.all_hi = min(first, t.k1 - 1), w.any_hi = min(last, t.k1 - 1);
    w.m = w.limit = -INFINITY, w.l = 0.0f, w.missed = 0;
#pragma unroll
    for (auto& o : w.o) o = typename H::Acc{};
  }

  // S^T of 32 keys in LDS.
  template <int X>
  __device__ static __forceinline__ void scores(const Rows<X>& w, const unsigned char* sk, float (&s)[Shape<T, D, X>::kScores]) {
    using H = Shape<T, D, X>;
    const int lane = threadIdx.x & 63;
    constexpr int kEach = H::kScores * X / 32;
#pragma unroll
    for (int i = 0; i < 32 / X; ++i) {
      typename H::Acc acc = {};
#pragma unroll
      for (int ks = 0; ks < D / H::kInner; ++ks)
        acc = H::mfma(*reinterpret_cast<const vec8*>(sk + k_off(i * X + lane % X, ks * (H::kInner / 8) + lane / X)), w.q[ks], acc);
#pragma unroll
      for (int e = 0; e < kEach; ++e) s[i * kEach + e] = acc[e];
    }
  }

  // The operand V^T of O's rows ob * kOuter .. and the keys of step t.
  template <int X>
  __device__ static __forceinline__ vec8 v_frag(const unsigned char* sv, int t, int ob) {
    const int lane = threadIdx.x & 63, grp = lane >> 4, l16 = lane & 15;
    const int col = ob * Shape<T, D, X>::kOuter + (X == 32 ? (grp & 1) * 16 : 0) + (l16 & 3) * 4, row = t * 16 + (X == 32 ? grp >> 1 : grp) * 4 + (l16 >> 2);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(sv + v_off(row, 0) + col * 2));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(sv + v_off(row + (X == 32 ? 8 : 16), 0) + col * 2));
    return __builtin_bit_cast(vec8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }

  // The softmax of B blocks of 32 keys, in steps.  What the lane's row does not see of S^T, from `key0` on:
  template <int X, int B, typename S>
  __device__ static __forceinline__ void hide(const Rows<X>& w, S (&s)[B], int32_t key0) {
    using H = Shape<T, D, X>;
    if (key0 + B * 32 - 1 <= w.all_hi && key0 >= w.all_lo) return;
    const int g = (threadIdx.x & 63) / X;
    const int32_t hi = w.hi - key0 - g * 4, lo = w.lo - key0 - g * 4;
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int e = 0; e < H::kScores; ++e) {
        const int kk = b * 32 + H::key_of(e, 0);
        s[b][e] = kk <= hi && kk >= lo ? s[b][e] : -INFINITY;
      }
  }
  template <int X, int B, typename S>
  __device__ static __forceinline__ float highest(S (&s)[B]) {
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int e = 0; e < Shape<T, D, X>::kScores; ++e) mx = fmaxf(mx, s[b][e]);
    return mx;
  }
  // The row's reference point, `mx` being the lane's highest new score.  It only has to bound the exponents: it moves when a row's maximum has risen by more than kSlack.
  // Weights are held 2^kLift times what they are against it, and so are O and their sum.  bf16 has the range of f32.  f16's ends at 2^16, and below 2^-14 its steps are 2^-24: lifted to
  // 2^15 at most, a weight is rounded like the others down to 2^-25 of the reference point and off by 2^-36 of it beyond (without the lift 2^-14 and 2^-25: 40000 keys of 2^-26 of the
  // largest each, 6 parts in 10000 of the row together, were lost).  A slack of 4 takes no longer than one of 8, whose lift would be 7: prompt of 8192 in f16 626 us against 627; 2: 631.
  static constexpr float kSlack = std::is_same<T, _Float16>::value ? 4.0f : 8.0f, kLift = std::is_same<T, _Float16>::value ? 15.0f - kSlack : 0.0f;
  // What the three roundings between a score and its exponent (the point's own, its lift, the limit) add stays below 2^-22 of the point; of f16, where 2^16 is too much, twice that is left
  // free above the point and below the limit, up to 2^25 (scores beyond are not told apart by f32 anyway).
  template <int X>
  __device__ static __forceinline__ void move(Rows<X>& w, float mx, float c) {
    const float top = Shape<T, D, X>::most(mx) * c;
    if (__builtin_amdgcn_ballot_w64(top > w.limit) == 0) return;
    auto free = [](float point) { return kLift > 0.0f ? fminf(fabsf(point) * 0x1p-21f, 16.0f) : 0.0f; };
    const float to = top > w.m ? top + free(top) : w.m;
    const float alpha = __builtin_amdgcn_exp2f(w.m - (to == -INFINITY ? 0.0f : to));
    w.l *= alpha;
#pragma unroll
    for (auto& o : w.o) o *= alpha;
    w.m = to, w.limit = to + (kSlack - free(to));
  }
  // Keeps the compiler from moving the making of x behind this place.
  template <typename U>
  __device__ static __forceinline__ void here(U& x) {
    asm volatile("" : "+v"(x));
  }
  // P in 16 bits, as V is: the weights' rounding stays below that of V (f16 weights below its normal range: move()), and their sum is that of the rounded ones.  All at once, or a
  // part at a time (m of `of`).
  template <int X, int B>
  struct Exponentials {
    using H = Shape<T, D, X>;
    static constexpr int kPairs = B * H::kScores / 2;
    Rows<X>& w;
    float (&s)[B][H::kScores];
    vec8 (&pf)[B][H::kSteps];
    const float c, m;
    float sum[2];
    u32x4 p[B][H::kSteps];
    __device__ __forceinline__ Exponentials(Rows<X>& rows, float (&scores)[B][H::kScores], vec8 (&weights)[B][H::kSteps], float scale)
        : w(rows), s(scores), pf(weights), c(scale), m((rows.m == -INFINITY ? 0.0f : rows.m) - kLift) {   // (nothing seen so far: keep exp2 finite)
      sum[0] = w.l, sum[1] = 0.0f;
    }
    __device__ __forceinline__ void raise(int i) {
      float& x = s[i / H::kScores][i % H::kScores];
      x = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c, -m));
    }
    __device__ __forceinline__ void pack(int i) {
      const int b = i / (H::kScores / 2), r = i % (H::kScores / 2);
      const uint32_t v = E::pack2(s[b][2 * r], s[b][2 * r + 1]);
      p[b][r / 4][r % 4] = v;
      sum[i % 2] = add_pair<T>(v, sum[i % 2]);
    }
    __device__ __forceinline__ void operator()(int part, int of) {
#pragma unroll
      for (int i = part * kPairs / of; i < (part + 1) * kPairs / of; ++i) raise(2 * i), raise(2 * i + 1);
#pragma unroll
      for (int i = part ? (part - 1) * kPairs / of : 0; i < part * kPairs / of; ++i) pack(i);
      if (part == of - 1) {
#pragma unroll
        for (int i = part * kPairs / of; i < kPairs; ++i) pack(i);
      }
      if (of > 1) {
#pragma unroll
        for (int i = 2 * (part * kPairs / of); i < 2 * ((part + 1) * kPairs / of); ++i) here(s[i / H::kScores][i % H::kScores]);
        here(sum[0]), here(sum[1]);
      }
    }
    __device__ __forceinline__ void end() {
      w.l = sum[0] + sum[1];
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int t = 0; t < H::kSteps; ++t) pf[b][t] = __builtin_bit_cast(vec8, p[b][t]);
    }
  };

  // B blocks of 32 keys from `key0` on, V at sv: `scores_of`(s) gives S^T, then the softmax so far and O^T.  Values of V that are no finite numbers must not reach
  // rows that do not see their keys, and 0 times them would: of keys that only some rows of the tile see they are kept out of LDS (`apart`), and come to the rows
  // that see them later (add_missed).
  template <int X, int B, typename F>
  __device__ static __forceinline__ void keys(Rows<X>& w, F&& scores_of, const unsigned char* sv, int32_t key0, float c, bool apart, int32_t* missed) {
    using H = Shape<T, D, X>;
    float s[B][H::kScores];   // s[b][e] belongs to key key0 + b * 32 + key_of(e, g) and to this lane's row
    scores_of(s);
    vec8 pf[B][H::kSteps];
    hide<X, B>(w, s, key0);
    move<X>(w, highest<X, B>(s), c);
    Exponentials<X, B> weights(w, s, pf, c);
    weights(0, 1);
    weights.end();
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int t = 0; t < H::kSteps; ++t)
#pragma unroll
        for (int ob = 0; ob < D / H::kOuter; ++ob) w.o[ob] = H::mfma(v_frag<X>(sv + b * 32 * kRowV, t, ob), pf[b][t], w.o[ob]);
    if (apart && w.missed < kMostMissed) missed[w.missed++] = key0;
  }

  // LDS operations of one wavefront happen in order; the compiler is kept to it.
  __device__ static __forceinline__ void ordered() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // What the values that were kept back in the noted steps of `blocks` x 32 keys make of the rows that see their keys, found by a product of marks with 0 and 1.
  // The steps' V goes through LDS at sv.
  template <int X>
  __device__ static __forceinline__ void add_missed(Rows<X>& w, const Tile& t, const PagedCache& c, unsigned char* sv, const int32_t* missed, int blocks) {
    using H = Shape<T, D, X>;
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    constexpr bool kHalf = std::is_same<T, _Float16>::value;
    constexpr uint16_t kOne = kHalf ? 0x3c00 : 0x3f80, k64 = kHalf ? 0x5400 : 0x4280, k4096 = kHalf ? 0x6c00 : 0x4580;
    const int lane = threadIdx.x & 63, g = lane / X, unit = lane % kLoadUnits;
#pragma unroll 1
    for (int n = 0; n < w.missed * blocks; ++n) {
      const int32_t key0 = missed[n / blocks] + n % blocks * 32;
#pragma unroll 1
      for (int r = lane / kLoadUnits; r < 32; r += 64 / kLoadUnits) {
        const int32_t at = key0 + r, entry = at < t.k1 ? t.pages[at / c.page_size] : -1;
        u32x4 v = {0, 0, 0, 0};
        uint32_t vs = 0;
        if ((uint32_t)entry < (uint32_t)c.pages) {
          v = *(const u32x4*)((const unsigned char*)c.v + (int64_t)entry * c.page_bytes + (int64_t)(at % c.page_size) * c.row_bytes + (int64_t)t.head * c.head_bytes + unit * 16);
          if constexpr (MX) vs = c.vs[(int64_t)entry * c.s_page + (int64_t)(at % c.page_size) * c.s_row + (int64_t)t.head * c.s_head + unit / 2];
        }
        if constexpr (MX) {
          u32x4 lo, hi;
          widen<T>(v, vs, lo, hi);
          *reinterpret_cast<u32x4*>(sv + v_off(r, unit * 2)) = lo;
          *reinterpret_cast<u32x4*>(sv + v_off(r, unit * 2 + 1)) = hi;
        } else {
          *reinterpret_cast<u32x4*>(sv + v_off(r, unit)) = v;
        }
      }
      ordered();
      vec8 sees[H::kSteps];   // 1 where the lane's row sees the key
#pragma unroll
      for (int t = 0; t < H::kSteps; ++t) {
        u16x8 x;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int32_t kk = key0 + H::key_of(t * 8 + i, g);
          x[i] = kk >= w.lo && kk <= w.hi ? kOne : 0;
        }
        sees[t] = __builtin_bit_cast(vec8, x);
      }
#pragma unroll
      for (int ob = 0; ob < D / H::kOuter; ++ob) {
        typename H::Acc marks = {};   // of the keys that the row sees: 1 for each NaN, 64 for each infinity, 4096 for each negative one
#pragma unroll
        for (int t = 0; t < H::kSteps; ++t) {
          const u16x8 f = __builtin_bit_cast(u16x8, v_frag<X>(sv, t, ob));
          u16x8 mark;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint16_t mag = f[i] & 0x7fff;
            mark[i] = mag > kInfinite ? kOne : mag < kInfinite ? (uint16_t)0 : f[i] >> 15 ? k4096 : k64;
          }
          marks = H::mfma(__builtin_bit_cast(vec8, mark), sees[t], marks);
        }
#pragma unroll
        for (int e = 0; e < (int)(sizeof(marks) / 4); ++e) {
          const int of = (int)marks[e];
          w.o[ob][e] += (of & 63 ? NAN : 0.0f) + (of & 4032 ? INFINITY : 0.0f) - (of >> 12 ? INFINITY : 0.0f);
        }
      }
      ordered();
    }
  }

  // Up to X rows: wavefront w has the keys k0 + 32 w, + 32 (w + W), ..., 32 of them at a time in LDS at sk and sv.
  template <int X>
  __device__ static __forceinline__ void own_keys(Rows<X>& w, const Tile& t, const PagedCache& c, float scale, unsigned char* sk, unsigned char* sv, int32_t* missed) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int kBy = W * 32;
    int32_t key0 = t.k0 + wave * 32;
    if (key0 < t.k1) {
      OwnKeys in(c, t, key0, kBy);
      in.load();
#pragma unroll 1
      for (; key0 < t.k1; key0 += kBy) {
        ordered();
        const bool apart = __builtin_amdgcn_ballot_w64(in.store(sk, sv, t.partly(key0, 32))) != 0;
        ordered();
        in.load();
        keys<X, 1>(w, [&](float (&s)[1][Shape<T, D, X>::kScores]) { scores<X>(w, sk, s[0]); }, sv, key0, scale, apart, missed);
      }
    }
    ordered();
    add_missed(w, t, c, sv, missed, 1);
  }

  // R x X rows: wavefront (r, s) has the rows of block r and the key blocks s * B .. of every step of S * B * 32 keys, which all wavefronts fetch together.
  template <int X, int R, int B>
  __device__ static __forceinline__ void shared_keys(Rows<X>& w, const Tile& t, const PagedCache& c, float scale, unsigned char* lds, int32_t* apart_at, int32_t* missed) {
    constexpr int S = W / R, N = S * B * 32, kStage = N * (kRowK + kRowV);
    static_assert(2 * kStage <= kLdsBytes, "two stages");
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ws = wave % S;
    if (t.k0 >= t.k1) return;
    Loader<N, kThreads> in(c, t, threadIdx.x, t.k0, N);
    // the step whose V in that stage had values kept back: known to all behind the barrier
    if (threadIdx.x < 2) apart_at[threadIdx.x] = -1;
    __syncthreads();
    in.load();
    if (in.store(lds, lds + N * kRowK, threadIdx.x, t.partly(t.k0, N))) apart_at[0] = t.k0;
    __syncthreads();
    int cur = 0;
#pragma unroll 1
    for (int32_t key = t.k0; key < t.k1; key += N) {
      const bool more = key + N < t.k1;
      if (more) in.load();
      const unsigned char* stage = lds + cur * kStage;
      const int32_t key0 = key + ws * B * 32;
      if (w.used && key0 <= w.any_hi && key0 + B * 32 > w.any_lo)
        keys<X, B>(w, [&](float (&s)[B][Shape<T, D, X>::kScores]) {
#pragma unroll
          for (int b = 0; b < B; ++b) scores<X>(w, stage + (ws * B + b) * 32 * kRowK, s[b]);
        }, stage + N * kRowK + ws * B * 32 * kRowV, key0, scale, __builtin_amdgcn_readfirstlane(apart_at[cur]) == key, missed);
      cur ^= 1;
      if (more && in.store(lds + cur * kStage, lds + cur * kStage + N * kRowK, threadIdx.x, t.partly(key + N, N))) apart_at[cur] = key + N;
      __syncthreads();
    }
  }

  // K of step g and V of step g - 1 on their way to LDS, by all wavefronts: what pipelined_keys takes together.  A load of a wavefront is a group of kGroup whole rows;
  // where a group never crosses the end of a page (grouped()) its place is a scalar address, and the vector ALU has nothing to do with it.
  template <int N>
  struct GroupLoader {
    static constexpr int kGroup = 64 / kLoadUnits, kLoads = N / (W * kGroup);
    static_assert(64 % kLoadUnits == 0 && N % (W * kGroup) == 0, "whole groups, equal shares");
    typedef const int32_t __attribute__((address_space(4))) * Entries;
    const PagedCache& c;
    const Tile& t;
    const int row, unit, wave;       // the lane's row of a group, its 16 bytes of it
    const int64_t at, s_at;          // its place in the group
    int32_t key[kLoads], page_at[kLoads], row_at[kLoads], entry[kLoads];   // of the groups to be asked for next
    int64_t off[kLoads], s_off[kLoads];                     // of the groups asked for last, or -1
    u32x4 k[kLoads], v[kLoads];
    uint32_t ks[MX ? kLoads : 1], vs[MX ? kLoads : 1];

    __device__ static __forceinline__ bool grouped(const PagedCache& c, const Tile& t) { return c.page_size % kGroup == 0 && t.k0 % kGroup == 0; }
    __device__ __forceinline__ GroupLoader(const PagedCache& cache, const Tile& tile)
        : c(cache), t(tile), row((threadIdx.x & 63) / kLoadUnits), unit(threadIdx.x % kLoadUnits), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
          at(row * c.row_bytes + unit * 16), s_at(row * c.s_row + unit / 2) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        key[i] = t.k0 + (wave + i * W) * kGroup;
        page_at[i] = key[i] / c.page_size, row_at[i] = key[i] % c.page_size;
        off[i] = -1, s_off[i] = 0;
      }
      ask();
    }
    __device__ __forceinline__ void ask() {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) entry[i] = key[i] < t.k1 ? ((Entries)t.pages)[page_at[i]] : -1;
    }
    __device__ __forceinline__ void load() {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        v[i] = u32x4{0, 0, 0, 0}, k[i] = u32x4{0, 0, 0, 0};
        if constexpr (MX) vs[i] = 0, ks[i] = 0;
        if (off[i] >= 0) {
          v[i] = *(const u32x4*)((const unsigned char*)c.v + off[i] + at);
          if constexpr (MX) vs[i] = *(c.vs + s_off[i] + s_at);
        }
        off[i] = -1;
        if ((uint32_t)entry[i] < (uint32_t)c.pages) {
          off[i] = (int64_t)entry[i] * c.page_bytes + (int64_t)row_at[i] * c.row_bytes + (int64_t)t.head * c.head_bytes;
          k[i] = *(const u32x4*)((const unsigned char*)c.k + off[i] + at);
          if constexpr (MX) {
            s_off[i] = (int64_t)entry[i] * c.s_page + (int64_t)row_at[i] * c.s_row + (int64_t)t.head * c.s_head;
            ks[i] = *(c.ks + s_off[i] + s_at);
          }
        }
        key[i] += N;
        page_at[i] += N / c.page_size;
        row_at[i] += N % c.page_size;
        if (row_at[i] >= c.page_size) row_at[i] -= c.page_size, ++page_at[i];
      }
      ask();
    }
    // True in a lane that kept a value of V back: `look`, as put().  What lies behind the context is among what only some rows see.
    __device__ __forceinline__ bool store(unsigned char* sk, unsigned char* sv, bool look) {
      bool found = false;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) found |= put(sk, sv, (wave + i * W) * kGroup + row, unit, k[i], v[i], ks[MX ? i : 0], vs[MX ? i : 0], look);
      return found;
    }
  };

  // Order of what stands in front of this: N matrix products, each with two reads of LDS for the third one behind it and an operation of the vector ALU.
  template <int N>
  __device__ static __forceinline__ void dealt() {
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
    }
  }

  // W x X rows, a wavefront to X of them, in steps of N = B x 32 keys (D of 128 and 256; rows of 64 are so short that a step is mostly exponentials and larger steps
  // gain more: 365 us against 390 for the prompt).  The vector ALU has the exponentials of a step while the matrix cores have the scores of the next,
  // then the highest of those while they have the product with V:  S(j + 1) | exponentials(j),  O(j) | highest(j + 1).
  // There are two buffers of K and of V; K(j + 2) and V(j + 1) are written over K(j) and V(j - 1) at the start of step j, from registers that were asked for in step j - 1.
  template <int X, int B>
  __device__ static __forceinline__ void pipelined_keys(Rows<X>& w, const Tile& t, const PagedCache& c, float scale, unsigned char* lds, int32_t* apart_at, int32_t* missed) {
    using H = Shape<T, D, X>;
    constexpr int N = B * 32, kBlocks = N / X, kEach = H::kScores * X / 32, KS = D / H::kInner, OB = D / H::kOuter;
    static_assert(2 * N * (kRowK + kRowV) <= kLdsBytes, "two buffers of each");
    const int lane = threadIdx.x & 63;
    const int32_t steps = (t.k1 - t.k0 + N - 1) / N;
    if (steps <= 0) return;
    auto k_at = [&](int32_t j) { return lds + (j & 1) * (N * kRowK); };
    auto v_at = [&](int32_t j) { return lds + 2 * N * kRowK + (j & 1) * (N * kRowV); };
    GroupLoader<N> in(c, t);
    auto store = [&](int32_t j) {   // V of step j, K of the next
      const int32_t key0 = t.k0 + j * N;
      if (in.store(k_at(j + 1), v_at(j), t.partly(key0, N))) apart_at[j & 1] = j;
      in.load();
    };
    // `beside`(m, of): what the vector ALU does at matrix product m.
    auto scores_of = [&](int32_t j, float (&s)[B][H::kScores], auto&& beside) {
      constexpr int kProducts = kBlocks * KS, kAhead = kProducts < 4 ? kProducts : 4;
      const unsigned char* sk = k_at(j);
      auto operand = [&](int m) { return *reinterpret_cast<const vec8*>(sk + k_off(m % kBlocks * X + lane % X, m / kBlocks * (H::kInner / 8) + lane / X)); };
      typename H::Acc acc[kBlocks] = {};
      vec8 ahead[kAhead];
#pragma unroll
      for (int m = 0; m < kAhead; ++m) ahead[m] = operand(m);
#pragma unroll
      for (int m = 0; m < kProducts; ++m) {
        acc[m % kBlocks] = H::mfma(ahead[m % kAhead], w.q[m / kBlocks], acc[m % kBlocks]);
        if (m + kAhead < kProducts) ahead[m % kAhead] = operand(m + kAhead);
        beside(m, kProducts);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int e = 0; e < kEach; ++e) s[i * X / 32][i * kEach % H::kScores + e] = acc[i][e];
    };
    if (threadIdx.x < 2) apart_at[threadIdx.x] = -2;
    in.load();
    __syncthreads();
    store(-1);
    store(0);
    __syncthreads();
    float s0[B][H::kScores], s1[B][H::kScores];
    scores_of(0, s0, [](int, int) {});
    hide<X, B>(w, s0, t.k0);
    move<X>(w, highest<X, B>(s0), scale);
    __syncthreads();
    auto step = [&](int32_t j, float (&s)[B][H::kScores], float (&next)[B][H::kScores]) {
      const int32_t key0 = t.k0 + j * N;
      store(j + 1);
      if (w.used && key0 <= w.any_hi) {   // (no row of the wavefront sees later keys)
        vec8 pf[B][H::kSteps];
        Exponentials<X, B> weights(w, s, pf, scale);
        scores_of(j + 1, next, weights);
        weights.end();
        hide<X, B>(w, next, key0 + N);
        const unsigned char* sv = v_at(j);
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
          for (int k = 0; k < H::kSteps; ++k)
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) w.o[ob] = H::mfma(v_frag<X>(sv + b * 32 * kRowV, k, ob), pf[b][k], w.o[ob]);
        float mx = highest<X, B>(next);
        dealt<B * H::kSteps * OB>();
        here(mx);
        if (__builtin_amdgcn_readfirstlane(apart_at[j & 1]) == j && w.missed < kMostMissed) missed[w.missed++] = key0;
        move<X>(w, mx, scale);
      }
      __syncthreads();
    };
#pragma unroll 1
    for (int32_t j = 0; j < steps; j += 2) {
      step(j, s0, s1);
      if (j + 1 < steps) step(j + 1, s1, s0);
    }
  }

  // Columns 4 u .. of a row, divided and rounded.
  __device__ static __forceinline__ void store_row(const PartitionArg<3>& out, const Tile& t, const PagedPlan& p, int32_t row, int u, const f32x4& o, float l) {
    const int32_t r = t.row0 + row, token = r / p.group, head = r % p.group;
    const float sum = l == 0.0f ? 1.0f : l;   // a row that saw no key: 0
    const u32x2 v = {E::pack2(o[0] / sum, o[1] / sum), E::pack2(o[2] / sum, o[3] / sum)};
    *reinterpret_cast<u32x2*>((T*)out.ptr + (int64_t)(t.first + token) * out.strides[0] + (int64_t)(t.head * p.group + head) * out.strides[1] + u * 4) = v;
  }

  // The results of the wavefronts, S to X rows, and of the tile's other workgroups to out.
  template <int X>
  __device__ static __forceinline__ void finish(Rows<X>& w, const Tile& t, const PartitionArg<3>& out, const PagedPlan& p, unsigned char* partials, int32_t slot_rows, unsigned char* lds,
                                                float (*stat)[2][32], uint32_t* flag, int S) {
    using H = Shape<T, D, X>;
    constexpr int U = D / 4, kRowsAtOnce = kThreads / U;
    const int tid = threadIdx.x, lane = tid & 63, row_of = lane % X, g = lane / X, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float l = H::sum(w.l);
    if (g == 0) stat[wave][0][row_of] = w.m, stat[wave][1][row_of] = l;
    unsigned char* band = lds + wave * kBandBytes + row_of * (D * 4);   // column unit u of a row lies at u ^ (row % 16)
#pragma unroll
    for (int ob = 0; ob < D / H::kOuter; ++ob)
#pragma unroll
      for (int e = 0; e < (int)(sizeof(typename H::Acc) / 4); e += 4)
        *reinterpret_cast<f32x4*>(band + (((ob * (H::kOuter / 4) + H::col_of(e, g) / 4) ^ (row_of & 15)) << 4)) = f32x4{w.o[ob][e], w.o[ob][e + 1], w.o[ob][e + 2], w.o[ob][e + 3]};
    __syncthreads();
    const uint32_t bytes = (uint32_t)slot_rows * (D + 4) * 4, stats = (uint32_t)slot_rows * D * 4;   // of a share of the workspace
    const __amdgpu_buffer_rsrc_t part = make_rsrc(partials, bytes * t.shares);
    const int u = tid % U;
#pragma unroll 1
    for (int row = tid / U; row < t.rows; row += kRowsAtOnce) {
      const int first = row / X * S, r = row % X;
      float top = -INFINITY;
      for (int s = 0; s < S; ++s) top = fmaxf(top, stat[first + s][0][r]);
      const float use = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
      f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int s = 0; s < S; ++s) {
        const float by = __builtin_amdgcn_exp2f(stat[first + s][0][r] - use);
        sum = __builtin_fmaf(stat[first + s][1][r], by, sum);
        const f32x4 v = *reinterpret_cast<const f32x4*>(lds + (first + s) * kBandBytes + r * (D * 4) + ((u ^ (r & 15)) << 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(v[e], by, o[e]);
      }
      if (t.shares == 1) {
        store_row(out, t, p, row, u, o, sum);
      } else {
        gemm::store_partial(o, part, t.share * bytes + (uint32_t)row * (D * 4) + u * 16);
        if (u == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{top, sum}), part, t.share * bytes + stats + row * 8, 0, gemm::kAgentScope);
      }
    }
    if (t.shares == 1 || !gemm::last_to_arrive(p.counters + t.slot, t.shares, flag)) return;
    // A read past the L2 takes a microsecond, so sixteen are under way together: of one row or two where there are many shares, of several where there are few (the chunk
    // of 512 tokens behind 16384, four shares of 256 rows: 157 us, 163 one row at a time).
    if (W == 4 || t.rows <= kRowsAtOnce) add_shares<1, 8>(t, out, p, part, bytes, lds);
    else if (t.shares > 4) add_shares<2, 8>(t, out, p, part, bytes, lds);
    else if (t.shares > 2) add_shares<4, 4>(t, out, p, part, bytes, lds);
    else add_shares<8, 2>(t, out, p, part, bytes, lds);
  }

  // A row's result so far: columns 4 u .., reference point and sum.
  struct Sum {
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    __device__ __forceinline__ void add(const f32x4& x, float top_of, float sum_of) {
      const float top = fmaxf(m, top_of), use = top == -INFINITY ? 0.0f : top, was = __builtin_amdgcn_exp2f(m - use), by = __builtin_amdgcn_exp2f(top_of - use);
      m = top, l = __builtin_fmaf(sum_of, by, l * was);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[e], by, o[e] * was);
    }
  };
  // The tile's shares in the order of the keys, R rows and K shares of a thread under way together; of few rows (R = 1) they are dealt to several groups of threads, whose
  // sums meet in LDS.
  template <int R, int K>
  __device__ static __forceinline__ void add_shares(const Tile& t, const PartitionArg<3>& out, const PagedPlan& p, __amdgpu_buffer_rsrc_t part, uint32_t bytes, unsigned char* lds) {
    constexpr int U = D / 4, kRowsAtOnce = kThreads / U;
    const int tid = threadIdx.x, u = tid % U;
    const uint32_t stats = bytes / (D + 4) * D;
    const int rows_at_once = min(kRowsAtOnce, t.rows <= 1 ? 1 : 1 << (32 - __builtin_clz(t.rows - 1))), groups = kRowsAtOnce / rows_at_once, group = tid / U / rows_at_once;
    const uint32_t each = (t.shares + groups - 1) / groups, k0 = group * each, k1 = min(k0 + each, t.shares);
#pragma unroll 1
    for (int base = 0; base < t.rows; base += rows_at_once * R) {
      const int row0 = base + tid / U % rows_at_once;
      Sum of[R];
#pragma unroll 1
      for (uint32_t k = k0; k < k1; k += K) {
        u32x4 v[R][K];
        u32x2 st[R][K];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (uint32_t i = 0; i < K; ++i) {
            const int row = row0 + r * rows_at_once;
            const bool there = k + i < k1 && row < t.rows;
            v[r][i] = __builtin_amdgcn_raw_buffer_load_b128(part, there ? (k + i) * bytes + (uint32_t)row * (D * 4) + u * 16 : kOob, 0, gemm::kAgentScope);
            st[r][i] = __builtin_amdgcn_raw_buffer_load_b64(part, there ? (k + i) * bytes + stats + row * 8 : kOob, 0, gemm::kAgentScope);
          }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (uint32_t i = 0; i < K; ++i) {
            const f32x2 both = __builtin_bit_cast(f32x2, st[r][i]);
            if (k + i < k1) of[r].add(__builtin_bit_cast(f32x4, v[r][i]), both[0], both[1]);
          }
      }
      if (R == 1 && groups > 1) {
        f32x4* const sums = reinterpret_cast<f32x4*>(lds);
        float* const stats_at = reinterpret_cast<float*>(lds + kThreads * 16);
        __syncthreads();
        sums[tid] = of[0].o;
        if (u == 0) stats_at[tid / U * 2] = of[0].m, stats_at[tid / U * 2 + 1] = of[0].l;
        __syncthreads();
        if (group != 0) continue;
        for (int g = 1; g < groups; ++g) {
          const int at = tid / U + g * rows_at_once;
          of[0].add(sums[at * U + u], stats_at[at * 2], stats_at[at * 2 + 1]);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row0 + r * rows_at_once < t.rows) store_row(out, t, p, row0 + r * rows_at_once, u, of[r].o, of[r].l);
    }
  }

  // FEW: tiles of up to so many rows, 16 or 32, are all there is (0: of any).
  template <int FEW>
  __device__ static __forceinline__ void run(const TensorArg<3>& q, const PartitionArg<3>& out, const PagedCache& c, const PagedPlan& p) {
    __shared__ __attribute__((aligned(1024))) unsigned char lds[kLdsBytes];
    __shared__ float stat[W][2][32];
    __shared__ uint32_t flag;
    __shared__ int32_t apart_at[2], all_missed[W * kMostMissed];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t heads = (uint32_t)c.heads, of_long = (uint32_t)p.long_tiles * p.long_shares;
    uint32_t head = blockIdx.x % heads, item = blockIdx.x / heads;
    if (FEW && MX && gridDim.x / heads % 8 == 0) {   // the heads of one part of a sequence on one XCD, one after another: their scales, and rows of D = 64, share lines
      const uint32_t slot = blockIdx.x / 8;
      head = slot % heads, item = slot / heads * 8 + blockIdx.x % 8;
    }
    // rows that have a wavefront's keys to themselves (of 256 values they take more registers on their way than 8 wavefronts have)
    constexpr int kMostOwn = FEW ? FEW : D == 256 ? 0 : 32;
    const bool is_long = !FEW && item < of_long;
    Tile t;
    t.head = (int32_t)head;
    int32_t b;
    uint32_t most, keys_each;
    paged::Sequence s;
    if (is_long) {
      // Tiles of sequence b have the numbers from starts[b] * group / tile_rows + b on: more than there are, so that nobody has to count them.  The last ones, whose rows see
      // the most keys, come first.
      const int32_t n = p.long_tiles - 1 - (int32_t)(item / p.long_shares);
      t.share = item % p.long_shares;
      auto number = [&](int32_t i) { return (int64_t)min(max(c.starts[i], 0), c.tokens) * p.group / p.tile_rows + i; };
      b = paged::find_sequence(c.batch, n, number);
      s = paged::sequence(c, b);
      const int64_t row0 = ((int64_t)n - number(b)) * p.tile_rows;
      if (s.count * p.group <= p.few_rows || row0 < 0 || row0 >= (int64_t)s.count * p.group) return;
      t.row0 = (int32_t)row0;
      t.rows = min(p.tile_rows, s.count * p.group - t.row0);
      most = p.long_shares, keys_each = p.long_keys;
      t.slot = (uint32_t)n * heads + head;
    } else {
      const uint32_t k = item - of_long;
      b = (int32_t)(k / p.few_shares);
      t.share = k % p.few_shares;
      s = paged::sequence(c, b);
      t.row0 = 0;
      t.rows = s.count * p.group;
      if (t.rows == 0 || t.rows > p.few_rows) return;   // (more than max_new allows: not promised)
      most = p.few_shares, keys_each = p.few_keys;
      t.slot = ((uint32_t)p.long_tiles + b) * heads + head;
    }
    t.first = s.first;
    t.pos0 = s.position(0);
    t.pages = c.table + (int64_t)b * c.table_row;
    const int32_t first = t.pos0 + t.row0 / p.group, last = t.pos0 + (t.row0 + t.rows - 1) / p.group;
    // (larger tiles start on a multiple of 64: whole groups of rows; rows whose window lies behind the table have no keys there, and no arithmetic next to 2^31)
    const int32_t seen = p.window > 0 && first >= p.window ? first - p.window + 1 : 0, hi = max(min(last + 1, s.held), 0), lo = min(t.rows > 16 ? seen & ~63 : seen, hi);
    // as many shares as it takes, as even as steps of all wavefronts allow
    const int32_t span = hi - lo, step = t.rows <= kMostOwn ? kOwners * 32 : 64, wanted = (int32_t)min(((uint32_t)span + keys_each - 1) / keys_each, most);
    const int32_t each = max((span + wanted - 1) / max(wanted, 1) + step - 1, step) / step * step;
    t.shares = max((span + each - 1) / each, 1);
    if (t.share >= t.shares) return;
    t.k0 = lo + (int32_t)t.share * each;
    t.k1 = min(hi, t.k0 + each);
    t.all_lo = p.window > 0 && last >= p.window ? last - p.window + 1 : 0, t.all_hi = min(first, t.k1 - 1);

    // Partial results: rows of the large tiles first, [head][row of all][share], then the others, [sequence][head][share].
    const int32_t slot_rows = is_long ? t.rows : p.few_slot_rows;
    constexpr uint64_t kRowBytes = (D + 4) * 4;
    const uint64_t all_rows = (uint64_t)c.tokens * p.group, of_shares = p.long_shares > 1 ? p.long_shares : 0;
    unsigned char* partials = (unsigned char*)p.partials + (is_long ? ((uint64_t)head * all_rows + (uint64_t)t.first * p.group + t.row0) * of_shares * kRowBytes
                                                                     : heads * all_rows * of_shares * kRowBytes + (uint64_t)(t.slot - (uint32_t)p.long_tiles * heads) * p.few_shares * slot_rows * kRowBytes);
    int32_t* const missed = all_missed + wave * kMostMissed;
    unsigned char *const sk = lds + wave % kOwners * kOwnBytes, *const sv = sk + 32 * kRowK;   // of 32 keys of the wavefront's own
    auto own = [&](auto rows) {
      Rows<decltype(rows)::value> w;
      begin(w, t, q, p, 0);
      own_keys(w, t, c, p.scale_log2e, sk, sv, missed);
      ordered();   // (a wavefront's results lie where its keys were)
      finish(w, t, out, p, partials, slot_rows, lds, stat, &flag, W);
    };
    if constexpr (FEW > 0) {
      own(std::integral_constant<int, FEW>{});
    } else if constexpr (kMostOwn > 0) {
      if (t.rows <= 16) return own(std::integral_constant<int, 16>{});
      if (t.rows <= kMostOwn) return own(std::integral_constant<int, kMostOwn>{});
    }
    if constexpr (!FEW) {
      constexpr int kMostShared = W * kRows / 64;
      const int shared_by = t.rows <= 64 ? kMostShared : t.rows <= BM / 2 ? 2 : 1;   // wavefronts to the keys of kRows rows
      int blocks = 1;
      Rows<kRows> w;
      begin(w, t, q, p, wave / shared_by);
      if (shared_by == 1) {
        blocks = kWideStep;
        bool done = false;
        if constexpr (D > 64)
          if ((done = GroupLoader<kWideStep * 32>::grouped(c, t))) pipelined_keys<kRows, kWideStep>(w, t, c, p.scale_log2e, lds, apart_at, missed);
        if (!done) shared_keys<kRows, W, kWideStep>(w, t, c, p.scale_log2e, lds, apart_at, missed);
      } else if (kMostShared > 2 && shared_by > 2) {
        shared_keys<kRows, W / kMostShared, 1>(w, t, c, p.scale_log2e, lds, apart_at, missed);
      } else {
        shared_keys<kRows, W / 2, kStep>(w, t, c, p.scale_log2e, lds, apart_at, missed);
        blocks = kStep;
      }
      __syncthreads();   // everybody is done with the stages
#pragma unroll 1
      for (int i = 0; i < W / kOwners; ++i) {
        if (wave / kOwners == i) add_missed(w, t, c, sv, missed, blocks);
        if (kOwners < W) __syncthreads();
      }
      finish(w, t, out, p, partials, slot_rows, lds, stat, &flag, shared_by);
    }
  }
};

}  // namespace

#define ATTENTION(NAME, T, MX, D)                                                                                                                                   \
  extern "C" __global__ void __launch_bounds__(512) paged_attention_entry__##NAME##_d##D(TensorArg<3> q, PartitionArg<3> out, PagedCache c, PagedPlan p) {  \
    Paged<T, MX, D, 8>::template run<0>(q, out, c, p);                                                                                                             \
  }
#define ATTENTION_FEW(NAME, T, MX, D, FEW, SUFFIX)                                                                                                                          \
  extern "C" __global__ void __launch_bounds__(256, D == 256 ? 1 : 2) paged_attention_entry__##NAME##_d##D##SUFFIX(TensorArg<3> q, PartitionArg<3> out, PagedCache c, PagedPlan p) { \
    Paged<T, MX, D, 4>::template run<FEW>(q, out, c, p);                                                                                                                   \
  }
#define ATTENTION_D(NAME, T, MX)                                                                                                                                    \
  ATTENTION(NAME, T, MX, 64) ATTENTION(NAME, T, MX, 128) ATTENTION(NAME, T, MX, 256)                                                                                \
  ATTENTION_FEW(NAME, T, MX, 64, 16, _few) ATTENTION_FEW(NAME, T, MX, 128, 16, _few) ATTENTION_FEW(NAME, T, MX, 256, 16, _few)                                      \
  ATTENTION_FEW(NAME, T, MX, 64, 32, _few32) ATTENTION_FEW(NAME, T, MX, 128, 32, _few32)
ATTENTION_D(f16, _Float16, false)
ATTENTION_D(bf16, __bf16, false)
ATTENTION_D(f16_mxfp8, _Float16, true)
ATTENTION_D(bf16_mxfp8, __bf16, true)
