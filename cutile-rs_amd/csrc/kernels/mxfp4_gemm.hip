// MXFP4 GEMM for gfx950:
//   z[M,N] = alpha * sum_k (x[i,k] * sx[i,k/32]) * (y[j,k] * sy[j,k/32])
// x [M,K/2] and y [N,K/2] are packed e2m1 pairs (low nibble first, both K-contiguous), sx [M,K/32] and sy [N,K/32] are e8m0 scale
// bytes (2^(b-127)), accumulation is f32.  K is a multiple of 128.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 on 4-bit operands (measured with random products): a lane (row l = lane % 16, group g = lane / 16) holds
// the 32 values of K block g of its row, 16 bytes, and supplies that block's scale in one byte of its scale register (op_sel names it).  Which
// of x's K blocks meets which of y's is free as long as both agree: here an instruction pair takes a K tile of 256 values, 128 bytes of a row,
// lane group g the bytes 32 g .. 32 g + 31, K blocks 2 g (first instruction, byte 0 of the scales) and 2 g + 1 (second, byte 1): data in
// two 16-byte units and both scales in one 16-bit LDS read.
// A loop of nothing but these instructions on random operands sustains 5700 to 6000 TFLOP/s, held by the power limit; the same loop on e4m3
// operands 3900 to 4100, with twice the bytes.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "gemm_common.h"
#include "kernel_args.h"

using namespace cutile;
using namespace cutile::gemm;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// Two stages of LDS, filled past the registers and refilled one K tile ahead.  Registers hold the x fragments of the K tile and two y fragments:
// a y fragment is reloaded as its last product issues, the x fragments with the next tile's during the last y block.  The
// hand-over of the stages sits one product before the last y block, where every read of the stage has had a block's products to complete; the
// refill of the stage just drained is dealt out over the products behind it.
// Scales: 16 bytes of a row serve two K tiles; they are fetched with the first of these into one of two buffers.
template <int BM, int BN, int WAVES_M, int WAVES_N, typename OutT>
struct Mxfp4Direct {
  static constexpr int kRow = 128;                                             // bytes of a row in a K tile of 256 values
  static constexpr int kWaves = WAVES_M * WAVES_N;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, TM = WM / 16, TN = WN / 16, NB = TM * TN;
  static constexpr int kAInstr = BM / 8 / kWaves, kBInstr = BN / 8 / kWaves;   // 1 KiB = 8 rows of 128 bytes
  static constexpr int kSInstr = (BM + BN) / 64 / kWaves;                      // 1 KiB = 64 rows x 16 scale bytes
  static constexpr int kABytes = BM * kRow, kBBytes = BN * kRow, kScaleBytes = (BM + BN) * 16;
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0 && (BM + BN) % (64 * kWaves) == 0 && BM % 64 == 0, "tile must split evenly");
  static_assert(TN % 2 == 0 && TN >= 4 && TM >= 2, "two y fragment slots: an even number of y blocks keeps a block in its slot from tile to tile");

  // Slot s of row r holds the 16-byte unit at position s ^ (r / 2 % 8), positions counted first units of all lane groups first: a 16-byte LDS read
  // takes lanes of two groups at a time, and only neighbouring positions keep their rows on distinct banks (units in their own order: half of
  // the LDS cycles were conflicts).
  __device__ static __forceinline__ int lds_off(int r, int position) { return r * kRow + ((position ^ ((r >> 1) & 7)) << 4); }
  __device__ static __forceinline__ int unit_at(int position) { return (position & 3) * 2 + (position >> 2); }

  __device__ static void run(const PartitionArg<2>& z, const TensorArg<2>& x, const TensorArg<2>& y, const TensorArg<2>& xs, const TensorArg<2>& ys, float alpha,
                             const TileGrid& g) {
    __shared__ __attribute__((aligned(4096))) unsigned char ys0[kBBytes];
    __shared__ __attribute__((aligned(4096))) unsigned char ys1[kBBytes];
    __shared__ __attribute__((aligned(1024))) unsigned char xs0[kABytes];
    __shared__ __attribute__((aligned(1024))) unsigned char xs1[kABytes];
    __shared__ __attribute__((aligned(1024))) unsigned char sc0[kScaleBytes];   // scales of K tiles 0, 1, 4, 5 ...
    __shared__ __attribute__((aligned(1024))) unsigned char sc1[kScaleBytes];   // scales of K tiles 2, 3, 6, 7 ...
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N, l16 = lane & 15, grp = lane >> 4;
    uint32_t pm, pn;
    tile_coords(g.x, g.y, &pm, &pn);
    const int32_t M = x.shape[0], N = y.shape[0], row_bytes = min(x.shape[1], y.shape[1]);
    const int32_t row0 = pm * BM, col0 = pn * BN;
    auto rsrc = [](const TensorArg<2>& t) { return make_rsrc(t.ptr, (uint32_t)((int64_t)(t.shape[0] - 1) * t.strides[0] + t.shape[1])); };
    const __amdgpu_buffer_rsrc_t ra = rsrc(x), rb = rsrc(y), rsa = rsrc(xs), rsb = rsrc(ys);
    constexpr uint32_t kOob = 0x80000000u;   // operands end below 2 GiB
    const int32_t k_tiles = (row_bytes + kRow - 1) / kRow;
    // A last K tile of 128 values: behind them lie the scales of another row, which may be NaN.  Zeros in their place, 2^-127 on both sides,
    // leave of whatever data lies there less than f32 holds.
    const int32_t half_tile = row_bytes % kRow != 0 && grp >= 2 ? k_tiles - 1 : -1;

    // Global side of the fetches (per lane, K tile 0; the K advance is scalar).  Rows outside read zeros.
    uint32_t a_goff[kAInstr], b_goff[kBInstr], s_goff[kSInstr];
#pragma unroll
    for (int i = 0; i < kAInstr; ++i) {
      const int r = (wave * kAInstr + i) * 8 + (lane >> 3), u = unit_at((lane & 7) ^ ((r >> 1) & 7));
      a_goff[i] = row0 + r < M ? (uint32_t)((int64_t)(row0 + r) * x.strides[0] + u * 16) : kOob;
    }
#pragma unroll
    for (int i = 0; i < kBInstr; ++i) {
      const int r = (wave * kBInstr + i) * 8 + (lane >> 3), u = unit_at((lane & 7) ^ ((r >> 1) & 7));
      b_goff[i] = col0 + r < N ? (uint32_t)((int64_t)(col0 + r) * y.strides[0] + u * 16) : kOob;
    }
#pragma unroll
    for (int i = 0; i < kSInstr; ++i) {
      const int sidx = wave * kSInstr + i;
      const bool is_x = sidx < BM / 64;
      const int r = (is_x ? sidx : sidx - BM / 64) * 64 + lane;
      s_goff[i] = is_x ? (row0 + r < M ? (uint32_t)((int64_t)(row0 + r) * xs.strides[0]) : kOob) : (col0 + r < N ? (uint32_t)((int64_t)(col0 + r) * ys.strides[0]) : kOob);
    }
    constexpr int NF = kAInstr + kBInstr;
    auto fetch_one = [&](unsigned char* xst, unsigned char* yst, unsigned char* sc, int32_t kt, int i) {
      const bool wanted = kt < k_tiles;   // past the last tile: out-of-range offsets, zeros
      const int32_t k0 = wanted ? kt * kRow : 0;
      if (i < kAInstr) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (LDS_PTR(void))(xst + (wave * kAInstr + i) * 1024), 16, wanted ? a_goff[i] : kOob, k0, 0, 0);
      } else if (i < NF) {
        const int b = i - kAInstr;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (LDS_PTR(void))(yst + (wave * kBInstr + b) * 1024), 16, wanted ? b_goff[b] : kOob, k0, 0, 0);
      } else {
        const int sidx = wave * kSInstr + i - NF;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(sidx < BM / 64 ? rsa : rsb, (LDS_PTR(void))(sc + sidx * 1024), 16, wanted ? s_goff[i - NF] : kOob, k0 / 16, 0, 0);
      }
    };
    // LDS side: the lane's two 16-byte units of its row and its two scale bytes.
    const int a_lo = lds_off(wm * WM + l16, grp), a_hi = lds_off(wm * WM + l16, 4 + grp);   // + tm * 16 rows
    const int b_lo = lds_off(wn * WN + l16, grp), b_hi = lds_off(wn * WN + l16, 4 + grp);   // + tn * 16 rows
    const int sa_addr = (wm * WM + l16) * 16 + 2 * grp;                                             // + tm * 16 rows, + 8 * (tile % 2)
    const int sb_addr = (BM + wn * WN + l16) * 16 + 2 * grp;                                        // + tn * 16 rows
    struct Frag {
      u32x4 lo, hi;
      int scale;
    };
    auto load = [&](Frag& f, const unsigned char* stage, int lo, int hi, const unsigned char* sc, int s_addr, int ph, int blk, bool far) {
      if (far) asm volatile("" : "+v"(lo), "+v"(hi));   // (x stages lie beyond the 16-bit offsets: no address register per fragment and stage)
      f.scale = *reinterpret_cast<const uint16_t*>(sc + s_addr + blk * 256 + 8 * ph);
      f.lo = *reinterpret_cast<const u32x4*>(stage + lo + blk * 16 * kRow);
      f.hi = *reinterpret_cast<const u32x4*>(stage + hi + blk * 16 * kRow);
    };
    auto wide = [](u32x4 v) { return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w}; };

    f32x4_acc acc[TN][TM];
#pragma unroll
    for (int tn = 0; tn < TN; ++tn)
#pragma unroll
      for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = f32x4_acc{0.0f, 0.0f, 0.0f, 0.0f};
    Frag af[TM], bf[2];

#pragma unroll
    for (int i = 0; i < NF + kSInstr; ++i) fetch_one(xs0, ys0, sc0, 0, i);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NF; ++i) fetch_one(xs1, ys1, sc0, 1, i);
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) load(af[tm], xs0, a_lo, a_hi, sc0, sa_addr, 0, tm, true);
#pragma unroll
    for (int tn = 0; tn < 2; ++tn) load(bf[tn], ys0, b_lo, b_hi, sc0, sb_addr, 0, tn, false);

    constexpr int kSteps = 2 * NB, kHandOverAt = (TN - 1) * 2 * TM - 1, kFetchSlots = kSteps - kHandOverAt;
    // Tile kt from `cur`; its scales are in sc_cur, the next tile's in sc_nxt.  An even tile fetches the scales of tiles kt + 2 and kt + 3 into sc_new.
    auto k_tile = [&](unsigned char* x_cur, unsigned char* y_cur, const unsigned char* x_nxt, const unsigned char* y_nxt, unsigned char* sc_cur, unsigned char* sc_nxt,
                      unsigned char* sc_new, int32_t kt, auto odd) {
      constexpr int PH = decltype(odd)::value;
      constexpr int NFT = NF + (PH == 0 ? kSInstr : 0);
      const int live = kt == half_tile ? 0 : 0xffff;
#pragma unroll
      for (int tn = 0; tn < TN; ++tn) {
        const Frag& b = bf[tn & 1];
        bf[tn & 1].scale &= live;
#pragma unroll
        for (int h = 0; h < 2; ++h) {   // both instructions of an output block TM products apart: they add to the same registers
#pragma unroll
          for (int tm = 0; tm < TM; ++tm) {
            const int j = (tn * 2 + h) * TM + tm;
            if (j == kHandOverAt) {
              __builtin_amdgcn_s_waitcnt(0);   // own reads of `cur` done, own share of tile kt + 1 landed
              __syncthreads();
              __builtin_amdgcn_sched_barrier(0);
            }
            if (j >= kHandOverAt) {
#pragma unroll
              for (int i = 0; i < NFT; ++i)
                if (i * kFetchSlots / NFT == j - kHandOverAt) fetch_one(x_cur, y_cur, sc_new, kt + 2, i);
            }
            if (j < TM) af[tm].scale &= live;
            const Frag& a = af[tm];
            acc[tn][tm] = h == 0 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(b.lo), wide(a.lo), acc[tn][tm], 4, 4, 0, b.scale, 0, a.scale)
                                 : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(b.hi), wide(a.hi), acc[tn][tm], 4, 4, 1, b.scale, 1, a.scale);
            __builtin_amdgcn_sched_barrier(0);   // a reload must follow the last reader, or it needs registers of its own
            if (h == 1 && tn == TN - 1) load(af[tm], x_nxt, a_lo, a_hi, sc_nxt, sa_addr, 1 - PH, tm, true);   // x block tm has done its last products of this tile
            if (h == 1 && tm == TM - 1) {                                                                       // so has y block tn: its slot takes y block tn + 2
              if (tn + 2 < TN) load(bf[tn & 1], y_cur, b_lo, b_hi, sc_cur, sb_addr, PH, tn + 2, false);
              else load(bf[tn & 1], y_nxt, b_lo, b_hi, sc_nxt, sb_addr, 1 - PH, tn + 2 - TN, false);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    };
    using Even = std::integral_constant<int, 0>;
    using Odd = std::integral_constant<int, 1>;
    int32_t kt = 0;
    for (; kt + 4 <= k_tiles; kt += 4) {
      k_tile(xs0, ys0, xs1, ys1, sc0, sc0, sc1, kt, Even{});
      k_tile(xs1, ys1, xs0, ys0, sc0, sc1, sc0, kt + 1, Odd{});
      k_tile(xs0, ys0, xs1, ys1, sc1, sc1, sc0, kt + 2, Even{});
      k_tile(xs1, ys1, xs0, ys0, sc1, sc0, sc0, kt + 3, Odd{});
    }
    if (kt < k_tiles) k_tile(xs0, ys0, xs1, ys1, sc0, sc0, sc1, kt, Even{});
    if (kt + 1 < k_tiles) k_tile(xs1, ys1, xs0, ys0, sc0, sc1, sc0, kt + 1, Odd{});
    if (kt + 2 < k_tiles) k_tile(xs0, ys0, xs1, ys1, sc1, sc1, sc0, kt + 2, Even{});

    // Every wavefront is past its operand reads and every fetch has landed: the stages are free to carry the output.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
#pragma unroll
    for (int tn = 0; tn < TN; ++tn)
#pragma unroll
      for (int tm = 0; tm < TM; ++tm) acc[tn][tm] *= alpha;
    static_assert(kWaves <= 8 && 2 * kEpilogueBytesPerWave<WN> <= kABytes && 2 * kEpilogueBytesPerWave<WN> <= kBBytes, "two output bands per stage array");
    unsigned char* band = (wave < 2 ? ys0 : wave < 4 ? ys1 : wave < 6 ? xs0 : xs1) + (wave & 1) * kEpilogueBytesPerWave<WN>;
    store_tile_staged16<TM, TN, OutT>(acc, band, (OutT*)z.ptr, z.strides[0], z.shape[0], z.shape[1], row0 + wm * WM, col0 + wn * WN, lane, 0);
  }
};

}  // namespace

#define MXFP4_KERNEL(NAME, BM, BN, WVM, WVN, OUT_T)                                                                                  \
  extern "C" __global__ void __launch_bounds__(WVM* WVN * 64)                                                                        \
      linear_tile_mxfp4_entry__##NAME(PartitionArg<2> z, TensorArg<2> x, TensorArg<2> y, TensorArg<2> xs, TensorArg<2> ys, float alpha, \
                                      TileGrid g) {                                                                                  \
    Mxfp4Direct<BM, BN, WVM, WVN, OUT_T>::run(z, x, y, xs, ys, alpha, g);                                                            \
  }
MXFP4_KERNEL(bf16_256x256x256_e4x2, 256, 256, 4, 2, __bf16)
MXFP4_KERNEL(f32_256x256x256_e4x2, 256, 256, 4, 2, float)
MXFP4_KERNEL(bf16_128x128x256_e2x2, 128, 128, 2, 2, __bf16)
MXFP4_KERNEL(f32_128x128x256_e2x2, 128, 128, 2, 2, float)
