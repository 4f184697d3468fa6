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
#include "split_k.h"

using namespace cutile;
using namespace cutile::gemm;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// Two stages of LDS, filled past the registers and refilled one K tile ahead.  Registers hold the x fragments of the K tile and two y fragments:
// a y fragment is reloaded as its last product issues, the x fragments with the next tile's during the last y block.  The
// hand-over of the stages sits one product before the last y block, where every read of the stage has had a block's products to complete; the
// refill of the stage just drained is dealt out over the products behind it.
// Scales: 16 bytes of a row serve two K tiles; they are fetched with the first of these into one of two buffers.
// (256 x 256: all 256 registers; 3 more, 5 with f32 out, are stored in front of the K loop and read back behind it.)
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

// 128 x 128 tiles that have a compute unit to themselves: eight wavefronts in two groups, each group on one half of every K tile, added up once at
// the end.  Wavefronts multiply 64 x 64 outputs: eight of 64 x 32 on all of K would read half as much again from LDS, whose bandwidth is what such a
// tile is short of (64 KiB read and 32 KiB written for 256 values of K, 512 clocks of products), and four alone on a compute unit would leave
// nobody to step in while one waits.
// A K tile is 256 values, 128 bytes of a row (fetched 64 bytes at a time, the L2 takes twice the requests: 1000 x 4096 x 14336 45.6 us).  A
// group's half is two products of v_mfma_scale_f32_32x32x64_f8f6f4 deep (a lane holds the 32 values of K block lane / 32 of row lane % 32 and
// supplies its scale).
// Four stages of LDS: tile kt + 3 goes into the stage of tile kt - 1 behind the one barrier of tile kt, where every wavefront has long
// multiplied with the last of it; what is waited for there is only its own share of tile kt + 1, requested two tiles ago.
// Registers hold the x fragments of the tile (the first ones are reloaded with the next tile's behind the barrier, the others at the start of their
// tile) and four y fragments, each reloaded as its last product issues.
// Scales: 32 bytes of a row serve four tiles, fetched with the first of these into one of two buffers; a lane reads its row's four of the
// tile and shifts its own to bytes 0 and 2.
// K may also be shared by several workgroups (split_k.h).
template <typename OutT>
struct Mxfp4Halves {
  static constexpr int BM = 128, BN = 128, kRow = 128, kWaves = 8, kThreads = 512, SLOTS = 4;
  static constexpr int WM = 64, WN = 64, TM = 2, TN = 2, BLOCKS = 2 * TN, NB = BLOCKS * TM;
  static constexpr int kAInstr = BM / 8 / kWaves, kFetch = (BM + BN) / 8 / kWaves;   // 1 KiB = 8 rows of 128 bytes
  static constexpr int kABytes = BM * kRow, kStageBytes = (BM + BN) * kRow, kScaleBytes = (BM + BN) * 32;   // scales: two tiles of all rows, then two more
  static constexpr int kHandOverAt = TM - 1, kBehind = NB - kHandOverAt;   // in front of the first read of the next tile
  static_assert(BLOCKS == SLOTS && (BM + BN) / 64 * 2 == kWaves, "a y fragment to each slot, 64 scale rows of two tiles to each wavefront");

  // Slot s of row r holds unit s ^ (r / 2 % 8).
  __device__ static __forceinline__ int lds_off(int r, int u) { return r * kRow + ((u ^ ((r >> 1) & 7)) << 4); }
  static constexpr int wait_vm(int n) { return (n & 15) | (7 << 4) | (15 << 8) | ((n >> 4) << 14); }   // vmcnt(n) alone

  __device__ static __forceinline__ void run(const PartitionArg<2>& z, const TensorArg<2>& x, const TensorArg<2>& y, const TensorArg<2>& xs, const TensorArg<2>& ys,
                                             float alpha, const TileGrid& g, float* partials, uint32_t* counters, uint32_t splits) {
    __shared__ __attribute__((aligned(4096))) unsigned char st0[kStageBytes];
    __shared__ __attribute__((aligned(4096))) unsigned char st1[kStageBytes];
    __shared__ __attribute__((aligned(4096))) unsigned char st2[kStageBytes];
    __shared__ __attribute__((aligned(4096))) unsigned char st3[kStageBytes];
    __shared__ __attribute__((aligned(1024))) unsigned char sc0[kScaleBytes];   // scales of tiles 0-3, 8-11 ...
    __shared__ __attribute__((aligned(1024))) unsigned char sc1[kScaleBytes];   // scales of tiles 4-7, 12-15 ...
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = wave >> 2;
    const int wm = (wave >> 1) & 1, wn = wave & 1, l32 = lane & 31, half = lane >> 5;
    // split-major order: an XCD's contiguous share is neighbouring tiles on one range of K
    const uint32_t tiles = g.x * g.y, pos = xcd_contiguous(blockIdx.x, tiles * splits), split = pos / tiles, tile = pos % tiles;
    uint32_t pm, pn;
    grouped_tile(tile, g.x, g.y, &pm, &pn);
    const int32_t row0 = (int32_t)pm * BM, col0 = (int32_t)pn * BN;
    const int32_t M = x.shape[0], N = y.shape[0], row_bytes = min(x.shape[1], y.shape[1]), all_tiles = (row_bytes + kRow - 1) / kRow;
    const int32_t first = (int32_t)((int64_t)all_tiles * split / splits), k_tiles = (int32_t)((int64_t)all_tiles * (split + 1) / splits) - first;
    // A last tile of 128 values is no work for the second group: behind it lie another row's scales, which may be NaN.  Zeros in their place, 2^-127 on
    // both sides, leave of whatever data lies there less than f32 holds.
    const int32_t none = group == 1 && row_bytes % kRow != 0 ? all_tiles - 1 - first : -1;
    auto rsrc = [](const TensorArg<2>& t) { return make_rsrc(t.ptr, (uint32_t)((int64_t)(t.shape[0] - 1) * t.strides[0] + t.shape[1])); };
    const __amdgpu_buffer_rsrc_t ra = rsrc(x), rb = rsrc(y), rsa = rsrc(xs), rsb = rsrc(ys);
    constexpr uint32_t kOob = 0x80000000u;   // operands end below 2 GiB

    // Global side of the fetches (per lane, K tile `first`; the K advance is scalar).  Rows outside read zeros.
    uint32_t goff[kFetch];
#pragma unroll
    for (int i = 0; i < kFetch; ++i) {
      const bool is_x = i < kAInstr;
      const int r = (wave * kAInstr + (is_x ? i : i - kAInstr)) * 8 + (lane >> 3), u = (lane & 7) ^ ((r >> 1) & 7);
      goff[i] = is_x ? (row0 + r < M ? (uint32_t)((int64_t)(row0 + r) * x.strides[0] + u * 16) : kOob)
                     : (col0 + r < N ? (uint32_t)((int64_t)(col0 + r) * y.strides[0] + u * 16) : kOob);
    }
    const int share = wave & 3, s_row = (share & 1) * 64 + lane;   // of the scale rows: x 0..63, x 64..127, y 0..63, y 64..127; two tiles to each group
    const uint32_t s_goff = share < 2 ? (row0 + s_row < M ? (uint32_t)((int64_t)(row0 + s_row) * xs.strides[0]) : kOob)
                                      : (col0 + s_row < N ? (uint32_t)((int64_t)(col0 + s_row) * ys.strides[0]) : kOob);
    auto fetch = [&](unsigned char* stage, unsigned char* sc, int32_t kt, int i) {
      if (i < kFetch) {
        const bool wanted = kt < k_tiles;   // past the last tile: out-of-range offsets, zeros, so that every tile counts the same requests
        const bool is_x = i < kAInstr;
        const int at = (is_x ? 0 : kABytes) + (wave * kAInstr + (is_x ? i : i - kAInstr)) * 1024;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(is_x ? ra : rb, (LDS_PTR(void))(stage + at), 16, wanted ? goff[i] : kOob, wanted ? (first + kt) * kRow : 0, 0, 0);
      } else {
        const bool wanted = kt + 2 * group < k_tiles;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(share < 2 ? rsa : rsb, (LDS_PTR(void))(sc + wave * 1024), 16, wanted ? s_goff : kOob,
                                                 wanted ? (first + kt + 2 * group) * 8 : 0, 0, 0);
      }
    };

    // LDS side: the lane's 16-byte unit of its row for each half of the tile, its row's scales.
    const int unit = 4 * group + half;
    const int a_addr[2] = {lds_off(wm * WM + l32, unit), lds_off(wm * WM + l32, unit + 2)};                       // + 32 rows a block
    const int b_addr[2] = {kABytes + lds_off(wn * WN + l32, unit), kABytes + lds_off(wn * WN + l32, unit + 2)};   // + 32 rows a block
    const int sa_addr = (wm * WM + l32) * 16 + 4 * group, sb_addr = (BM + wn * WN + l32) * 16 + 4 * group;        // + 32 rows a block, + the tile's place
    auto place = [](int ph) { return (ph >> 1) * (kScaleBytes / 2) + (ph & 1) * 8; };
    u32x4 af[2][TM], bf[SLOTS];
    uint32_t sa[2][TM], sb[2][TN];   // by tile parity
    auto read_a = [&](const unsigned char* stage, int ks, int tm) { af[ks][tm] = *reinterpret_cast<const u32x4*>(stage + a_addr[ks] + tm * 32 * kRow); };
    auto read_b = [&](const unsigned char* stage, int q) { bf[q] = *reinterpret_cast<const u32x4*>(stage + b_addr[q / TN] + q % TN * 32 * kRow); };
    auto scale = [&](const unsigned char* at) { return *reinterpret_cast<const uint32_t*>(at); };
    auto wide = [](u32x4 v) { return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w}; };

    f32x16 acc[TN][TM];
#pragma unroll
    for (int tn = 0; tn < TN; ++tn)
#pragma unroll
      for (int tm = 0; tm < TM; ++tm)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[tn][tm][v] = 0.0f;

    // The first three tiles on their way (scales with the first), the first fragments in registers.
#pragma unroll
    for (int i = 0; i < kFetch + 1; ++i) fetch(st0, sc0, 0, i);
#pragma unroll
    for (int i = 0; i < kFetch; ++i) fetch(st1, sc0, 1, i);
#pragma unroll
    for (int i = 0; i < kFetch; ++i) fetch(st2, sc0, 2, i);
    __builtin_amdgcn_s_waitcnt(wait_vm(2 * kFetch));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) sa[0][tm] = scale(sc0 + sa_addr + tm * 512), read_a(st0, 0, tm);
#pragma unroll
    for (int tn = 0; tn < TN; ++tn) sb[0][tn] = scale(sc0 + sb_addr + tn * 512);
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) read_b(st0, q);

    // Tile kt (phase = kt % 4) from `cur`; `nxt`: the stage of tile kt + 1, `prev`: of tile kt - 1, which tile kt + 3 goes into.  sc_nxt: scales of tile kt + 1,
    // sc_new: where those of tile kt + 3 go if it opens new ones.
    auto k_tile = [&](unsigned char* prev, const unsigned char* cur, const unsigned char* nxt, const unsigned char* sc_nxt, unsigned char* sc_new, int32_t kt, auto phase) {
      constexpr int PH = decltype(phase)::value, PHN = (PH + 1) & 3, P = PH & 1;
      constexpr int kRequests = kFetch + (PH == 1 ? 1 : 0), kFreeA = TN * TM;
      const uint32_t live = kt == none ? 0u : 0xffffffffu;
#pragma unroll
      for (int tm = 0; tm < TM; ++tm) sa[P][tm] = (sa[P][tm] & live) >> (8 * half);
#pragma unroll
      for (int q = 0; q < BLOCKS; ++q) {
        const int ks = q / TN, tn = q % TN;
        if (ks == 0) sb[P][tn] = (sb[P][tn] & live) >> (8 * half);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
          const int j = q * TM + tm;
          if (j == kHandOverAt) {
            // tile kt + 1 has landed: the one behind it, and the scales that came with it, may be outstanding
            __builtin_amdgcn_s_waitcnt(wait_vm(kFetch + (PH == 2 ? 1 : 0)));
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
          }
          acc[tn][tm] = ks == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(bf[q]), wide(af[ks][tm]), acc[tn][tm], 4, 4, 0, (int)sb[P][tn], 0, (int)sa[P][tm])
                                : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(bf[q]), wide(af[ks][tm]), acc[tn][tm], 4, 4, 2, (int)sb[P][tn], 2, (int)sa[P][tm]);
          __builtin_amdgcn_sched_barrier(0);   // a reload must follow the last reader, or it needs registers of its own
          if (j < TM) read_a(cur, 1, j);       // (the tile before is through with them)
          if (tm == TM - 1) {                  // y fragment q has done its last product
            if (ks == 0) sb[1 - P][tn] = scale(sc_nxt + sb_addr + tn * 512 + place(PHN));
            read_b(nxt, q);
          }
          if (j >= kFreeA && j < kFreeA + TM) {
            sa[1 - P][j - kFreeA] = scale(sc_nxt + sa_addr + (j - kFreeA) * 512 + place(PHN));
            read_a(nxt, 0, j - kFreeA);
          }
          if (j >= kHandOverAt) {
#pragma unroll
            for (int i = 0; i < kRequests; ++i)
              if (i * kBehind / kRequests == j - kHandOverAt) fetch(prev, sc_new, kt + 3, i);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    using P0 = std::integral_constant<int, 0>;
    using P1 = std::integral_constant<int, 1>;
    using P2 = std::integral_constant<int, 2>;
    using P3 = std::integral_constant<int, 3>;
    int32_t kt = 0;
    for (; kt + 8 <= k_tiles; kt += 8) {
      k_tile(st3, st0, st1, sc0, sc1, kt, P0{});
      k_tile(st0, st1, st2, sc0, sc1, kt + 1, P1{});
      k_tile(st1, st2, st3, sc0, sc1, kt + 2, P2{});
      k_tile(st2, st3, st0, sc1, sc1, kt + 3, P3{});
      k_tile(st3, st0, st1, sc1, sc0, kt + 4, P0{});
      k_tile(st0, st1, st2, sc1, sc0, kt + 5, P1{});
      k_tile(st1, st2, st3, sc1, sc0, kt + 6, P2{});
      k_tile(st2, st3, st0, sc0, sc0, kt + 7, P3{});
    }
    if (kt < k_tiles) k_tile(st3, st0, st1, sc0, sc1, kt, P0{});
    if (kt + 1 < k_tiles) k_tile(st0, st1, st2, sc0, sc1, kt + 1, P1{});
    if (kt + 2 < k_tiles) k_tile(st1, st2, st3, sc0, sc1, kt + 2, P2{});
    if (kt + 3 < k_tiles) k_tile(st2, st3, st0, sc1, sc1, kt + 3, P3{});
    if (kt + 4 < k_tiles) k_tile(st3, st0, st1, sc1, sc0, kt + 4, P0{});
    if (kt + 5 < k_tiles) k_tile(st0, st1, st2, sc1, sc0, kt + 5, P1{});
    if (kt + 6 < k_tiles) k_tile(st1, st2, st3, sc1, sc0, kt + 6, P2{});

    // Every wavefront is past its operand reads and every fetch has landed.  The groups exchange: each wavefront gives the 32 rows that its namesake
    // in the other group stores and adds those it gets.  Register by register, lane by lane: 16 bytes a lane, free of conflicts.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    f32x4 sum[TN][4];
    {
      unsigned char* const give = group == 0 ? st0 : st1;
      const unsigned char* const take = group == 0 ? st1 : st0;
#pragma unroll
      for (int tn = 0; tn < TN; ++tn)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const f32x16 &other = group == 0 ? acc[tn][1] : acc[tn][0], &own = group == 0 ? acc[tn][0] : acc[tn][1];
          *reinterpret_cast<f32x4*>(give + ((wave & 3) * 8 + tn * 4 + v) * 1024 + lane * 16) = f32x4{other[4 * v], other[4 * v + 1], other[4 * v + 2], other[4 * v + 3]};
          sum[tn][v] = f32x4{own[4 * v], own[4 * v + 1], own[4 * v + 2], own[4 * v + 3]};
        }
      __syncthreads();
#pragma unroll
      for (int tn = 0; tn < TN; ++tn)
#pragma unroll
        for (int v = 0; v < 4; ++v) sum[tn][v] += *reinterpret_cast<const f32x4*>(take + ((wave & 3) * 8 + tn * 4 + v) * 1024 + lane * 16);
    }
    if (splits > 1 && !combine_tile<4, TN, kThreads>(sum, partials + (size_t)tile * splits * (BM * BN), counters + tile, split, splits, reinterpret_cast<uint32_t*>(sc0))) return;
    f32x16 out[TN][1];
#pragma unroll
    for (int tn = 0; tn < TN; ++tn)
#pragma unroll
      for (int v = 0; v < 16; ++v) out[tn][0][v] = sum[tn][v / 4][v % 4] * alpha;
    static_assert(4 * kEpilogueBytesPerWave<WN> <= kStageBytes && 4 * 8 * 1024 <= kStageBytes, "the output bands of a group must fit a stage, and what a group gives too");
    store_tile_staged<1, TN, OutT>(out, (group == 0 ? st2 : st3) + (wave & 3) * kEpilogueBytesPerWave<WN>, (OutT*)z.ptr, z.strides[0], z.shape[0], z.shape[1],
                                   row0 + wm * WM + group * 32, col0 + wn * WN, lane, 0);
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
#define MXFP4_HALVES(NAME, OUT_T)                                                                                                    \
  extern "C" __global__ void __launch_bounds__(512)                                                                                  \
      linear_tile_mxfp4_entry__##NAME(PartitionArg<2> z, TensorArg<2> x, TensorArg<2> y, TensorArg<2> xs, TensorArg<2> ys, float alpha, \
                                      TileGrid g, float* partials, uint32_t* counters, uint32_t splits) {                            \
    Mxfp4Halves<OUT_T>::run(z, x, y, xs, ys, alpha, g, partials, counters, splits);                                                  \
  }
MXFP4_HALVES(bf16_128x128x256_e2x2_lone, __bf16)
MXFP4_HALVES(f32_128x128x256_e2x2_lone, float)
