// Matrix products of consecutive row groups (one expert each) for sm_100a, in
// bf16 and in fp8 with one scale per block of 128.
//
//   forward, dlhs:  out[t][r]    = sum_k B[t][k] A[g(t)][r][k]
//   drhs:           out[g][t][r] = sum_{k in group g} B[t][k] A[r][k]
//
// Which operand is on which side of the MMA. The dense index r -- a weight
// matrix's rows -- takes the 256 rows of a CTA pair's tile, and the index that
// may be short or ragged, t, takes the columns: an MMA's time scales with its
// columns, so a group with 40 rows costs 64 columns, not a 256-row tile, and a
// decode batch streams its weights at memory speed. Each tile issues MMAs only
// as wide as the rows it has (a multiple of 32).
//
// Persistent kernel, a CTA pair (cta_group::2) per two SMs, or, for fp8 tiles of
// at most 128 columns, single CTAs with 128 rows each; 12 or 20 warps a CTA:
//   warp 0      TMA producer, 128-byte k-slabs, 128-byte swizzle, no multicast
//   warp 1      MMA issuer (of a pair: in its even CTA)
//   warp 2      first the scan of the groups, then scales (fp8; MX: warp 3 too)
//   warp 3      of wide fp8 tiles, not MX: a look at the scales' range (narrow: warp 2)
//   warps 4-    epilogue: two or four per TMEM lane quarter, up to 64 columns each
// Warps 0 and 1 run whole, with one elected lane issuing. bf16 accumulates the
// whole contraction in TMEM (two 256-column accumulators: the epilogue of one tile
// runs under the next tile's MMAs). fp8 accumulates one 128-block there; the
// epilogue warps read it, multiply by the two scales and add it to f32 registers
// (up to 64 a thread) while the tensor core fills the other half of TMEM, which
// holds two or four blocks of a narrow tile. Wide fp8 tiles whose scales are powers
// of two (MX) are scaled by the tensor core (kind::mxf8f6f4, one 8-bit exponent for
// 32 elements, the same for the four MMAs of a block), so that they too accumulate
// the whole contraction in TMEM: warps 2 and 3 turn the f32 scales into exponents,
// warp 1 copies them to TMEM four blocks at a time.
//
// Group sizes stay on the device: every CTA scans them once (prefix sums in
// shared memory) and finds its tiles from that, so no call waits for the host.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <cstring>

#include "block_scales.cuh"
#include "groups.cuh"
#include "tcgen05.cuh"

namespace aqtb200 {

int sm_count();
int gemm_sms();

// Epilogue warps: SLICES for each TMEM lane quarter, COLS columns each; a tile is
// up to SLICES * COLS columns wide. Four more warps carry the other roles.
// Registers (setmaxnreg): the first warpgroup gives up what the epilogue takes.
//   2 slices: 384 threads start with 168: 128 *  88 + 256 * 208 = 64512
//   4 slices: 640 threads start with  96: 128 *  32 + 512 * 112 = 61440 (fp8)
//                                         128 *  64 + 512 * 104 = 61440 (bf16)
// k-slabs a stage of the ring holds: two where that leaves four slabs and more in
// flight, since each stage costs its producer and the MMA warp a wait
constexpr int gg_slabs(bool fp8, int tile) { return fp8 && tile > 128 ? 1 : 2; }
constexpr int gg_threads(int slices) { return 128 * (1 + slices); }
constexpr int GG_A_STAGE = 128 * 128;        // this CTA's 128 rows of A, 128 bytes of k
constexpr int GG_MAX_STAGES = 5;
// Whether fp8 tiles are a CTA pair's (cta_group::2) or one CTA's.
constexpr bool GG_PAIR_NARROW = false, GG_PAIR_WIDE = true;
constexpr int GG_RING = 192 * 1024;          // bytes of the operand ring
// Scales travel in batches of GG_BATCH slabs: one barrier round for four of them.
constexpr int GG_BATCH = 4;
constexpr int GG_SLOTS = 2;                  // batches on their way or in use
constexpr int GG_SLOT = 256 + 128;           // floats a slab: 256 columns, this CTA's 128 rows
constexpr int GG_SCALE_BYTES = GG_SLOTS * GG_BATCH * GG_SLOT * 4;
// Scales on the tensor core (MX): two batches of words in TMEM behind the columns
// of either accumulator. Of each, eight columns for 256 columns of the tile and
// four for 128 rows.
constexpr int GG_MX_COLS = 224;
constexpr int GG_MX_AHEAD = 3;               // batches of f32 scales on their way
constexpr int GG_MX_SLOTS = 4;               // batches of exponents
// of a slab: 256 columns and 128 rows, each with up to 3 floats more at both ends
// (whole 16-byte pieces), and how far the first one lies in its piece
constexpr int GG_MX_ROWS = 264, GG_MX_SHIFTS = GG_MX_ROWS + 136, GG_MX_SLOT = GG_MX_SHIFTS + 4;
constexpr int GG_STAGE_OUT = 512;            // a warp's staging: 8 columns by 32 rows of bf16,
constexpr int GG_STAGE_WIDE = 4096;          // or all of its 64 columns
constexpr int GG_RING_WIDE = 128 * 1024;
constexpr int GG_RING_MX = 180 * 1024;       // three stages of two slabs for 224 columns
constexpr size_t GG_SMEM = GG_RING + GG_SCALE_BYTES + 16 * GG_STAGE_OUT + 1024;
constexpr int GG_MX_BYTES = GG_MX_SLOTS * 3 * 512 + GG_MX_AHEAD * GG_BATCH * GG_MX_SLOT * 4;
constexpr size_t GG_SMEM_MX = GG_RING_MX + GG_MX_BYTES + 16 * GG_STAGE_OUT + 1024;
static_assert(GG_RING_WIDE + GG_SCALE_BYTES + 16 * GG_STAGE_WIDE + 1024 <= GG_SMEM, "shared memory");
constexpr int GG_MAX_SEG = AQTB200_MAX_GROUPS + 1;
constexpr int GG_TAIL = 64;                  // k-slab of bf16 elements

struct GGParams {
  int mode;  // 0: t is grouped; 1: the contraction is grouped
  int nt;    // columns of a full tile
  int stages, b_stage;
  // TMEM: two halves of 256 columns, handed over one at a time; each holds
  // `half_kb` accumulators `buf_cols` columns apart (fp8: of consecutive slabs)
  int half_kb, buf_cols;
  int one_half;        // MX: one accumulator, the scales in the other half
  int split;           // CTAs or pairs of a cluster that share one tile's contraction
  int a_mn, b_mn, bk;  // bk: elements of k per slab
  uint32_t idesc;      // without the column count
  int r, t, rows;
  int r_tiles, t_tiles, num_kb;
  const void* sizes;
  int sizes64, groups;  // groups 0: one group holds everything
  const float* a_scale;
  int64_t sa_g, sa_k, sa_r;
  const float* b_scale;
  int64_t sb_k;
  // the quantizer's notes on a's rows (row scales) or b's, one for 128 of them and a
  // slab, or none; note_padded: by 128 rows of each group
  const uint4* note;
  int64_t note_k, note_t;
  int note_padded;
  // fp8 operands as far_tile reads them
  const uint8_t *a, *b;
  int64_t a_ld, a_g, b_ld;
  int k, a_e5, b_e5;
  void* out;
  int out_f32;
  int out_staged;  // bf16 rows of whole 16-byte pieces
  int tma_out;     // and a map of them
  int64_t o_ld, o_g;
  int32_t* status;
};

// MN-major operand tile in the 128-byte swizzle: 64 elements of the kept index
// per 128-byte row, one row per k; 8-row groups 1024 bytes apart (stride byte
// offset), chunks of 64 kept elements `lbo` bytes apart.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr, uint32_t lbo) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(lbo >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// The four MMAs of one 128-byte slab, issued by the elected lane. The whole warp
// runs this, so that descriptors stay in uniform registers: issued from a
// one-lane branch each MMA took about 70 clocks of moves, and the issuing thread
// was what bounded every fp8 product.
#define GG_MMA4(KIND, GROUP)                                                                \
  asm volatile(                                                                             \
      "{\n\t.reg .pred q, p, t;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"                     \
      "setp.ne.b32 q, %8, 0;\n\tsetp.ne.b32 p, %7, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"            \
      "mov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"                                    \
      "@q tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], a, b, %9, p;\n\t"                   \
      "add.u32 x, %1, %5;\n\tadd.u32 y, %3, %6;\n\t"                                        \
      "mov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"                                      \
      "@q tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], a, b, %9, t;\n\t"                   \
      "add.u32 x, x, %5;\n\tadd.u32 y, y, %6;\n\t"                                          \
      "mov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"                                      \
      "@q tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], a, b, %9, t;\n\t"                   \
      "add.u32 x, x, %5;\n\tadd.u32 y, y, %6;\n\t"                                          \
      "mov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"                                      \
      "@q tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], a, b, %9, t;\n\t}" ::"r"(d_tmem),   \
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(a_step), "r"(b_step), "r"(accumulate), \
      "r"(elected), "r"(idesc)                                                              \
      : "memory")
template <bool FP8, bool PAIR>
__device__ __forceinline__ void gg_mma4(uint32_t elected, uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi,
                                        uint32_t b_lo, uint32_t b_hi, uint32_t a_step, uint32_t b_step,
                                        uint32_t idesc, uint32_t accumulate) {
  if constexpr (FP8 && PAIR) GG_MMA4("f8f6f4", "2");
  else if constexpr (FP8) GG_MMA4("f8f6f4", "1");
  else if constexpr (PAIR) GG_MMA4("f16", "2");
  else GG_MMA4("f16", "1");
}
#undef GG_MMA4


// The same with the tensor core's own block scales, one 8-bit exponent for 32
// elements: of the bytes of a column's word in TMEM, the one `idesc` names.
__device__ __forceinline__ void gg_mma4_scaled(uint32_t elected, uint32_t d_tmem, uint32_t a_lo,
                                               uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                               uint32_t idesc, uint32_t sa, uint32_t sb,
                                               uint32_t accumulate) {
#define GG_MMA_SCALED(ACC)                                                                      \
  "@q tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %7, [%8], [%9], " ACC \
  ";\n\t"
#define GG_MMA_STEP                                                                             \
  "add.u32 x, x, 2;\n\tadd.u32 y, y, 2;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
  asm volatile(
      "{\n\t.reg .pred q, p, t;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"
      "setp.ne.b32 q, %6, 0;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "mov.b32 x, %1;\n\tmov.b32 y, %3;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
      GG_MMA_SCALED("p") GG_MMA_STEP GG_MMA_SCALED("t") GG_MMA_STEP GG_MMA_SCALED("t")
      GG_MMA_STEP GG_MMA_SCALED("t") "}" ::"r"(d_tmem),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(accumulate), "r"(elected), "r"(idesc), "r"(sa),
      "r"(sb)
      : "memory");
#undef GG_MMA_STEP
#undef GG_MMA_SCALED
}
// Copies 32 pieces of 16 bytes, one after the other in shared memory, to four
// columns of TMEM, the same in every lane quarter, in both CTAs of the pair.
__device__ __forceinline__ void tc_copy_scales(uint32_t elected, uint32_t tmem, uint32_t at) {
  // no swizzle, groups of eight pieces 128 bytes apart
  const uint64_t desc = (uint64_t)((at & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 |
                        (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(tmem),
      "l"(desc), "r"(elected)
      : "memory");
}

// Notes that a bounded wait ran out. A plain store, since the words may lie in the
// host's memory; of several codes either may stay.
__device__ __forceinline__ void report(int32_t* status, int code) {
  if (status != nullptr) *(volatile int32_t*)status = code;
}

// Waits for what a kernel launched before this one wrote; returns at once unless
// this one was launched early.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Hands an accumulator back: only this warp's reads of it have to be over, which
// the fence before orders (see mbar_arrive_cluster).
template <bool PAIR>
__device__ __forceinline__ void gg_arrive(uint32_t bar) {
  if constexpr (PAIR) mbar_arrive_cluster(bar);
  else asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e;
}
// A wait of the whole warp with one answer for all of its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag) ? 1 : 0) != 0;
}

template <bool PAIR>
__device__ __forceinline__ void tma_load_3d(uint32_t elected, uint32_t dst, const CUtensorMap* tm,
                                            uint32_t bar, int c0, int c1, int c2) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];\n\t}" ::"r"(dst),
        "l"(tm), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(elected)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];\n\t}" ::"r"(dst),
        "l"(tm), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(elected)
        : "memory");
}
__device__ __forceinline__ void expect_tx_if(uint32_t elected, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes), "r"(elected)
      : "memory");
}
// Two f32 multiply-adds in one instruction: (a0, a1) += (x0, x1) * (y0, y1).
__device__ __forceinline__ void fma2(float& a0, float& a1, float x0, float x1, float y0, float y1) {
  asm("{\n\t.reg .b64 x, y, a;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 a, {%0, %1};\n\t"
      "fma.rn.f32x2 a, x, y, a;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(x0), "f"(x1), "f"(y0), "f"(y1));
}
// Arrives, at both CTAs of a pair, once every MMA issued so far has completed.
template <bool PAIR>
__device__ __forceinline__ void gg_commit(uint32_t elected, uint32_t bar, uint32_t lead) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;\n\t}" ::"r"(bar),
        "h"((uint16_t)(3u << lead)), "r"(elected)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
        "r"(elected)
        : "memory");
}

// 16 lanes by 32 columns of TMEM; of every 8 columns a thread gets columns
// 2 (lane % 4) and the next of lane / 4, then of lane / 4 + 8.
__device__ __forceinline__ void tc_ld_16x256(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
// Waits for the loads; what they brought passes through, so that no use of it can
// be moved ahead of the wait.
__device__ __forceinline__ void tc_wait_for(uint32_t (*v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0][0]), "+r"(v[0][1]), "+r"(v[0][2]), "+r"(v[0][3]), "+r"(v[0][4]), "+r"(v[0][5]),
                 "+r"(v[0][6]), "+r"(v[0][7]), "+r"(v[0][8]), "+r"(v[0][9]), "+r"(v[0][10]), "+r"(v[0][11]),
                 "+r"(v[0][12]), "+r"(v[0][13]), "+r"(v[0][14]), "+r"(v[0][15]), "+r"(v[1][0]), "+r"(v[1][1]),
                 "+r"(v[1][2]), "+r"(v[1][3]), "+r"(v[1][4]), "+r"(v[1][5]), "+r"(v[1][6]), "+r"(v[1][7]),
                 "+r"(v[1][8]), "+r"(v[1][9]), "+r"(v[1][10]), "+r"(v[1][11]), "+r"(v[1][12]), "+r"(v[1][13]),
                 "+r"(v[1][14]), "+r"(v[1][15])
               :
               : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Where the groups lie: one entry per group and, when t is grouped, one more for
// the rows behind the last group (whose output is zero).
struct Segments {
  int32_t off[GG_MAX_SEG + 1];   // first row; [n] = end
  int32_t tile[GG_MAX_SEG + 1];  // mode 0: tiles before it. mode 1, fp8: 128-blocks before it
};

struct TileAt {
  int seg;
  int r0, t0;  // first row and column of the tile
  int tvalid;  // columns that exist
  int n;       // columns of the MMAs
  int k0;      // mode 1: first contraction position of the group
  int klen;    // mode 1: positions in the group
  int nkb;     // slabs of k
};

template <bool FP8, bool PAIR>
__device__ __forceinline__ TileAt gg_tile(const GGParams& P, const Segments& S, int nseg, int tile,
                                          int& cur) {
  TileAt T;
  int local;
  int tt;  // column tiles of this segment
  if (P.mode == 0) {
    while (cur + 1 < nseg && tile >= S.tile[cur + 1]) ++cur;
    local = tile - S.tile[cur];
    tt = (S.off[cur + 1] - S.off[cur] + P.nt - 1) / P.nt;
  } else {
    const int per = P.r_tiles * P.t_tiles;
    cur = tile / per;
    local = tile - cur * per;
    tt = P.t_tiles;
  }
  // bands of up to eight column tiles, walked row tile by row tile, keep the
  // operands of the tiles in flight in L2
  constexpr int G = 8;
  const int band = local / (G * P.r_tiles), in = local - band * (G * P.r_tiles);
  const int gt = min(G, tt - band * G);
  const int ri = in / gt, ti = band * G + (in - ri * gt);
  T.seg = cur;
  T.r0 = ri * (PAIR ? 256 : 128);
  T.k0 = 0;
  T.klen = 0;
  if (P.mode == 0) {
    T.t0 = S.off[cur] + ti * P.nt;
    T.tvalid = min(P.nt, S.off[cur + 1] - T.t0);
    T.nkb = (P.groups > 0 && cur == P.groups) ? 0 : P.num_kb;
  } else {
    T.t0 = ti * P.nt;
    T.tvalid = min(P.nt, P.t - T.t0);
    T.klen = S.off[cur + 1] - S.off[cur];
    T.nkb = (T.klen + P.bk - 1) / P.bk;
    T.k0 = FP8 ? S.tile[cur] * 128 : S.off[cur];
  }
  T.n = (T.tvalid + 31) & ~31;
  return T;
}

// First slab of share `part` of a tile's contraction.
__device__ __forceinline__ int share_of(int nkb, int part, int split) {
  return (int)((int64_t)nkb * part / split);
}

// A block's sum times its two scales, where a factor or a product on the way leaves
// f32's range and the result does not. |sum| is zero or between 2^-32 and 2^39 (128
// products of e5m2 values), so the epilogue's one multiplication ahead of its add is
// right with
//   weights' blocks  the two scales' product as the factor, where that is normal
//   row scales       the sum times the row's scale, where that lies in ROW_MIN .. ROW_MAX
// Elements with a block of other scales are computed again, by far_tile, when all is
// stored. (Nothing of this is in the epilogue's loop or between its tiles: choosing
// slab by slab cost 2 to 5 %, and a decision on each tile 1 to 2 %.) 8192 x 4096 x 14336
// with operands of 2^-60 and 2^-62, all of it: 82 ms in place of 0.6; cotangents of
// 2^-95, where it only looks: 5.0 ms backward in place of 1.3.
constexpr float GG_ROW_MIN = 0x1p-94f, GG_ROW_MAX = 0x1p89f;
template <bool A_ROW>
__device__ __forceinline__ bool is_far(float ra, float s) {
  if (!finite_nonzero(ra)) return false;
  if constexpr (A_ROW) return fabsf(ra) < GG_ROW_MIN || fabsf(ra) > GG_ROW_MAX;
  const float p = fabsf(s * ra);
  return finite_nonzero(s) && (p < SCALE_MIN_NORMAL || p > SCALE_MAX_FLOAT);
}
// acc + sum * ra * s. Part of a far factor goes to the sum first; a far row scale is
// brought 2^40 nearer to 1 for both products and sent back in the add.
template <bool A_ROW>
__device__ __forceinline__ float far_add(float acc, float sum, float ra, float s) {
  const bool far = is_far<A_ROW>(ra, s);
  if constexpr (A_ROW) {
    if (!far) return fmaf(sum * ra, s, acc);
    const bool small = fabsf(ra) < GG_ROW_MIN;
    return fmaf(sum * (ra * (small ? 0x1p40f : 0x1p-40f)) * s, small ? 0x1p-40f : 0x1p40f, acc);
  }
  if (!far) return fmaf(sum, s * ra, acc);
  if (fabsf(s * ra) < 1.f) return fmaf(sum * 0x1p-90f, (s * 0x1p45f) * (ra * 0x1p45f), acc);
  return fmaf(sum * 0x1p120f, (s * 0x1p-60f) * (ra * 0x1p-60f), acc);
}
// A look at the range of slabs kb0 .. kb1 of a CTA's tile, rows from row0 on: whether a
// pair of scales may be far, by the quantizer's notes and, weights' blocks, their own
// scales. In two steps, so that the reads of the first 32 slabs are on their way
// meanwhile (but for those of a block of 128 between the first and the last that the
// tile touches).
template <bool A_ROW>
struct FarLook {
  const float* a;   // scales of the weights' blocks
  const uint4* m0;  // notes on the first and the last block of 128
  const uint4* m1;
  int blocks;
  float a_first;
  uint4 m0_first, m1_first;

  __device__ __forceinline__ void begin(const GGParams& P, const Segments& S, const TileAt& T, int kb0, int kb1,
                                        int row0, int lane) {
    row0 = min(row0, P.r - 1);
    a = P.a_scale + (P.mode == 0 ? (int64_t)T.seg * P.sa_g : 0) + (int64_t)(T.k0 >> 7) * P.sa_k +
        (int64_t)(row0 >> 7) * P.sa_r;
    int first = row0 >> 7, last = first;
    if constexpr (!A_ROW) {
      int t = T.t0, before = 0;
      if (P.note_padded) {
        t -= S.off[T.seg];
        for (int g = lane; g < T.seg; g += 32) before += (S.off[g + 1] - S.off[g] + 127) >> 7;
        before = __reduce_add_sync(0xffffffffu, before);
      }
      first = before + (t >> 7);
      last = before + ((t + T.tvalid - 1) >> 7);
    }
    m0 = P.note + (int64_t)(T.k0 >> 7) * P.note_k + first * P.note_t;
    m1 = m0 + (last - first) * P.note_t;
    blocks = last - first + 1;
    a_first = 0.f;
    m0_first = m1_first = make_uint4(0, 0, 0, 0);
    const int kb = kb0 + lane;
    if (kb < kb1) {
      if constexpr (!A_ROW) a_first = a[kb * P.sa_k];
      if (P.note != nullptr) {
        m0_first = m0[kb * P.note_k];
        if constexpr (!A_ROW) m1_first = m1[kb * P.note_k];
      }
    }
  }
  static __device__ __forceinline__ bool may_be_far(float a, uint32_t note) {
    const float least = note_least(note), most = note_most(note);
    if constexpr (A_ROW) return (least > 0.f && least < GG_ROW_MIN) || most > GG_ROW_MAX;
    return finite_nonzero(a) && most > 0.f &&
           (least * fabsf(a) < SCALE_MIN_NORMAL || most * fabsf(a) > SCALE_MAX_FLOAT);
  }
  __device__ __forceinline__ bool finish(const GGParams& P, int kb0, int kb1, int lane) const {
    const bool noted = P.note != nullptr;
    bool may = kb0 + lane < kb1 &&
               may_be_far(a_first, noted ? __vmaxu4(join_notes(m0_first), join_notes(m1_first)) : NOTE_ORDINARY);
    for (int kb = kb0 + 32 + lane; kb < kb1; kb += 32) {
      float s = 0.f;
      uint32_t note = NOTE_ORDINARY;
      if constexpr (!A_ROW) s = a[kb * P.sa_k];
      if (noted) {
        note = join_notes(m0[kb * P.note_k]);
        if constexpr (!A_ROW) note = __vmaxu4(note, join_notes(m1[kb * P.note_k]));
      }
      may |= may_be_far(s, note);
    }
    if constexpr (!A_ROW)
      if (noted)
        for (int x = 1; x < blocks - 1; ++x)
          for (int kb = kb0 + lane; kb < kb1; kb += 32)
            may |= may_be_far(a[kb * P.sa_k], join_notes(m0[kb * P.note_k + x * P.note_t]));
    return __any_sync(0xffffffffu, may);
  }
};

// Sixteen fp8 values, zeros from the `left`-th on.
__device__ __forceinline__ uint4 fp8_piece(const uint8_t* p, int left) {
  if (left <= 0) return make_uint4(0, 0, 0, 0);
  uint4 v = *(const uint4*)p;
  if (left < 16) {
    uint32_t* w = (uint32_t*)&v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = left - 4 * i;
      w[i] = n <= 0 ? 0u : n < 4 ? w[i] & ((1u << (8 * n)) - 1u) : w[i];
    }
  }
  return v;
}
// Two of them as f16, which holds both formats exactly.
__device__ __forceinline__ uint32_t fp8_pair(uint32_t v, int e5) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)v, e5 ? __NV_E5M2 : __NV_E4M3);
  return (uint32_t)h.x | (uint32_t)h.y << 16;
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Writes the elements of a warp's part of a tile -- 32 rows from r0 on, `n` columns from
// c0 on -- that a far block may have spoilt, from the operands in global memory. Other
// elements keep their value, so that no result depends on its neighbours. A call of its
// own, off the epilogue's registers.
//
// A far block has spoilt nothing where the stored value is finite (what overflows on the
// way stays infinite or NaN) and large beside all that may have been lost below the
// normal numbers, for each block at most 2^-150, half the smallest of them, times the
// column's scale (row scales) or the sum of at most 2^39 (a product of scales): less
// than 2^-24 of the value. So it is with small cotangents beside ordinary activations.
//
// Eight columns at a time, each 128-block's sum by the warp's own MMAs on f16 copies of
// the values. A thread's sixteen bytes of a row serve four MMAs: the order of the
// positions is the same in both operands, and no other than any other.
template <bool A_ROW, bool PAIR>
__device__ __noinline__ void far_tile(const GGParams& P, const Segments& S, int nseg, int tile, int r0, int c0,
                                      int n, int lane) {
  int cur = 0;
  const TileAt T = gg_tile<true, PAIR>(P, S, nseg, tile, cur);
  const int row0 = T.r0 + r0, rows = min(32, P.r - row0), col0 = T.t0 + c0, cols = min(n, T.tvalid - c0);
  if (rows <= 0) return;
  const int64_t g = P.mode == 0 ? T.seg : 0, at = T.k0 / 128;
  const int lr = lane >> 2, lq = lane & 3;
  const float* sa = P.a_scale + g * P.sa_g + at * P.sa_k;
  const float* sb = P.b_scale + at * P.sb_k + col0;
  // this thread's elements: rows lr + 8 h, columns first + 2 lq + x
  const auto a_scale = [&](int kb, int h) {
    const int row = row0 + min(lr + 8 * h, rows - 1);
    return sa[kb * P.sa_k + (int64_t)(A_ROW ? row : row >> 7) * P.sa_r];
  };
  const auto place = [&](int h, int c) {
    return (P.mode == 1 ? (int64_t)T.seg * P.o_g : 0) + (int64_t)(col0 + c) * P.o_ld + row0 + lr + 8 * h;
  };
  for (int first = 0; first < cols; first += 8) {
    const int c[2] = {first + 2 * lq, first + 2 * lq + 1};
    uint32_t far = 0;  // bit 2 h + x
    float most[2] = {0.f, 0.f};
#pragma unroll 2
    for (int kb = 0; kb < T.nkb; ++kb) {
      float s[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s[x] = sb[kb * P.sb_k + min(c[x], cols - 1)];
        most[x] = fmaxf(most[x], fabsf(s[x]));
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float ra = a_scale(kb, h);
#pragma unroll
        for (int x = 0; x < 2; ++x) far |= (uint32_t)is_far<A_ROW>(ra, s[x]) << (2 * h + x);
      }
    }
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t bit = 1u << (2 * h + x);
        if (lr + 8 * h >= rows || c[x] >= cols) far &= ~bit;
        if (!(far & bit)) continue;
        const int64_t o = place(h, c[x]);
        const float have =
            fabsf(P.out_f32 ? ((const float*)P.out)[o] : __bfloat162float(((const __nv_bfloat16*)P.out)[o]));
        if (have <= SCALE_MAX_FLOAT && have >= (float)T.nkb * (A_ROW ? 0x1p-126f * most[x] : 0x1p-87f))
          far &= ~bit;
      }
    if (!__any_sync(0xffffffffu, far != 0)) continue;
    float total[4][2] = {};
#pragma unroll 1
    for (int kb = 0; kb < T.nkb; ++kb) {
      const int begin = T.k0 + kb * 128, end = min(begin + 128, P.k);
      float sum[2][4] = {};
#pragma unroll 1
      for (int k = begin + 16 * lq; k < begin + 128; k += 64) {
        uint4 va[4];
#pragma unroll
        for (int h = 0; h < 4; ++h)
          va[h] = fp8_piece(P.a + g * P.a_g + (int64_t)(row0 + lr + 8 * h) * P.a_ld + k,
                            lr + 8 * h < rows ? end - k : 0);
        const uint4 vb = fp8_piece(P.b + (int64_t)(col0 + first + lr) * P.b_ld + k, first + lr < cols ? end - k : 0);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t a[4][2];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const uint32_t v = ((const uint32_t*)&va[h])[w];
            a[h][0] = fp8_pair(v & 0xffffu, P.a_e5);
            a[h][1] = fp8_pair(v >> 16, P.a_e5);
          }
          const uint32_t v = ((const uint32_t*)&vb)[w];
          const uint32_t b0 = fp8_pair(v & 0xffffu, P.b_e5), b1 = fp8_pair(v >> 16, P.b_e5);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            mma_f16(sum[i], a[2 * i][0], a[2 * i + 1][0], a[2 * i][1], a[2 * i + 1][1], b0, b1);
        }
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float ra = a_scale(kb, h);
#pragma unroll
        for (int x = 0; x < 2; ++x)
          total[h][x] = far_add<A_ROW>(total[h][x], sum[h >> 1][2 * (h & 1) + x], ra,
                                       sb[kb * P.sb_k + min(c[x], cols - 1)]);
      }
    }
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (far >> (2 * h + x) & 1u) {
          const int64_t o = place(h, c[x]);
          if (P.out_f32) ((float*)P.out)[o] = total[h][x];
          else ((__nv_bfloat16*)P.out)[o] = __float2bfloat16_rn(total[h][x]);
        }
  }
}

template <bool FP8, bool A_ROW, bool PAIR, int SLICES, int COLS, bool MX = false>
__global__ void __launch_bounds__(gg_threads(SLICES), 1)
grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmAt, const __grid_constant__ CUtensorMap tmBt,
                    const __grid_constant__ GGParams P) {
  static_assert(!MX || (FP8 && PAIR && SLICES * COLS > 128), "scales on the tensor core: wide fp8 tiles");
  constexpr bool SUMS = FP8 && !MX;  // the epilogue scales and adds every 128-block
  constexpr int KS = MX ? 2 : gg_slabs(FP8, SLICES * COLS);
  constexpr int SLOTS = MX ? GG_MX_SLOTS : GG_SLOTS;
  constexpr bool SHARES = SLICES * COLS <= 128;  // a contraction may be shared (P.split)
  // Wide fp8 tiles keep every warp busy with the sums, so their results leave
  // through the TMA unit: written to shared memory (4 KB a warp) and stored from
  // there under the next tile. Stored by the warps themselves they cost 65 us of
  // the 626 us of an 8192 x 4096 x 14336 forward product.
  constexpr bool TMA_OUT = SUMS && SLICES * COLS > 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full_bar[GG_MAX_STAGES];   // used in the pair's even CTA
  __shared__ __align__(8) uint64_t empty_bar[GG_MAX_STAGES];  // one per CTA
  __shared__ __align__(8) uint64_t tfull_bar[2];              // one per CTA
  __shared__ __align__(8) uint64_t tempty_bar[2];             // used in the pair's even CTA
  __shared__ __align__(8) uint64_t sfull_bar[SLOTS];       // a batch of scales; one per CTA
  __shared__ __align__(8) uint64_t sempty_bar[SLOTS];
  __shared__ __align__(8) uint64_t raw_bar[MX ? 2 * GG_MX_AHEAD : 1];  // MX: f32 scales, by warp
  __shared__ int far_flag;  // some tile has far scales
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int nseg_s;
  __shared__ int total_s;
  __shared__ Segments S;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  constexpr int CTAS = PAIR ? 2 : 1;       // that share a tile
  const uint32_t rank = PAIR ? crank & 1u : 0u;   // within the pair
  const uint32_t lead = PAIR ? crank & ~1u : crank;  // the pair's even CTA
  const int part = (int)(crank / CTAS);
  const bool leader = rank == 0;
  const int cluster_id = blockIdx.x / (CTAS * P.split);
  const int num_clusters = gridDim.x / (CTAS * P.split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < P.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&tfull_bar[s], 1);
      mbar_init(&tempty_bar[s], CTAS * 4 * SLICES);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&sfull_bar[s], MX ? 2 * CTAS : 32);
      mbar_init(&sempty_bar[s], MX ? 1 : 4 * SLICES);
    }
    if constexpr (MX)
      for (int s = 0; s < 2 * GG_MX_AHEAD; ++s) mbar_init(&raw_bar[s], 1);
    far_flag = 0;
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                       smem_u32(&tmem_slot))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                       smem_u32(&tmem_slot))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  if (warp == 2) {
    // prefix sums of the groups
    const int64_t limit = P.rows;  // sums in 64 bits, results within 32
    if (P.groups == 0) {
      if (lane == 0) {
        S.off[0] = 0;
        S.off[1] = P.rows;
        S.tile[0] = 0;
        nseg_s = 1;
        total_s = (P.mode == 0 ? (P.rows + P.nt - 1) / P.nt : P.t_tiles) * P.r_tiles;
        S.tile[1] = P.mode == 0 ? total_s : 0;
      }
    } else {
      int64_t off = 0, acc = 0;
      const int64_t unit = P.mode == 0 ? P.nt : 128;
      const int64_t per = P.mode == 0 ? P.r_tiles : 1;
      for (int g0 = 0; g0 < P.groups; g0 += 32) {
        const int g = g0 + lane;
        const int64_t n = g < P.groups ? min(group_size_at(P.sizes, P.sizes64, g), limit) : 0;
        const int64_t end = min(off + warp_scan(n, lane), limit);
        int64_t begin = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) begin = off;
        const int64_t tiles = (end - begin + unit - 1) / unit * per;
        const int64_t tend = acc + warp_scan(tiles, lane);
        if (g < P.groups) {
          S.off[g] = (int32_t)begin;
          S.tile[g] = (int32_t)(tend - tiles);
        }
        off = __shfl_sync(0xffffffffu, end, 31);
        acc = __shfl_sync(0xffffffffu, tend, 31);
      }
      if (lane == 0) {
        S.off[P.groups] = (int32_t)off;
        S.tile[P.groups] = (int32_t)acc;
        nseg_s = P.groups;
        if (P.mode == 0) {
          const int64_t rest = (limit - off + P.nt - 1) / P.nt * P.r_tiles;
          S.off[P.groups + 1] = P.rows;
          S.tile[P.groups + 1] = (int32_t)(acc + rest);
          nseg_s = P.groups + 1;
          total_s = (int)(acc + rest);
        } else {
          total_s = P.groups * P.r_tiles * P.t_tiles;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  // the barriers of every CTA of the cluster exist before anyone signals them
  if (PAIR || P.split > 1) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  const int nseg = nseg_s;
  const int total = total_s;
  volatile int* abortp = &abort_flag;
  // A role whose wait ran out: every CTA of the cluster stops waiting, and no part of
  // a shared contraction is added up (all signals come before the barrier ahead of
  // the sum).
  auto give_up = [&](int code) {
    if (lane != 0) return;
    const uint32_t flag = smem_u32(&abort_flag);
    for (int c = 0; c < CTAS * P.split; ++c) st_cluster_u32(map_to_cta(flag, c), 1u);
    report(P.status, code);
  };
  const int slab_bytes = GG_A_STAGE + P.b_stage, stage_bytes = KS * slab_bytes;
  float* const slots = (float*)(smem + P.stages * stage_bytes);
  int fail = 0;

  if (warp < 4) {
    if constexpr (SLICES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    else if constexpr (SUMS) asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == 0) {
    // ---------------- TMA producer (both CTAs, whole warp) ----------------
    {
      int stage = 0, cur = 0;
      uint32_t phase = 0;
      const uint32_t elected = elect_one();
      const uint32_t expecting = leader ? elected : 0u;
      const bool a_mn = !FP8 && P.a_mn, b_mn = !FP8 && P.b_mn;
      const int b_boxes = b_mn ? (P.nt / CTAS + 63) / 64 : 1;
      const uint32_t full0 = smem_u32(&full_bar[0]), lbar0 = PAIR ? map_to_cta(full0, lead) : full0;
      const uint32_t ring = smem_u32(smem);
      // The weights of the first stages are asked for while the quantizer of the
      // other operand may still run (see `follows_quantize`); what reads its results
      // waits for it, in every CTA, so that this grid ends after it. In a graph it took
      // 1.5 us off the 13.7 of 1 x 4096 x 4096 with its quantizer, 1.8 off the 47.8 of
      // 16 x 8192 x 28672, 4.3 off the 42.4 of 257 rows of 64 experts 2048 x 1408.
      int ahead = 0;
      if constexpr (FP8) {
        if (P.mode == 0 && cluster_id < total) {
          const TileAt T = gg_tile<FP8, PAIR>(P, S, nseg, cluster_id, cur);
          const int nkb = __shfl_sync(0xffffffffu, T.nkb, 0);
          const int kb0 = share_of(nkb, part, P.split), kb1 = share_of(nkb, part + 1, P.split);
          const int ra = __shfl_sync(0xffffffffu, T.r0, 0) + (int)rank * 128;
          const int ga = __shfl_sync(0xffffffffu, T.seg, 0);
          for (int ks = kb0; ks < kb1 && ahead < P.stages; ks += KS, ++ahead) {
            const int ke = min(ks + KS, kb1);
            expect_tx_if(expecting, full0 + ahead * 8, CTAS * (ke - ks) * slab_bytes);
            for (int kb = ks; kb < ke; ++kb)
              tma_load_3d<PAIR>(elected, ring + ahead * stage_bytes + (kb - ks) * slab_bytes, &tmA,
                                lbar0 + ahead * 8, kb * P.bk, ra, ga);
          }
          cur = 0;
        }
        grid_wait();
      }
      for (int tile = cluster_id; tile < total && !fail; tile += num_clusters) {
        const TileAt T = gg_tile<FP8, PAIR>(P, S, nseg, tile, cur);
        const int nkb = __shfl_sync(0xffffffffu, T.nkb, 0);
        const int kb0 = share_of(nkb, part, P.split), kb1 = share_of(nkb, part + 1, P.split);
        const int ra = __shfl_sync(0xffffffffu, T.r0, 0) + (int)rank * 128;
        const int tb = __shfl_sync(0xffffffffu, T.t0 + (int)rank * (T.n / CTAS), 0);
        const int seg = __shfl_sync(0xffffffffu, T.seg, 0);
        const int k0 = __shfl_sync(0xffffffffu, T.k0, 0);
        const int ga = P.mode == 0 ? seg : 0;
        // the slab a group of the contraction ends in, if it ends inside one
        int tail = -1;
        if (!FP8 && P.mode == 1 && P.groups > 0) {
          const int klen = __shfl_sync(0xffffffffu, T.klen, 0);
          if (klen % GG_TAIL) tail = klen / GG_TAIL;
        }
        for (int ks = kb0; ks < kb1; ks += KS) {
          const uint32_t lbar = lbar0 + stage * 8;
          const int ke = min(ks + KS, kb1);
          const bool asked = FP8 && ahead > 0;  // for the weights
          if (asked) {
            --ahead;
          } else {
            if (!warp_wait(&empty_bar[stage], phase ^ 1, abortp)) { fail = 1; break; }
            expect_tx_if(expecting, full0 + stage * 8, CTAS * (ke - ks) * slab_bytes);
          }
          uint32_t sa = ring + stage * stage_bytes;
          for (int kb = ks; kb < ke; ++kb, sa += slab_bytes) {
            const uint32_t sb = sa + GG_A_STAGE;
            const bool last = kb == tail;  // read the copy filled up with zeros
            const CUtensorMap* ma = last ? &tmAt : &tmA;
            const CUtensorMap* mb = last ? &tmBt : &tmB;
            const int kk = last ? 0 : k0 + kb * P.bk, za = last ? seg : ga, zb = last ? seg : 0;
            if (asked) {
            } else if (a_mn) {
              tma_load_3d<PAIR>(elected, sa, ma, lbar, ra, kk, za);
              tma_load_3d<PAIR>(elected, sa + 8192, ma, lbar, ra + 64, kk, za);
            } else {
              tma_load_3d<PAIR>(elected, sa, ma, lbar, kk, ra, za);
            }
            if (b_mn) {
              tma_load_3d<PAIR>(elected, sb, mb, lbar, tb, kk, zb);
              for (int j = 1; j < b_boxes; ++j)
                tma_load_3d<PAIR>(elected, sb + j * 8192, mb, lbar, tb + j * 64, kk, zb);
            } else {
              tma_load_3d<PAIR>(elected, sb, mb, lbar, kk, tb, zb);
            }
          }
          if (++stage == P.stages) { stage = 0; phase ^= 1; }
        }
      }
      if (fail) give_up(1);
    }
    __syncwarp();
    if (P.split > 1) cluster_sync_all();
  } else if (warp == 1) {
    // ---------------- MMA issuer (of a pair: the even CTA; whole warp) ----------------
    if (leader) {
      int stage = 0, cur = 0;
      uint32_t phase = 0;
      uint32_t half = 0, hphase = 0;
      const uint32_t elected = elect_one();
      const bool a_mn = !FP8 && P.a_mn, b_mn = !FP8 && P.b_mn;
      const uint32_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;
      const uint64_t a_desc = a_mn ? smem_desc_mn(0, 8192) : make_smem_desc(0);
      const uint64_t b_desc = b_mn ? smem_desc_mn(0, 8192) : make_smem_desc(0);
      const uint32_t a_hi = (uint32_t)(a_desc >> 32), b_hi = (uint32_t)(b_desc >> 32);
      // offset within this CTA: the address carries the CTA's rank above bit 18
      const uint32_t ring = (smem_u32(smem) & 0x3FFFFu) >> 4;
      const uint32_t a_lo0 = (uint32_t)a_desc + ring, b_lo0 = (uint32_t)b_desc + ring + (GG_A_STAGE >> 4);
      const uint32_t empty0 = smem_u32(&empty_bar[0]);
      const uint32_t tfull0 = smem_u32(&tfull_bar[0]);
      const uint32_t sempty0 = smem_u32(&sempty_bar[0]), slots0 = smem_u32(slots);
      int slot = 0;  // batch of scales (MX)
      uint32_t sphase = 0;
      for (int tile = cluster_id; tile < total && !fail; tile += num_clusters) {
        const TileAt T = gg_tile<FP8, PAIR>(P, S, nseg, tile, cur);
        const int nkb = __shfl_sync(0xffffffffu, T.nkb, 0);
        const int kb0 = share_of(nkb, part, P.split), kb1 = share_of(nkb, part + 1, P.split);
        const uint32_t idesc = P.idesc | ((uint32_t)(__shfl_sync(0xffffffffu, T.n, 0) >> 3) << 17);
        int in_half = 0;  // accumulators of the current half already filled
        for (int ks = kb0; ks < kb1; ks += KS) {
          if (!warp_wait(&full_bar[stage], phase, abortp)) { fail = 2; break; }
          const int ke = min(ks + KS, kb1);
          uint32_t slab = (uint32_t)(stage * stage_bytes) >> 4;
          for (int kb = ks; kb < ke; ++kb, slab += (uint32_t)slab_bytes >> 4) {
            if (SUMS ? in_half == 0 : kb == kb0) {
              if (!warp_wait(&tempty_bar[half], hphase ^ 1u, abortp)) { fail = 2; break; }
            }
            const bool last = kb + 1 == kb1;
            if constexpr (MX) {
              const int j = (kb - kb0) & (GG_BATCH - 1);
              const uint32_t ts = tmem_base + (P.one_half ? 256u + slot * 16u
                                                      : GG_MX_COLS + (slot & 1) * 16u + (slot >> 1) * 256u);
              if (j == 0) {
                if (!warp_wait(&sfull_bar[slot], sphase, abortp)) { fail = 2; break; }
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 3; ++c)
                  tc_copy_scales(elected, ts + c * 4, slots0 + (slot * 3 + c) * 512);
              }
              tc_fence_after();
              gg_mma4_scaled(elected, tmem_base + half * 256u, a_lo0 + slab, a_hi, b_lo0 + slab, b_hi,
                             idesc | (uint32_t)j << 29 | (uint32_t)j << 4, ts + 8, ts, kb > kb0 ? 1u : 0u);
              if (j == GG_BATCH - 1 || last) {
                gg_commit<PAIR>(elected, sempty0 + slot * 8, lead);
                if (++slot == SLOTS) { slot = 0; sphase ^= 1u; }
              }
            } else {
              tc_fence_after();
              gg_mma4<FP8, PAIR>(elected, tmem_base + half * 256u + (FP8 ? in_half * P.buf_cols : 0),
                                 a_lo0 + slab, a_hi, b_lo0 + slab, b_hi, a_step, b_step, idesc,
                                 (!FP8 && kb > kb0) ? 1u : 0u);
            }
            if (SUMS ? (++in_half == P.half_kb || last) : last) {
              gg_commit<PAIR>(elected, tfull0 + half * 8, lead);
              in_half = 0;
              half = MX && P.one_half ? 0u : half ^ 1u;
              if (half == 0) hphase ^= 1u;
            }
          }
          if (fail) break;
          gg_commit<PAIR>(elected, empty0 + stage * 8, lead);
          if (++stage == P.stages) { stage = 0; phase ^= 1; }
        }
      }
      if (fail) give_up(2);
    }
    __syncwarp();
    if (P.split > 1) cluster_sync_all();
  } else {
    // ---------------- scales, ahead of the epilogue (one warp) ----------------
    // A load issued by the epilogue warps a slab ahead put a memory round trip on
    // every 128-block (0.7 us a slab on the 8192 x 28672 decode, 90 us in all).
    if constexpr (FP8) grid_wait();
    if constexpr (MX) {
      // Warp 2: of the columns; warp 3: of this CTA's rows. GG_MX_AHEAD batches are
      // on their way at once, across tiles, as bulk copies: loaded and waited for
      // one by one a batch took up to 8000 clocks, in 4-byte asynchronous copies
      // 2100, and its MMAs take 1800. Four batches of exponents may be ready ahead
      // (with two 8192 x 8192 x 8192 took 495 us, with none to convert 460).
      const bool rows = warp == 3, square = rows && !A_ROW;
      int slot = 0, cur = 0, issued = 0, done = 0;
      uint32_t phase = 0;
      const uint32_t sfull0 = map_to_cta(smem_u32(&sfull_bar[0]), lead);
      uint64_t* const bars = raw_bar + (rows ? GG_MX_AHEAD : 0);
      float* const raw = slots + GG_MX_SLOTS * 384 + (rows ? GG_MX_ROWS : 0);
      int* const shifts = (int*)(slots + GG_MX_SLOTS * 384 + GG_MX_SHIFTS + (rows ? 1 : 0));
      auto convert = [&]() {
        const int at = (done % GG_MX_AHEAD) * GG_BATCH * GG_MX_SLOT;
        if (!warp_wait(&bars[done % GG_MX_AHEAD], (done / GG_MX_AHEAD) & 1, abortp)) return false;
        uint32_t w[8] = {0};
        const float* x[GG_BATCH];
#pragma unroll
        for (int b = 0; b < GG_BATCH; ++b)
          x[b] = raw + at + b * GG_MX_SLOT + (shifts[at + b * GG_MX_SLOT] & 3) + (square ? 0 : lane);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (e < (A_ROW ? 4 : 1) || !rows) {
            // the exponents are the top bytes once the signs are shifted out
            uint32_t v[GG_BATCH];
#pragma unroll
            for (int b = 0; b < GG_BATCH; ++b) v[b] = __float_as_uint(x[b][e * 32]) << 1;
            w[e] = __byte_perm(__byte_perm(v[0], v[1], 0x0073), __byte_perm(v[2], v[3], 0x0073), 0x5410);
          }
        }
        if (square) w[1] = w[2] = w[3] = w[0];
        ++done;
        if (!warp_wait(&sempty_bar[slot], phase ^ 1u, abortp)) return false;
        uint4* out = (uint4*)slots + slot * 96 + lane + (rows ? 64 : 0);
        out[0] = make_uint4(w[0], w[1], w[2], w[3]);
        if (!rows) out[32] = make_uint4(w[4], w[5], w[6], w[7]);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0)
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(sfull0 + slot * 8)
                       : "memory");
        if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
        return true;
      };
      for (int tile = cluster_id; tile < total && !fail; tile += num_clusters) {
        const TileAt T = gg_tile<FP8, PAIR>(P, S, nseg, tile, cur);
        const int row = min(T.r0 + (int)rank * 128, P.r - 1);
        const int have = !rows ? T.tvalid : A_ROW ? min(128, P.r - row) : 1;
        const int64_t step_k = rows ? P.sa_k : P.sb_k;
        const float* p = !rows ? P.b_scale + T.t0
                               : P.a_scale + (P.mode == 0 ? (int64_t)T.seg * P.sa_g : 0) +
                                     (int64_t)(A_ROW ? row : row >> 7) * P.sa_r;
        p += (T.k0 / 128 + lane) * step_k;  // a lane each for the slabs of a batch
        for (int kb = 0; kb < T.nkb; kb += GG_BATCH, p += GG_BATCH * step_k) {
          uint64_t* const bar = &bars[issued % GG_MX_AHEAD];
          const int at = ((issued % GG_MX_AHEAD) * GG_BATCH + lane) * GG_MX_SLOT;
          // whole 16-byte pieces around the scales
          const uintptr_t first = (uintptr_t)p & ~(uintptr_t)15;
          const bool mine = lane < min(GG_BATCH, T.nkb - kb);
          const uint32_t bytes = mine ? (uint32_t)((((uintptr_t)(p + have) + 15) & ~(uintptr_t)15) - first) : 0u;
          const uint32_t all = __reduce_add_sync(0xffffffffu, bytes);
          if (lane == 0) mbar_expect_tx(bar, all);
          if (mine) shifts[at] = (int)((uintptr_t)p - first) >> 2;
          __syncwarp();
          if (mine) bulk_load(raw + at, (const void*)first, bytes, bar);
          if (++issued - done == GG_MX_AHEAD && !convert()) { fail = 4; break; }
          __syncwarp();
        }
      }
      while (done < issued && !fail)
        if (!convert()) fail = 4;
      if (fail) give_up(4);
    }
    // The range of a tile's scales is looked at beside the products; nothing but the
    // kernel's end waits for it. Wide tiles: by warp 3 (by warp 2 a prompt of 2047 x 4096
    // x 14336 took 2 % longer). Narrow ones: by warp 2, around the copies of the tile's
    // scales: one token of 4096 x 4096 takes 12.5 us with its quantizer, 12.0 without the
    // look, 13.1 with warp 3 doing it, for the instructions it fetches beside the first
    // tile's. Read from the slots, or scale by scale, it took longer than the products.
    auto tell = [&]() {  // the CTA that stores the tile
      if (lane == 0) st_cluster_u32(map_to_cta(smem_u32(&far_flag), P.split > 1 ? rank : crank), 1u);
    };
    bool arrived = false;  // at the barrier ahead of the sum of a shared contraction
    if (SUMS && warp == 2) {
      int slot = 0, cur = 0;
      uint32_t phase = 0;
      bool far = false;
      for (int tile = cluster_id; tile < total && !fail; tile += num_clusters) {
        const TileAt T = gg_tile<FP8, PAIR>(P, S, nseg, tile, cur);
        const int kb0 = share_of(T.nkb, part, P.split), kb1 = share_of(T.nkb, part + 1, P.split);
        const int64_t kabs = T.k0 / 128 + kb0;
        const int row = min(T.r0 + (int)rank * 128, P.r - 1);
        const float* pa = P.a_scale + (P.mode == 0 ? (int64_t)T.seg * P.sa_g : 0) + kabs * P.sa_k +
                          (int64_t)(A_ROW ? row : row >> 7) * P.sa_r;
        const float* pb = P.b_scale + kabs * P.sb_k + T.t0;
        const int rows = A_ROW ? min(128, P.r - row) : 1;
        FarLook<A_ROW> look;
        if (SHARES) look.begin(P, S, T, kb0, kb1, T.r0 + (int)rank * 128, lane);
        for (int kb = kb0; kb < kb1; kb += GG_BATCH) {
          const int ok = mbar_wait(&sempty_bar[slot], phase ^ 1, abortp) ? 1 : 0;
          if (!__all_sync(0xffffffffu, ok)) { fail = 4; break; }
          const int m = min(GG_BATCH, kb1 - kb);
          for (int b = 0; b < m; ++b) {
            const uint32_t dst = smem_u32(slots + (slot * GG_BATCH + b) * GG_SLOT);
            for (int c = lane; c < T.tvalid; c += 32)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + c * 4), "l"(pb + c)
                           : "memory");
            for (int c = lane; c < rows; c += 32)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + (256 + c) * 4),
                           "l"(pa + c * P.sa_r)
                           : "memory");
            pa += P.sa_k;
            pb += P.sb_k;
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(
                           smem_u32(&sfull_bar[slot]))
                       : "memory");
          if (++slot == SLOTS) { slot = 0; phase ^= 1; }
        }
        if (fail) break;
        if (SHARES && P.split > 1) {
          cluster_arrive();
          arrived = true;
        }
        if (SHARES && !far) far = look.finish(P, kb0, kb1, lane);
      }
      if (far) tell();
      if (fail) give_up(4);
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    if (SUMS && !SHARES && warp == 3) {
      bool far = false;
      int cur = 0;
      for (int tile = cluster_id; tile < total && !far; tile += num_clusters) {
        const TileAt T = gg_tile<FP8, PAIR>(P, S, nseg, tile, cur);
        FarLook<A_ROW> look;
        look.begin(P, S, T, 0, T.nkb, T.r0 + (int)rank * 128, lane);
        far = look.finish(P, 0, T.nkb, lane);
      }
      if (far) tell();
    }
    __syncwarp();
    if (P.split > 1) {
      if (!arrived) cluster_arrive();
      cluster_wait();
    }
  }
  } else {
    // ---------------- epilogue (every CTA, its own 128 rows) ----------------
    if constexpr (SLICES == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    else if constexpr (SUMS) asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // rows behind the last group are zeros that wait for no operand: nothing is stored
    // before what was put on the stream last has ended, be it torch filling the result
    if constexpr (FP8) grid_wait();
    // A warp reads its 32 rows by COLS columns with 16x256b loads: a thread then
    // holds, of every 8 columns, two neighbouring ones in four rows,
    //   acc[g][h][i]: column 8 g + 2 (lane % 4) + i % 2, row 16 h + lane / 4 + 8 (i / 2),
    // so a column's scale serves four of its elements. (With one row a thread
    // every element needs a factor of its own from shared memory, and those
    // reads, 512 bytes to a warp each, took longer than the MMAs.)
    constexpr int GROUPS = COLS / 8;
    constexpr int HALF_KB = SLICES > 2 ? 1 : 128 / COLS;  // = P.half_kb
    const int quarter = warp & 3;
    const int c0 = ((warp - 4) >> 2) * COLS;  // first column of this warp
    uint32_t half = 0, hphase = 0;
    int slot = 0, cur = 0;
    uint32_t sphase = 0;
    bool have = false;
    float acc[GROUPS][2][4];
    const uint32_t tlane = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c0;
    const uint32_t tempty0 = PAIR ? map_to_cta(smem_u32(&tempty_bar[0]), lead) : smem_u32(&tempty_bar[0]);
    uint8_t* const stage_out =
        (uint8_t*)slots + (MX ? GG_MX_BYTES : GG_SCALE_BYTES) + (warp - 4) * (TMA_OUT ? GG_STAGE_WIDE : GG_STAGE_OUT);
    // The place in the output is worked out anew (`again` hides that from the
    // compiler): kept across the contraction it would cost registers there.
    auto store = [&](int again) {
      asm volatile("" : "+r"(again));
      const TileAt T = gg_tile<FP8, PAIR>(P, S, nseg, again, cur);
      const int r0 = T.r0 + (int)rank * 128 + quarter * 32;
      const int m = T.tvalid - c0;
      const int64_t at = (P.mode == 1 ? (int64_t)T.seg * P.o_g : 0) + (int64_t)(T.t0 + c0) * P.o_ld + r0;
      if (P.out_staged) {
        // bf16, aligned rows: eight columns at a time are turned round by a
        // transposing matrix store and leave as 64-byte pieces of output rows
        const uint32_t st = smem_u32(stage_out);
        // 16-byte piece `lane / 8` of row `lane % 8`, XOR-ed so that pieces of
        // neighbouring rows lie in different banks
        const uint32_t put = st + (lane & 7) * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) << 4);
        const int col = lane >> 2, piece = lane & 3;
        const uint8_t* get = stage_out + col * 64 + ((piece ^ ((col >> 1) & 3)) << 4);
        const int left = P.r - r0 - piece * 8;
        if (TMA_OUT && P.tma_out && m >= COLS) {
          // all of this warp's columns are the group's: one box of them
          if (lane == 0) tma_store_wait_read();  // of the tile before
          __syncwarp();
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const __nv_bfloat162 v =
                  __floats2bfloat162_rn(acc[g][q >> 1][(q & 1) * 2], acc[g][q >> 1][(q & 1) * 2 + 1]);
              w[q] = *(const uint32_t*)&v;
            }
            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                             put + g * 512),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && r0 < P.r) {
            asm volatile(
                "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                    &tmAt),
                "r"(st), "r"(r0), "r"(T.t0 + c0), "r"(P.mode == 1 ? T.seg : 0)
                : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          return;
        }
        if (TMA_OUT) {
          if (lane == 0) tma_store_wait_read();
          __syncwarp();
        }
        __nv_bfloat16* o = (__nv_bfloat16*)P.out + at + (int64_t)col * P.o_ld + piece * 8;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          if (g * 8 >= m) break;
          uint32_t w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {  // rows 8 q .. 8 q + 7
            const __nv_bfloat162 v =
                __floats2bfloat162_rn(acc[g][q >> 1][(q & 1) * 2], acc[g][q >> 1][(q & 1) * 2 + 1]);
            w[q] = *(const uint32_t*)&v;
          }
          asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(put),
                       "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                       : "memory");
          __syncwarp();
          const uint4 v = *(const uint4*)get;
          __syncwarp();
          if (g * 8 + col < m && left > 0) {
            if (left >= 8) {
              *(uint4*)o = v;
            } else {
              const uint16_t* e = (const uint16_t*)&v;
#pragma unroll
              for (int q = 0; q < 8; ++q)
                if (q < left) ((uint16_t*)o)[q] = e[q];
            }
          }
          o += 8 * P.o_ld;
        }
      } else {
        const int r = lane >> 2, c = (lane & 3) * 2;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int rr = 16 * h + r + 8 * (i >> 1), cc = 8 * g + c + (i & 1);
              if (cc < m && r0 + rr < P.r) {
                const int64_t x = at + (int64_t)cc * P.o_ld + rr;
                if (P.out_f32) ((float*)P.out)[x] = acc[g][h][i];
                else ((__nv_bfloat16*)P.out)[x] = __float2bfloat16_rn(acc[g][h][i]);
              }
            }
          }
        }
      }
    };
    for (int tile = cluster_id; tile < total; tile += num_clusters) {
      const TileAt T = gg_tile<FP8, PAIR>(P, S, nseg, tile, cur);
      have = true;
      const int kb0 = share_of(T.nkb, part, P.split), kb1 = share_of(T.nkb, part + 1, P.split);
      const int cols = T.n - c0;  // this warp's columns that the MMAs write
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[g][i >> 2][i & 3] = 0.f;
      int in_batch = 0;  // slabs of the current batch of scales already used
      for (int kb = kb0; kb < kb1;) {
        if (SUMS && in_batch == 0) {
          const int got = mbar_wait(&sfull_bar[slot], sphase, abortp) ? 1 : 0;
          if (!__all_sync(0xffffffffu, got)) { fail = 3; break; }
        }
        float2 f[GROUPS];  // this thread's two column scales of every 8 columns
        float ra[4];       // its four row scales, or the one of the whole block
        const float* sc = slots + (slot * GG_BATCH + in_batch) * GG_SLOT;
        auto factors = [&]() {
          if constexpr (A_ROW) {
#pragma unroll
            for (int q = 0; q < 4; ++q) ra[q] = sc[256 + quarter * 32 + (lane >> 2) + 8 * q];
          } else {
            ra[0] = sc[256];
          }
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            f[g] = *(const float2*)(sc + c0 + g * 8 + (lane & 3) * 2);
            if constexpr (!A_ROW) {
              f[g].x *= ra[0];
              f[g].y *= ra[0];
            }
          }
        };
        if (SUMS && HALF_KB == 1) factors();  // while the MMAs still run
        int ok = mbar_wait(&tfull_bar[half], hphase, abortp) ? 1 : 0;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) { fail = 3; break; }
        tc_fence_after();
        auto hand_back = [&]() {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) gg_arrive<PAIR>(tempty0 + half * 8);
        };
        const int here = SUMS && HALF_KB > 1 ? min(HALF_KB, kb1 - kb) : 1;  // accumulators in this half
        if (cols > 0) {
          uint32_t ta = tlane + half * 256u;
          for (int b = 0; b < here; ++b, ta += P.buf_cols, sc += GG_SLOT) {
            if (SUMS && HALF_KB > 1) factors();
#pragma unroll
            for (int c = 0; c < COLS; c += 32) {
              if (c >= cols) break;  // the same for the whole warp
              uint32_t p[2][16];
              tc_ld_16x256(ta + c, p[0]);
              tc_ld_16x256(ta + c + (16u << 16), p[1]);
              tc_wait_for(p);
#pragma unroll
              for (int g = 0; g < 4; ++g) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                  for (int i = 0; i < 4; i += 2) {
                    float* a = &acc[c / 8 + g][h][i];
                    float x = __uint_as_float(p[h][g * 4 + i]);
                    float y = __uint_as_float(p[h][g * 4 + i + 1]);
                    if constexpr (!SUMS) {
                      a[0] = x;
                      a[1] = y;
                    } else {
                      if constexpr (A_ROW) {
                        x *= ra[h * 2 + (i >> 1)];
                        y *= ra[h * 2 + (i >> 1)];
                      }
                      fma2(a[0], a[1], x, y, f[c / 8 + g].x, f[c / 8 + g].y);
                    }
                  }
                }
              }
            }
          }
        }
        hand_back();
        half = MX && P.one_half ? 0u : half ^ 1u;
        if (half == 0) hphase ^= 1u;
        if constexpr (SUMS) {
          kb += here;
          in_batch += here;
          if (in_batch == GG_BATCH || kb == kb1) {
            if (lane == 0) mbar_arrive(&sempty_bar[slot]);
            if (++slot == SLOTS) { slot = 0; sphase ^= 1u; }
            in_batch = 0;
          }
        } else {
          kb = kb1;
        }
      }
      if (fail) break;
      if (!SHARES || P.split == 1) store(tile);
    }
    if (fail) give_up(3);
    if (SHARES && P.split > 1) {
      // Parts of one tile: parts 1.. leave their sums in their own shared memory
      // (the operand ring is idle by now), part 0 adds them in part order.
      float4* mine = (float4*)smem + (warp - 4) * (GROUPS * 2 * 32) + lane;
      const bool busy = have && !fail && c0 < P.nt;
      if (busy && part > 0) {
#pragma unroll
        for (int g = 0; g < GROUPS * 2; ++g) {
          const float* a = acc[g >> 1][g & 1];
          mine[g * 32] = make_float4(a[0], a[1], a[2], a[3]);
        }
      }
      __syncwarp();
      cluster_sync_all();
      if (busy && part == 0 && !*abortp) {
        for (int p = 1; p < P.split; ++p) {
          const uint32_t from = map_to_cta(smem_u32(mine), CTAS * p + rank);
          float4 v[GROUPS * 2];
#pragma unroll
          for (int g = 0; g < GROUPS * 2; ++g) v[g] = ld_cluster_f32x4(from + g * 512);
#pragma unroll
          for (int g = 0; g < GROUPS * 2; ++g) {
            float* a = acc[g >> 1][g & 1];
            a[0] += v[g].x;
            a[1] += v[g].y;
            a[2] += v[g].z;
            a[3] += v[g].w;
          }
        }
        store(cluster_id);
      }
    }
    if (TMA_OUT && lane == 0) tma_store_wait_read();  // shared memory outlives its last store
  }

  __syncwarp();
  if (*abortp) {
    // copies still in flight land in shared memory that is still ours
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) { }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR || P.split > 1) cluster_sync_all();
  if constexpr (SUMS) {
    if (warp >= 4 && part == 0 && *(volatile int*)&far_flag && !*abortp) {
      if (TMA_OUT && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      __syncwarp();  // behind every lane's stores
      for (int tile = cluster_id; tile < total; tile += num_clusters)
        far_tile<A_ROW, PAIR>(P, S, nseg, tile, (int)rank * 128 + (warp & 3) * 32, ((warp - 4) >> 2) * COLS, COLS,
                              lane);
    }
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
}

// The last, partial k-slab of every group, filled up with zeros to 64 rows:
// what the drhs product reads instead of rows that belong to the next group.
// out[g][64][ld] for both operands, 8 columns a thread.
struct TailParams {
  const uint16_t* x[2];
  uint16_t* out[2];
  int64_t ld[2], width[2], ld_out[2];
  const void* sizes;
  int sizes64, groups;
  int64_t rows;
};

__global__ void __launch_bounds__(256) group_tails_kernel(TailParams P) {
  __shared__ int64_t first_s, count_s;
  const int g = blockIdx.x, lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    int64_t before = 0, own = 0;
    for (int g0 = 0; g0 <= g; g0 += 32) {
      const int i = g0 + lane;
      const int64_t n = i <= g ? min(group_size_at(P.sizes, P.sizes64, i), P.rows) : 0;
      before += __shfl_sync(0xffffffffu, warp_scan(i < g ? n : 0, lane), 31);
      own += __shfl_sync(0xffffffffu, warp_scan(i == g ? n : 0, lane), 31);
    }
    if (lane == 0) {
      const int64_t begin = min(before, P.rows), end = min(before + own, P.rows);
      count_s = (end - begin) % GG_TAIL;
      first_s = end - count_s;
    }
  }
  __syncthreads();
  const int64_t first = first_s, count = count_s;
  if (count == 0) return;
  for (int s = 0; s < 2; ++s) {
    const int64_t vecs = P.ld_out[s] / 8;
    const int64_t n = GG_TAIL * vecs;
    for (int64_t i = (int64_t)blockIdx.y * blockDim.x + threadIdx.x; i < n;
         i += (int64_t)gridDim.y * blockDim.x) {
      const int64_t k = i / vecs, c = (i - k * vecs) * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (k < count) {
        const uint16_t* x = P.x[s] + (first + k) * P.ld[s] + c;
        if (c + 8 <= P.width[s]) {
          v = __ldg((const uint4*)x);
        } else {  // the row ends inside this piece, and so may the tensor's memory
          __align__(16) uint16_t e[8] = {0};
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (c + q < P.width[s]) e[q] = __ldg(x + q);
          v = *(const uint4*)e;
        }
      }
      *(uint4*)(P.out[s] + ((int64_t)g * GG_TAIL + k) * P.ld_out[s] + c) = v;
    }
  }
}

// One warp a row, four elements a lane. Contiguous columns are read as aligned
// words and shifted into place, so that a row may start at any element; the words
// that hold a row's first and last elements are not read whole, since they may lie
// half outside the tensor. With sizes, the matrices of groups without rows are
// left out: a few tokens use a few of many experts (9 rows, 33 experts of 3394 x
// 2386: 282 -> 103 us for both copies).
__global__ void __launch_bounds__(256) pack_bf16_kernel(const uint16_t* x, int64_t rows, int64_t cols,
                                                        int64_t b1, int64_t bs0, int64_t bs1, int64_t rs,
                                                        int64_t cs, uint16_t* out, int64_t ld, int64_t n,
                                                        const void* sizes, int sizes64) {
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t r = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); r < n; r += step) {
    const int64_t b = r / rows, row = r - b * rows;
    if (sizes != nullptr && group_size_at(sizes, sizes64, b) == 0) continue;
    const uint16_t* src = x + (b / b1) * bs0 + (b % b1) * bs1 + row * rs;
    uint16_t* dst = out + r * ld;  // ld: a multiple of 4, 8-byte aligned rows
    if (cs == 1) {
#pragma unroll 2
      for (int64_t c = lane * 4; c < ld; c += 128) {
        uint32_t lo = 0, hi = 0;
        const uint16_t* p = src + c;
        const bool odd = (uintptr_t)p & 2;
        if (c + 4 < cols && (c > 0 || !odd)) {
          const uint32_t* w = (const uint32_t*)((uintptr_t)p & ~(uintptr_t)3);
          lo = __ldg(w);
          hi = __ldg(w + 1);
          if (odd) {
            lo = __funnelshift_r(lo, hi, 16);
            hi = __funnelshift_r(hi, __ldg(w + 2), 16);
          }
        } else {
          if (c < cols) lo = __ldg(p);
          if (c + 1 < cols) lo |= (uint32_t)__ldg(p + 1) << 16;
          if (c + 2 < cols) hi = __ldg(p + 2);
          if (c + 3 < cols) hi |= (uint32_t)__ldg(p + 3) << 16;
        }
        *(uint2*)(dst + c) = make_uint2(lo, hi);
      }
    } else {
      for (int64_t c = lane; c < ld; c += 32) dst[c] = c < cols ? __ldg(src + c * cs) : 0;
    }
  }
}

// ---------------------------------------------------------------------------
// host side

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return (EncodeTiledFn)p;
    return (EncodeTiledFn) nullptr;
  }();
  return fn;
}

// A thread whose first CUDA call this is (a backward pass runs on one of its own) has
// no context yet, and the driver call that encodes a map needs one: then the runtime's
// device is bound. A context that is current already stays so.
template <class Encode>
static CUresult with_context(Encode&& encode) {
  CUresult r = encode();
  int dev = 0;
  if (r == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess)
    r = encode();
  return r;
}

// 3-D map [outer][mid][inner] with 128-byte wide boxes of `box_mid` rows.
static int operand_map(CUtensorMap* tm, const void* ptr, bool fp8, int64_t inner, int64_t mid,
                       int64_t outer, int64_t ld, int64_t s_outer, int box_mid) {
  EncodeTiledFn enc = encode_fn();
  AQT_REQUIRE(enc != nullptr, AQTB200_EDRIVER, "cuTensorMapEncodeTiled entry point not found");
  const int es = fp8 ? 1 : 2;
  AQT_REQUIRE(ptr != nullptr && ((uintptr_t)ptr & 15) == 0, AQTB200_EINVAL, "operand not 16-byte aligned");
  if (mid <= 1 && (ld * es) % 16 != 0) ld = (inner * es + 15) / 16 * 16 / es;
  if (outer <= 1) s_outer = ld * std::max<int64_t>(mid, 1);
  AQT_REQUIRE(ld > 0 && s_outer > 0 && (ld * es) % 16 == 0 && (s_outer * es) % 16 == 0, AQTB200_EINVAL,
              "operand strides must be positive multiples of 16 bytes");
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)mid, (cuuint64_t)outer};
  cuuint64_t strides[2] = {(cuuint64_t)(ld * es), (cuuint64_t)(s_outer * es)};
  cuuint32_t box[3] = {(cuuint32_t)(128 / es), (cuuint32_t)box_mid, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = with_context([&] {
    return enc(tm, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
               const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
  AQT_REQUIRE(r == CUDA_SUCCESS, AQTB200_EDRIVER, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return 0;
}

// Map of bf16 results [group][t][r]: boxes of 64 t by 32 r in the 64-byte swizzle.
static bool output_map(CUtensorMap* tm, void* ptr, int64_t r, int64_t t, int64_t groups, int64_t ld,
                       int64_t s_group) {
  EncodeTiledFn enc = encode_fn();
  if (groups <= 1) s_group = ld * t;
  if (enc == nullptr || ld < r || ld % 8 || s_group % 8 || s_group <= 0) return false;
  cuuint64_t dims[3] = {(cuuint64_t)r, (cuuint64_t)t, (cuuint64_t)groups};
  cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)s_group * 2};
  cuuint32_t box[3] = {32, 64, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return with_context([&] {
           return enc(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, ptr, dims, strides, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                      CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
         }) == CUDA_SUCCESS;
}

static bool is_fp8_dtype(int dt) { return dt == AQTB200_E4M3 || dt == AQTB200_E5M2; }

// How many clusters of `ctas` CTAs the device holds at once (clusters do not cross
// its processor groups: of 148 SMs, not 18 clusters of eight but fewer than 16).
// Looked up once for each device and size.
static int clusters_at_once(int dev, int ctas) {
  static std::atomic<int> known[64][9];
  std::atomic<int>& slot = known[dev & 63][ctas];
  int n = slot.load(std::memory_order_relaxed);
  if (n == 0) {
    auto* fn = grouped_gemm_kernel<true, false, GG_PAIR_NARROW, 2, 64>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(gg_threads(2));
    cfg.dynamicSmemBytes = GG_SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)GG_SMEM) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
    slot.store(n, std::memory_order_relaxed);
  }
  return n;
}

static size_t tail_bytes(const aqtb200_grouped_gemm_desc* d) {
  if (d->contract_groups != 1 || d->group_sizes == nullptr || is_fp8_dtype(d->a_dtype)) return 0;
  const int64_t ra = (d->r + 7) / 8 * 8, tb = (d->t + 7) / 8 * 8;
  return (size_t)d->groups * GG_TAIL * (size_t)(ra + tb) * 2 + 512;
}

static int grouped_gemm(const aqtb200_grouped_gemm_desc* d, int32_t* status, cudaStream_t st) {
  AQT_REQUIRE(d != nullptr, AQTB200_EINVAL, "null grouped gemm descriptor");
  AQT_REQUIRE(d->r >= 0 && d->t >= 0 && d->k >= 0 && d->rows >= 0 && d->groups >= 0, AQTB200_EINVAL,
              "negative extent");
  AQT_REQUIRE(d->contract_groups == 0 || d->contract_groups == 1, AQTB200_EINVAL, "contract_groups: 0 or 1");
  const bool fp8 = is_fp8_dtype(d->a_dtype) && is_fp8_dtype(d->b_dtype);
  AQT_REQUIRE(fp8 || (d->a_dtype == AQTB200_BF16 && d->b_dtype == AQTB200_BF16), AQTB200_EUNSUPPORTED,
              "operand dtypes %d x %d: need bf16 x bf16 or fp8 x fp8", d->a_dtype, d->b_dtype);
  AQT_REQUIRE(d->out_dtype == AQTB200_F32 || d->out_dtype == AQTB200_BF16, AQTB200_EINVAL,
              "out dtype must be f32 or bf16");
  AQT_REQUIRE(!fp8 || (!d->a_mn_major && !d->b_mn_major), AQTB200_EUNSUPPORTED,
              "fp8 operands have the contraction contiguous");
  const bool grouped = d->group_sizes != nullptr;
  AQT_REQUIRE(!grouped || (d->groups >= 1 && d->groups <= AQTB200_MAX_GROUPS), AQTB200_EUNSUPPORTED,
              "between 1 and %d groups (got %lld)", AQTB200_MAX_GROUPS, (long long)d->groups);
  // such a copy's first column is a group's first row, and has to be a multiple of eight
  AQT_REQUIRE(!(grouped && d->contract_groups == 0 && d->b_mn_major), AQTB200_EUNSUPPORTED,
              "grouped rows of b are contiguous along k");
  const int64_t groups = grouped ? d->groups : 1;
  if (grouped && d->contract_groups == 1)
    // the groups' positions are worked out from the sizes and `rows` alone
    AQT_REQUIRE(fp8 ? d->k / 128 >= d->rows / 128 + std::min(groups, d->rows) : d->k >= d->rows,
                AQTB200_EINVAL, "k = %lld positions do not hold %lld grouped rows", (long long)d->k,
                (long long)d->rows);
  if (d->r == 0 || d->t == 0) return 0;
  AQT_REQUIRE(d->out != nullptr, AQTB200_EINVAL, "null output");
  const int64_t lim = (int64_t)1 << 31;
  AQT_REQUIRE(d->r < lim - 512 && d->t < lim - 512 && d->k < lim - 512 && d->rows < lim - 512,
              AQTB200_EUNSUPPORTED, "extent too large for a tensor map");
  const int64_t k = d->k;
  AQT_REQUIRE(k == 0 || !fp8 || (d->a_scale != nullptr && d->b_scale != nullptr), AQTB200_EINVAL,
              "fp8 operands need their scales");
  AQT_REQUIRE(((uintptr_t)d->note & 15) == 0, AQTB200_EINVAL, "notes on scales: 16-byte aligned");

  GGParams P{};
  P.mode = d->contract_groups;
  P.bk = fp8 ? 128 : 64;
  P.a_mn = d->a_mn_major; P.b_mn = d->b_mn_major;
  P.r = (int)d->r; P.t = (int)d->t;
  P.rows = (int)(P.mode == 0 ? d->t : (grouped ? d->rows : k));
  P.sizes = d->group_sizes; P.sizes64 = d->sizes_int64; P.groups = grouped ? (int)d->groups : 0;
  P.num_kb = (int)((k + P.bk - 1) / P.bk);
  const int64_t len = P.mode == 0 ? (d->t + groups - 1) / groups : d->t;
  const bool a_row = fp8 && !d->a_scale_square;
  // Uneven groups: room for one and a half times the average before a second
  // pass. fp8 hands over an accumulator per 128-block, bf16 one per tile.
  const int64_t want = grouped && P.mode == 0 ? len + len / 2 : len;
  // Scales that are powers of two can be left to the tensor core, which then sums
  // the whole contraction (8192 x 4096 x 14336: 432 / 419 / 526 us against 588 / 537
  // / 711; 8192 x 8192 x 8192: 471 / 469 / 465 against 620 / 615 / 762). Its sums drop what
  // does not fit 24 bits, each step of 32 products less than 2^-23 of the running
  // sum (measured, all products positive: 2^-26 a step, 8e-6 over 14336): nothing
  // beside a bf16 result's rounding of 2^-8 as long as the steps' total stays below
  // 2^-10. f32 results keep the f32 registers.
  const bool po2 = fp8 && d->scales_po2 && d->out_dtype == AQTB200_BF16 && P.num_kb * 4 <= 1 << 13 &&
                   (d->a_scale_square || d->a_scale_r_stride == 1);
  const auto ctas_of = [&](int nt) { return !fp8 || (nt <= 128 ? GG_PAIR_NARROW : GG_PAIR_WIDE) ? 2 : 1; };
  const auto units_of = [&](int nt) { return std::max(1, gemm_sms() / ctas_of(nt)); };
  // Tiles, or the most there can be: groups that end inside a tile add one each.
  const auto tiles_of = [&](int nt) {
    const int64_t per = (d->t + nt - 1) / nt, rows = 128 * ctas_of(nt);
    return (d->r + rows - 1) / rows *
           (P.mode == 1 ? groups * per : grouped ? d->t / nt + std::min<int64_t>(d->groups + 1, d->t) : per);
  };
  // Scales in TMEM leave two accumulators of 224 columns, or one of 256: enough
  // where no CTA pair has a second tile to overlap (1024 x 4096 x 4096, 64 tiles on
  // 74 pairs and not 80: 25 / 25 / 34 us against 37 / 37 / 36).
  P.one_half = po2 && tiles_of(256) <= units_of(256);
  const int most = po2 && !P.one_half ? GG_MX_COLS : 256;
  // Columns of a tile. A group of `want` rows costs ceil(want / nt) passes over its
  // weights, and an MMA's time goes with its columns.
  P.nt = want <= most ? (int)std::max<int64_t>(32, (want + 31) / 32 * 32) : most;
  if (want > most && !grouped) {
    // The width whose rounds cost least in total; each tile has a cost of its own
    // besides, in columns: 80 where the epilogue adds every 128-block, 8 otherwise. With
    // f32 scales 2047 x 4096 x 14336 takes 174 us at 80 or 160 and 242 at 0 or 8, 4096 x
    // 4096 x 4096 109 and 128, 3300 x 4096 x 3500 87 and 113, 700 x 4096 x 20000 103 and
    // 123; on the tensor core 0, 8 and 80 give the same to 1 % but for the last but one
    // (86, 86, 77 us). Products with groups are left out: the number of their tiles, or
    // how long each group's contraction is, is known on the device only.
    const int extra = po2 || !fp8 ? 8 : 80;
    int64_t least = INT64_MAX;
    for (int nt = most; nt >= 160; nt -= 32) {
      const int64_t cost = (tiles_of(nt) + units_of(nt) - 1) / units_of(nt) * (nt + extra);
      if (cost < least) { least = cost; P.nt = nt; }
    }
  }
  // Where narrow tiles too fit the device at once, they share the work out further
  // (449 x 173 x 5426, forward and gradients: 64 us wide, 33 us so; 775 x 3418 x 386
  // in two groups, bf16: 59, 47 us). 32 columns gain nothing on 64 and lost up to
  // 10 %. Short products over the rows divide the contraction instead (`split`).
  if (want > (P.mode == 1 ? 64 : 128))
    for (int nt = 64; nt <= 128 && nt < P.nt; nt += 32)
      if (tiles_of(nt) <= units_of(nt)) { P.nt = nt; break; }
  const bool mx = po2 && P.nt > 128;
  P.one_half = P.one_half && mx;
  const int ctas = ctas_of(P.nt), units = units_of(P.nt);
  P.r_tiles = (int)((d->r + 128 * ctas - 1) / (128 * ctas));
  P.t_tiles = (int)((d->t + P.nt - 1) / P.nt);
  const uint32_t fa = fp8 ? (d->a_dtype == AQTB200_E5M2) : 1, fb = fp8 ? (d->b_dtype == AQTB200_E5M2) : 1;
  P.idesc = (1u << 4) | (fa << 7) | (fb << 10) | ((uint32_t)P.a_mn << 15) | ((uint32_t)P.b_mn << 16) |
            ((ctas == 2 ? 16u : 8u) << 24);
  // with scales: no accumulator type, 8-bit exponents
  if (mx) P.idesc = (P.idesc & ~(1u << 4)) | (1u << 23);
  P.b_stage = P.b_mn ? (P.nt / ctas + 63) / 64 * 8192 : P.nt / ctas * 128;
  P.stages = std::min(GG_MAX_STAGES, (mx ? GG_RING_MX : fp8 && P.nt > 128 ? GG_RING_WIDE : GG_RING) /
                                         ((mx ? 2 : gg_slabs(fp8, P.nt)) * (GG_A_STAGE + P.b_stage)));
  P.buf_cols = P.nt <= 64 ? 64 : P.nt <= 128 ? 128 : 256;
  P.half_kb = 256 / P.buf_cols;
  P.a_scale = d->a_scale; P.sa_g = d->a_scale_group_stride; P.sa_k = d->a_scale_k_stride;
  P.sa_r = d->a_scale_r_stride;
  P.b_scale = d->b_scale; P.sb_k = d->b_scale_k_stride;
  P.note = (const uint4*)d->note; P.note_k = d->note_k_stride; P.note_t = d->note_stride;
  P.note_padded = P.mode == 0 && grouped && d->note_padded;
  P.a = (const uint8_t*)d->a; P.a_ld = d->a_ld; P.a_g = d->a_group_stride;
  P.b = (const uint8_t*)d->b; P.b_ld = d->b_ld;
  P.k = (int)k; P.a_e5 = d->a_dtype == AQTB200_E5M2; P.b_e5 = d->b_dtype == AQTB200_E5M2;
  P.out = d->out; P.out_f32 = d->out_dtype == AQTB200_F32;
  P.o_ld = d->out_ld; P.o_g = d->out_group_stride;
  P.out_staged = !P.out_f32 && ((uintptr_t)d->out & 15) == 0 && d->out_ld % 8 == 0 &&
                 (P.mode == 0 || !grouped || d->out_group_stride % 8 == 0);
  P.status = status;

  const int64_t tiles = tiles_of(P.nt);
  AQT_REQUIRE(tiles < lim - 65536, AQTB200_EUNSUPPORTED, "more than 2^31 output tiles");
  int dev = 0;
  AQT_CUDA_OK(cudaGetDevice(&dev));
  // Few tiles: the contraction of each is shared by up to four of a cluster, which
  // add their sums through distributed shared memory, in order -- as many as keep
  // every cluster on the device at once (1 x 4096 x 4096 fp8 on CTA pairs: one a
  // tile 13.7 us, two 10.9 us, four, in two rounds, 18.3 us).
  P.split = 1;
  if (P.mode == 0 && P.nt <= 128)
    for (int s = 2; s <= 4 && P.num_kb >= s * 4 && tiles * s <= units; ++s)
      if (tiles <= clusters_at_once(dev, ctas * s)) P.split = s;

  CUtensorMap tmA, tmB, tmAt, tmBt;
  memset(&tmA, 0, sizeof(tmA));
  tmB = tmAt = tmBt = tmA;
  int rc;
  if (k > 0) {
    const int64_t ga = P.mode == 0 ? groups : 1;
    rc = P.a_mn ? operand_map(&tmA, d->a, fp8, d->r, k, ga, d->a_ld, d->a_group_stride, 64)
                : operand_map(&tmA, d->a, fp8, k, d->r, ga, d->a_ld, d->a_group_stride, 128);
    if (rc) return rc;
    rc = P.b_mn ? operand_map(&tmB, d->b, fp8, d->t, k, 1, d->b_ld, 0, 64)
                : operand_map(&tmB, d->b, fp8, k, d->t, 1, d->b_ld, 0, P.nt / ctas);
    if (rc) return rc;
  }
  if (P.mode == 1 && !fp8 && grouped && k > 0) {
    AQT_REQUIRE(P.a_mn && P.b_mn, AQTB200_EUNSUPPORTED, "bf16 over grouped rows: both operands row by row");
    AQT_REQUIRE(d->workspace != nullptr && d->workspace_bytes >= tail_bytes(d) &&
                    ((uintptr_t)d->workspace & 255) == 0,
                AQTB200_EWORKSPACE, "grouped contraction: workspace too small or not 256-byte aligned");
    TailParams Q{};
    Q.x[0] = (const uint16_t*)d->a; Q.x[1] = (const uint16_t*)d->b;
    Q.ld[0] = d->a_ld; Q.ld[1] = d->b_ld;
    Q.width[0] = d->r; Q.width[1] = d->t;
    Q.ld_out[0] = (d->r + 7) / 8 * 8; Q.ld_out[1] = (d->t + 7) / 8 * 8;
    Q.out[0] = (uint16_t*)d->workspace;
    Q.out[1] = Q.out[0] + ((size_t)d->groups * GG_TAIL * Q.ld_out[0] + 127) / 128 * 128;
    Q.sizes = d->group_sizes; Q.sizes64 = d->sizes_int64; Q.groups = (int)d->groups;
    Q.rows = P.rows;
    const int64_t vecs = GG_TAIL * std::max(Q.ld_out[0], Q.ld_out[1]) / 8;
    const unsigned gy = (unsigned)std::max<int64_t>(1, std::min<int64_t>(32, (vecs + 1023) / 1024));
    group_tails_kernel<<<dim3((unsigned)d->groups, gy), 256, 0, st>>>(Q);
    AQT_CUDA_OK(cudaGetLastError()); count_launch();
    rc = operand_map(&tmAt, Q.out[0], false, d->r, GG_TAIL, d->groups, Q.ld_out[0],
                     Q.ld_out[0] * GG_TAIL, 64);
    if (rc) return rc;
    rc = operand_map(&tmBt, Q.out[1], false, d->t, GG_TAIL, d->groups, Q.ld_out[1],
                     Q.ld_out[1] * GG_TAIL, 64);
    if (rc) return rc;
  }

  if (fp8 && !mx && P.nt > 128 && P.out_staged) {
    // the results' map travels in the place of the tails', which fp8 has no use for
    P.tma_out = output_map(&tmAt, d->out, d->r, d->t, P.mode == 1 ? groups : 1, d->out_ld,
                           d->out_group_stride);
  }

  const size_t smem = mx ? GG_SMEM_MX : GG_SMEM;
  // Whole tiles round robin: the fewest CTAs that keep the number of rounds.
  const int64_t rounds = (tiles + units - 1) / units;
  const int64_t clusters = P.split > 1 ? tiles
                           : grouped   ? std::min<int64_t>(tiles, units)
                                       : (tiles + rounds - 1) / rounds;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * ctas * P.split));
  cfg.blockDim = dim3(gg_threads(P.nt <= 128 ? 2 : 4));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas * P.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  // Launched while the quantizer of b still runs, in forward and dlhs products: with
  // no positions to sum there was no quantizer.
  cfg.numAttrs = fp8 && P.mode == 0 && k > 0 && d->follows_quantize ? 2 : 1;
#define AQT_GG(...)                                                                                \
  do {                                                                                             \
    static std::atomic<bool> attr_done[64]; /* calls come from several threads */                  \
    if (!attr_done[dev & 63].load(std::memory_order_acquire)) {                                    \
      AQT_CUDA_OK(cudaFuncSetAttribute(grouped_gemm_kernel<__VA_ARGS__>,                           \
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)); \
      attr_done[dev & 63].store(true, std::memory_order_release);                                  \
    }                                                                                              \
    AQT_CUDA_OK(cudaLaunchKernelEx(&cfg, grouped_gemm_kernel<__VA_ARGS__>, tmA, tmB, tmAt, tmBt, P)); \
  } while (0)
  if (!fp8) {
    if (P.nt <= 64) AQT_GG(false, false, true, 2, 32);
    else if (P.nt <= 128) AQT_GG(false, false, true, 2, 64);
    else AQT_GG(false, false, true, 4, 64);
  } else if (mx) {
    if (a_row) AQT_GG(true, true, true, 4, 64, true);
    else AQT_GG(true, false, true, 4, 64, true);
  } else if (!a_row) {
    if (P.nt <= 64) AQT_GG(true, false, GG_PAIR_NARROW, 2, 32);
    else if (P.nt <= 128) AQT_GG(true, false, GG_PAIR_NARROW, 2, 64);
    else AQT_GG(true, false, GG_PAIR_WIDE, 4, 64);
  } else {
    if (P.nt <= 64) AQT_GG(true, true, GG_PAIR_NARROW, 2, 32);
    else if (P.nt <= 128) AQT_GG(true, true, GG_PAIR_NARROW, 2, 64);
    else AQT_GG(true, true, GG_PAIR_WIDE, 4, 64);
  }
#undef AQT_GG
  AQT_CUDA_OK(cudaGetLastError()); count_launch();
  return 0;
}

}  // namespace aqtb200

using namespace aqtb200;

extern "C" {

size_t aqtb200_grouped_gemm_workspace_bytes(const aqtb200_grouped_gemm_desc* d) {
  return d == nullptr ? 0 : tail_bytes(d);
}

int aqtb200_grouped_gemm(const aqtb200_grouped_gemm_desc* d, int32_t* status, void* stream) {
  return grouped_gemm(d, status, (cudaStream_t)stream);
}

int aqtb200_pack_bf16(const aqtb200_view* x, void* out, int64_t ld, void* stream) {
  return aqtb200_pack_bf16_groups(x, nullptr, 0, out, ld, stream);
}

int aqtb200_pack_bf16_groups(const aqtb200_view* x, const void* group_sizes, int32_t sizes_int64, void* out,
                             int64_t ld, void* stream) {
  AQT_REQUIRE(x != nullptr && x->dtype == AQTB200_BF16, AQTB200_EINVAL, "pack: a bf16 view");
  AQT_REQUIRE(x->b0 >= 0 && x->b1 >= 0 && x->rows >= 0 && x->cols >= 0 && ld >= x->cols, AQTB200_EINVAL,
              "pack: bad extents");
  const int64_t n = x->b0 * x->b1 * x->rows;
  if (n == 0 || ld == 0) return 0;
  AQT_REQUIRE(ld % 8 == 0 && ((uintptr_t)out & 15) == 0, AQTB200_EINVAL,
              "pack: rows of whole 16-byte pieces, 16-byte aligned");
  AQT_REQUIRE(out != nullptr && (x->ptr != nullptr || x->cols == 0), AQTB200_EINVAL, "pack: null pointer");
  const int64_t blocks = std::min<int64_t>((n + 7) / 8, (int64_t)sm_count() * 16);
  pack_bf16_kernel<<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(
      (const uint16_t*)x->ptr, x->rows, x->cols, x->b1, x->b0_stride, x->b1_stride, x->row_stride,
      x->col_stride, (uint16_t*)out, ld, n, group_sizes, sizes_int64);
  AQT_CUDA_OK(cudaGetLastError()); count_launch();
  return 0;
}

}  // extern "C"
