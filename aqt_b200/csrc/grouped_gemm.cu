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
// Persistent kernel, one CTA pair (cta_group::2) per two SMs, 12 warps a CTA:
//   warp 0      TMA producer, 128-byte k-slabs, 128-byte swizzle, no multicast
//   warp 1      MMA issuer (even CTA)
//   warps 4-11  epilogue: two per TMEM lane quarter, 128 columns each
// bf16 accumulates the whole contraction in TMEM (two 256-column accumulators:
// the epilogue of one tile runs under the next tile's MMAs). fp8 accumulates
// one 128-block there; the epilogue warps read it, multiply by the two scales
// and add it to f32 registers (128 a thread) while the tensor core fills the
// other accumulator.
//
// Group sizes stay on the device: every CTA scans them once (prefix sums in
// shared memory) and finds its tiles from that, so no call waits for the host.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>

#include "groups.cuh"
#include "tcgen05.cuh"

namespace aqtb200 {

int sm_count();

constexpr int GG_EPI = 8;
constexpr int GG_COLS = 128;                 // columns an epilogue warp holds
constexpr int GG_THREADS = 32 * (4 + GG_EPI);  // whole warpgroups, for the register split
// Registers: 384 threads start with 168 each (64512). The first warpgroup keeps
// 88 of them and the two epilogue warpgroups, whose threads hold 128 sums, take
// 208: 128 * 88 + 256 * 208 = 64512.
#define GG_REGS_FEW "88"
#define GG_REGS_MANY "208"
constexpr int GG_A_STAGE = 128 * 128;        // this CTA's 128 rows of A, 128 bytes of k
constexpr int GG_MAX_STAGES = 10;
constexpr int GG_RING = 192 * 1024;          // bytes of the operand ring
constexpr int GG_F_BYTES = GG_EPI * GG_COLS * 4;  // scale factors, one a column and warp
constexpr int GG_MAX_SEG = AQTB200_MAX_GROUPS + 1;
constexpr int GG_TAIL = 64;                  // k-slab of bf16 elements

struct GGParams {
  int mode;  // 0: t is grouped; 1: the contraction is grouped
  int nt;    // columns of a full tile
  int stages, b_stage;
  int split;           // CTA pairs of a cluster that share one tile's contraction
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
  void* out;
  int out_f32;
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

__device__ __forceinline__ void gg_mma(bool fp8, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                       uint32_t idesc, uint32_t accumulate) {
  if (fp8) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* tm, uint32_t leader_bar,
                                                 int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(tm), "r"(leader_bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
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

template <bool FP8>
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
  T.r0 = ri * 256;
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

// Slabs [kb0, kb1) of the pair's share of a tile's contraction.
__device__ __forceinline__ int share_of(int nkb, int part, int split) {
  return (int)((int64_t)nkb * part / split);
}

template <bool FP8, bool A_ROW>
__global__ void __launch_bounds__(GG_THREADS, 1)
grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmAt, const __grid_constant__ CUtensorMap tmBt,
                    GGParams P) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full_bar[GG_MAX_STAGES];   // used in the pair's even CTA
  __shared__ __align__(8) uint64_t empty_bar[GG_MAX_STAGES];  // one per CTA
  __shared__ __align__(8) uint64_t tfull_bar[2];              // one per CTA
  __shared__ __align__(8) uint64_t tempty_bar[2];             // used in the pair's even CTA
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int nseg_s;
  __shared__ int total_s;
  __shared__ Segments S;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const uint32_t rank = crank & 1u;        // within the pair
  const uint32_t lead = crank & ~1u;       // the pair's even CTA
  const int part = (int)(crank >> 1);
  const bool leader = rank == 0;
  const int cluster_id = blockIdx.x / (2 * P.split);
  const int num_clusters = gridDim.x / (2 * P.split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < P.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&tfull_bar[s], 1);
      mbar_init(&tempty_bar[s], 2 * GG_EPI);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
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
  cluster_sync_all();  // both CTAs' barriers exist before anyone signals them
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  const int nseg = nseg_s;
  const int total = total_s;
  volatile int* abortp = &abort_flag;
  const uint32_t peer_abort = map_to_cta(smem_u32(&abort_flag), crank ^ 1u);
  const int stage_bytes = GG_A_STAGE + P.b_stage;
  int fail = 0;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 " GG_REGS_FEW ";");
  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    if (lane == 0) {
      int stage = 0, cur = 0;
      uint32_t phase = 0;
      const int b_boxes = P.b_mn ? (P.nt / 2 + 63) / 64 : 1;
      for (int tile = cluster_id; tile < total && !fail; tile += num_clusters) {
        const TileAt T = gg_tile<FP8>(P, S, nseg, tile, cur);
        const int kb0 = share_of(T.nkb, part, P.split), kb1 = share_of(T.nkb, part + 1, P.split);
        const int ra = T.r0 + (int)rank * 128, tb = T.t0 + (int)rank * (T.n / 2);
        const int ga = P.mode == 0 ? T.seg : 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abortp)) { fail = 1; break; }
          const uint32_t lbar = map_to_cta(smem_u32(&full_bar[stage]), lead);
          if (leader) mbar_expect_tx(&full_bar[stage], 2 * stage_bytes);
          uint8_t* sa = smem + stage * stage_bytes;
          uint8_t* sb = sa + GG_A_STAGE;
          if (P.mode == 1 && !FP8 && T.klen - kb * GG_TAIL < GG_TAIL && P.groups > 0) {
            // the group ends inside this slab: its copy, filled up with zeros
            for (int j = 0; j < 2; ++j)
              tma_load_3d_pair(sa + j * 8192, &tmAt, lbar, ra + j * 64, 0, T.seg);
            for (int j = 0; j < b_boxes; ++j)
              tma_load_3d_pair(sb + j * 8192, &tmBt, lbar, tb + j * 64, 0, T.seg);
          } else {
            const int kk = T.k0 + kb * P.bk;
            if (P.a_mn) {
              for (int j = 0; j < 2; ++j)
                tma_load_3d_pair(sa + j * 8192, &tmA, lbar, ra + j * 64, kk, ga);
            } else {
              tma_load_3d_pair(sa, &tmA, lbar, kk, ra, ga);
            }
            if (P.b_mn) {
              for (int j = 0; j < b_boxes; ++j)
                tma_load_3d_pair(sb + j * 8192, &tmB, lbar, tb + j * 64, kk, 0);
            } else {
              tma_load_3d_pair(sb, &tmB, lbar, kk, tb, 0);
            }
          }
          if (++stage == P.stages) { stage = 0; phase ^= 1; }
        }
      }
      if (fail) {
        *abortp = 1;
        st_cluster_u32(peer_abort, 1u);
        if (P.status) atomicCAS(P.status, 0, 1);
      }
    }
    __syncwarp();
    if (P.split > 1) cluster_sync_all();
  } else if (warp == 1) {
    // ---------------- MMA issuer (even CTA) ----------------
    if (lane == 0 && leader) {
      int stage = 0, cur = 0;
      uint32_t phase = 0;
      uint32_t unit = 0;  // accumulator uses so far
      const uint64_t a_step = P.a_mn ? 128 : 2, b_step = P.b_mn ? 128 : 2;
      for (int tile = cluster_id; tile < total && !fail; tile += num_clusters) {
        const TileAt T = gg_tile<FP8>(P, S, nseg, tile, cur);
        const int kb0 = share_of(T.nkb, part, P.split), kb1 = share_of(T.nkb, part + 1, P.split);
        const uint32_t idesc = P.idesc | ((uint32_t)(T.n >> 3) << 17);
        for (int kb = kb0; kb < kb1; ++kb) {
          const uint32_t buf = unit & 1u;
          if (FP8 || kb == kb0) {
            if (!mbar_wait(&tempty_bar[buf], ((unit >> 1) & 1u) ^ 1u, abortp)) { fail = 2; break; }
          }
          if (!mbar_wait(&full_bar[stage], phase, abortp)) { fail = 2; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * stage_bytes), sb = sa + GG_A_STAGE;
          const uint64_t ad = P.a_mn ? smem_desc_mn(sa, 8192) : make_smem_desc(sa);
          const uint64_t bd = P.b_mn ? smem_desc_mn(sb, 8192) : make_smem_desc(sb);
          const uint32_t d = tmem_base + buf * 256u;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            gg_mma(FP8, d, ad + a_step * k, bd + b_step * k, idesc,
                   (k > 0 || (!FP8 && kb > kb0)) ? 1u : 0u);
          // delivered to both CTAs of this pair
          asm volatile(
              "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
              " [%0], %1;" ::"r"(smem_u32(&empty_bar[stage])),
              "h"((uint16_t)(3u << lead))
              : "memory");
          if (FP8 || kb + 1 == kb1) {
            asm volatile(
                "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
                " [%0], %1;" ::"r"(smem_u32(&tfull_bar[buf])),
                "h"((uint16_t)(3u << lead))
                : "memory");
            ++unit;
          }
          if (++stage == P.stages) { stage = 0; phase ^= 1; }
        }
      }
      if (fail) {
        *abortp = 1;
        st_cluster_u32(peer_abort, 1u);
        if (P.status) atomicCAS(P.status, 0, 2);
      }
    }
    __syncwarp();
    if (P.split > 1) cluster_sync_all();
  } else {
    if (P.split > 1) cluster_sync_all();
  }
  } else {
    // ---------------- epilogue (both CTAs, own 128 rows) ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 " GG_REGS_MANY ";");
    const int quarter = warp & 3;
    const int c0 = ((warp - 4) >> 2) * GG_COLS;  // first column of this warp
    float* const fac = (float*)(smem + P.stages * stage_bytes) + (warp - 4) * GG_COLS;
    uint32_t unit = 0;
    int cur = 0;
    bool have = false;
    float acc[GG_COLS];
    const uint32_t tlane = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c0;
    // The place in the output is worked out anew (`again` hides that from the
    // compiler): kept across the contraction it would cost registers there.
    auto store = [&](int again) {
      asm volatile("" : "+r"(again));
      const TileAt T = gg_tile<FP8>(P, S, nseg, again, cur);
      const int r = T.r0 + (int)rank * 128 + quarter * 32 + lane;
      if (r < P.r) {
        const int64_t at = (P.mode == 1 ? (int64_t)T.seg * P.o_g : 0) + (int64_t)(T.t0 + c0) * P.o_ld + r;
        const int m = T.tvalid - c0;
        if (P.out_f32) {
          float* o = (float*)P.out + at;
#pragma unroll
          for (int j = 0; j < GG_COLS; ++j)
            if (j < m) o[j * P.o_ld] = acc[j];
        } else {
          __nv_bfloat16* o = (__nv_bfloat16*)P.out + at;
#pragma unroll
          for (int j = 0; j < GG_COLS; ++j)
            if (j < m) o[j * P.o_ld] = __float2bfloat16_rn(acc[j]);
        }
      }
    };
    for (int tile = cluster_id; tile < total; tile += num_clusters) {
      const TileAt T = gg_tile<FP8>(P, S, nseg, tile, cur);
      have = true;
      const int kb0 = share_of(T.nkb, part, P.split), kb1 = share_of(T.nkb, part + 1, P.split);
      const int cols = T.n - c0;  // this warp's columns that the MMAs write
#pragma unroll
      for (int j = 0; j < GG_COLS; ++j) acc[j] = 0.f;
      const float* pa = nullptr;
      const float* pb = nullptr;
      if constexpr (FP8) {
        const int64_t kabs = T.k0 / 128 + kb0;
        const int row = min(T.r0 + (int)rank * 128 + (A_ROW ? quarter * 32 + lane : 0), P.r - 1);
        pa = P.a_scale + (P.mode == 0 ? (int64_t)T.seg * P.sa_g : 0) + kabs * P.sa_k +
             (int64_t)(A_ROW ? row : row >> 7) * P.sa_r;
        pb = P.b_scale + kabs * P.sb_k + T.t0 + c0 + lane;
      }
      float na = 0.f, nb[4] = {0.f, 0.f, 0.f, 0.f};  // scales of the next slab
      auto scales = [&]() {
        const int m = T.tvalid - c0 - lane;
        na = __ldg(pa);
#pragma unroll
        for (int q = 0; q < 4; ++q) nb[q] = m > 32 * q ? __ldg(pb + 32 * q) : 0.f;
        pa += P.sa_k;
        pb += P.sb_k;
      };
      if (FP8 && kb0 < kb1) scales();
      for (int kb = kb0; kb < kb1; kb = FP8 ? kb + 1 : kb1) {
        const uint32_t buf = unit & 1u;
        float fa = 1.f;
        if constexpr (FP8) {
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q) fac[lane + 32 * q] = A_ROW ? nb[q] : nb[q] * na;
          fa = na;
          __syncwarp();
          if (kb + 1 < kb1) scales();
        }
        int ok = mbar_wait(&tfull_bar[buf], (unit >> 1) & 1u, abortp) ? 1 : 0;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) { fail = 3; break; }
        tc_fence_after();
        if (cols > 0) {
          uint32_t v[2][16];
          tc_ld16(tlane + buf * 256u, v[0]);
#pragma unroll
          for (int c = 0; c < GG_COLS / 16; ++c) {
            if (c * 16 >= cols) break;  // the same for the whole warp
            tc_wait_ld();
            if ((c + 1) * 16 < cols && c + 1 < GG_COLS / 16)
              tc_ld16(tlane + buf * 256u + (c + 1) * 16, v[(c + 1) & 1]);
            const uint32_t* p = v[c & 1];
            if constexpr (FP8) {
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                const float4 f = *(const float4*)(fac + c * 16 + j);
                const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const float w = __uint_as_float(p[j + q]);
                  acc[c * 16 + j + q] = A_ROW ? fmaf(w * fs[q], fa, acc[c * 16 + j + q])
                                              : fmaf(w, fs[q], acc[c * 16 + j + q]);
                }
              }
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[c * 16 + j] = __uint_as_float(p[j]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&tempty_bar[buf]), lead));
        ++unit;
      }
      if (fail) break;
      if (P.split == 1) store(tile);
    }
    if (P.split > 1) {
      // Parts of one tile: parts 1.. leave their sums in their own shared memory
      // (the operand ring is idle by now), part 0 adds them in part order.
      float* mine = (float*)smem + (size_t)c0 * 128 + quarter * 32 + lane;
      if (have && !fail && part > 0 && c0 < P.nt) {
#pragma unroll
        for (int j = 0; j < GG_COLS; ++j)
          if (c0 + j < P.nt) mine[j * 128] = acc[j];
      }
      __syncwarp();
      cluster_sync_all();
      if (have && !fail && part == 0 && c0 < P.nt) {
        for (int p = 1; p < P.split; ++p) {
          const uint32_t from = map_to_cta(smem_u32(mine), 2 * p + rank);
#pragma unroll
          for (int j = 0; j < GG_COLS; ++j)
            if (c0 + j < P.nt) acc[j] += ld_cluster_f32(from + j * 512);
        }
        store(cluster_id);
      }
    }
    if (fail && lane == 0) {
      *abortp = 1;
      st_cluster_u32(peer_abort, 1u);
      if (P.status) atomicCAS(P.status, 0, 3);
    }
  }

  __syncwarp();
  if (*abortp) {
    // copies still in flight land in shared memory that is still ours
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) { }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512)
                 : "memory");
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
      // operands are padded to whole 8-element pieces (strides are multiples of 8)
      if (k < count) v = __ldg((const uint4*)(P.x[s] + (first + k) * P.ld[s] + c));
      *(uint4*)(P.out[s] + ((int64_t)g * GG_TAIL + k) * P.ld_out[s] + c) = v;
    }
  }
}

__global__ void __launch_bounds__(256) pack_bf16_kernel(const uint16_t* x, int64_t rows, int64_t cols,
                                                        int64_t b1, int64_t bs0, int64_t bs1, int64_t rs,
                                                        int64_t cs, uint16_t* out, int64_t ld, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t c = i % ld, rr = i / ld, row = rr % rows, b = rr / rows;
    out[i] = c < cols ? __ldg(x + (b / b1) * bs0 + (b % b1) * bs1 + row * rs + c * cs) : 0;
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
  CUresult r = enc(tm, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                   const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  AQT_REQUIRE(r == CUDA_SUCCESS, AQTB200_EDRIVER, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return 0;
}

static bool is_fp8_dtype(int dt) { return dt == AQTB200_E4M3 || dt == AQTB200_E5M2; }

// Columns of a tile. A group of `len` rows costs ceil(len / nt) passes over its
// weights, an MMA's time goes with its columns.
static int choose_nt(int64_t len, int64_t r_tiles, bool one_group, int pairs) {
  if (len <= 256) return (int)std::max<int64_t>(32, (len + 31) / 32 * 32);
  if (!one_group) return 256;
  // one group, all sizes known: the width whose waves cost least in total
  int best = 256;
  double least = 1e300;
  for (int nt = 256; nt >= 160; nt -= 32) {
    const int64_t tiles = r_tiles * ((len + nt - 1) / nt);
    const double cost = (double)((tiles + pairs - 1) / pairs) * (nt + 8);
    if (cost < least) { least = cost; best = nt; }
  }
  return best;
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
  const int64_t groups = grouped ? d->groups : 1;
  if (d->r == 0 || d->t == 0) return 0;
  AQT_REQUIRE(d->out != nullptr, AQTB200_EINVAL, "null output");
  const int64_t lim = (int64_t)1 << 31;
  AQT_REQUIRE(d->r < lim - 512 && d->t < lim - 512 && d->k < lim - 512 && d->rows < lim - 512,
              AQTB200_EUNSUPPORTED, "extent too large for a tensor map");
  const int64_t k = d->k;
  AQT_REQUIRE(k == 0 || !fp8 || (d->a_scale != nullptr && d->b_scale != nullptr), AQTB200_EINVAL,
              "fp8 operands need their scales");

  GGParams P{};
  P.mode = d->contract_groups;
  P.bk = fp8 ? 128 : 64;
  P.a_mn = d->a_mn_major; P.b_mn = d->b_mn_major;
  P.r = (int)d->r; P.t = (int)d->t;
  P.rows = (int)(P.mode == 0 ? d->t : (grouped ? d->rows : k));
  P.sizes = d->group_sizes; P.sizes64 = d->sizes_int64; P.groups = grouped ? (int)d->groups : 0;
  P.r_tiles = (int)((d->r + 255) / 256);
  P.num_kb = (int)((k + P.bk - 1) / P.bk);
  const int pairs = std::max(1, sm_count() / 2);
  const int64_t len = P.mode == 0 ? (d->t + groups - 1) / groups : d->t;
  // uneven groups: room for one and a half times the average before a second pass
  P.nt = choose_nt(grouped && P.mode == 0 ? len + len / 2 : len, P.r_tiles, !grouped, pairs);
  P.t_tiles = (int)((d->t + P.nt - 1) / P.nt);
  const uint32_t fa = fp8 ? (d->a_dtype == AQTB200_E5M2) : 1, fb = fp8 ? (d->b_dtype == AQTB200_E5M2) : 1;
  P.idesc = (1u << 4) | (fa << 7) | (fb << 10) | ((uint32_t)P.a_mn << 15) | ((uint32_t)P.b_mn << 16) |
            (16u << 24);
  P.b_stage = P.b_mn ? (P.nt / 2 + 63) / 64 * 8192 : P.nt / 2 * 128;
  P.stages = std::min(GG_MAX_STAGES, GG_RING / (GG_A_STAGE + P.b_stage));
  P.a_scale = d->a_scale; P.sa_g = d->a_scale_group_stride; P.sa_k = d->a_scale_k_stride;
  P.sa_r = d->a_scale_r_stride;
  P.b_scale = d->b_scale; P.sb_k = d->b_scale_k_stride;
  P.out = d->out; P.out_f32 = d->out_dtype == AQTB200_F32;
  P.o_ld = d->out_ld; P.o_g = d->out_group_stride;
  P.status = status;

  // Tiles, or the most there can be: groups that end inside a tile add one each.
  const int64_t t_most = P.mode == 1 ? groups * P.t_tiles
                         : grouped   ? d->t / P.nt + std::min<int64_t>(d->groups + 1, d->t)
                                     : P.t_tiles;
  const int64_t tiles = t_most * P.r_tiles;
  AQT_REQUIRE(tiles < lim - 65536, AQTB200_EUNSUPPORTED, "more than 2^31 output tiles");
  // Few tiles: the contraction of each is shared by up to four CTA pairs of one
  // cluster, which add their sums through distributed shared memory, in order.
  P.split = 1;
  if (P.mode == 0 && P.nt <= 128)
    while (P.split < 4 && tiles * P.split * 2 <= pairs && P.num_kb >= P.split * 4) P.split *= 2;

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
                : operand_map(&tmB, d->b, fp8, k, d->t, 1, d->b_ld, 0, P.nt / 2);
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

  const size_t smem = (size_t)P.stages * (GG_A_STAGE + P.b_stage) + GG_F_BYTES + 1024;
  const int64_t clusters = P.split > 1 ? tiles : std::min<int64_t>(tiles, pairs);
  int dev = 0;
  AQT_CUDA_OK(cudaGetDevice(&dev));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * 2 * P.split));
  cfg.blockDim = dim3(GG_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2 * P.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
#define AQT_GG(F, R)                                                                                  \
  do {                                                                                                \
    static bool attr_done[64] = {false};                                                              \
    if (!attr_done[dev & 63]) {                                                                       \
      AQT_CUDA_OK(cudaFuncSetAttribute(grouped_gemm_kernel<F, R>,                                     \
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,                   \
                                       GG_RING + GG_F_BYTES + 1024));                                 \
      attr_done[dev & 63] = true;                                                                     \
    }                                                                                                 \
    AQT_CUDA_OK(cudaLaunchKernelEx(&cfg, grouped_gemm_kernel<F, R>, tmA, tmB, tmAt, tmBt, P));        \
  } while (0)
  if (!fp8) AQT_GG(false, false);
  else if (d->a_scale_square) AQT_GG(true, false);
  else AQT_GG(true, true);
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
  AQT_REQUIRE(x != nullptr && x->dtype == AQTB200_BF16, AQTB200_EINVAL, "pack: a bf16 view");
  AQT_REQUIRE(x->b0 >= 0 && x->b1 >= 0 && x->rows >= 0 && x->cols >= 0 && ld >= x->cols, AQTB200_EINVAL,
              "pack: bad extents");
  const int64_t n = x->b0 * x->b1 * x->rows * ld;
  if (n == 0) return 0;
  AQT_REQUIRE(out != nullptr && (x->ptr != nullptr || x->cols == 0), AQTB200_EINVAL, "pack: null pointer");
  const int64_t blocks = std::min<int64_t>((n + 255) / 256, (int64_t)sm_count() * 16);
  pack_bf16_kernel<<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(
      (const uint16_t*)x->ptr, x->rows, x->cols, x->b1, x->b0_stride, x->b1_stride, x->row_stride,
      x->col_stride, (uint16_t*)out, ld, n);
  AQT_CUDA_OK(cudaGetLastError()); count_launch();
  return 0;
}

}  // extern "C"
