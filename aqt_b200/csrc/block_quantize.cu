// Block quantizer: f32 / bf16 -> fp8 with one f32 scale for each block of 128
// elements along the contraction (1 x 128), or for each 128 x 128 block.
//
//   a = max |x| over the block            s = (a == 0 ? 1 : a) / bound
//   s = max(s, 2^-126) [, rounded up to a power of two]
//   q = fp8(clip(x * (1 / s), -bound, bound))          all in f32, ties to even
//
// One CTA takes one 128 x 128 tile, reads it ONCE and can write it twice: with
// blocks along the columns (q_row, columns contiguous) and, transposed, with
// blocks along the rows (q_col, rows contiguous) -- what a training step needs
// of an activation or a cotangent -- or as one 128 x 128 block in either or
// both orders. Each thread holds 8 x 8 elements: eight columns (one 16- or
// 32-byte load per row) of eight consecutive rows, so that both outputs leave
// in 8-byte pieces; the transposed one passes through a 16 KB tile in shared
// memory whose 8-byte slots are XOR-ed with the column group, which makes both
// its writes and its reads conflict free. Bound: HBM, es + 1 bytes per element
// (es + 2 with both outputs). Measured on 8192 x 14336 bf16: one order 56 us (0.97
// of the copy bandwidth), the transposed one 62 us, both 88 us (0.81), square in
// both orders 79 us; four blocks a SM, since with three the instructions, not the
// memory, are the bound (61, 71, 97, 88 us). 8192 x 7168 f32: 47, 53, 67, 61 us.
// Each warp can also note the range of its scales, in bytes of its own (block_scales.cuh)
// that are written whatever they say, so that no call has to clear them first.
#include <algorithm>

#include "block_scales.cuh"
#include "groups.cuh"

namespace aqtb200 {

constexpr int QB = 128;        // block edge
constexpr int BQ_THREADS = 256;

struct BqParams {
  const void* x;
  int64_t rows, cols, bs0, bs1, b1, rs, cs;  // element strides of the view
  uint8_t* q_row;
  int64_t ld_row;
  float* s_row;
  uint8_t* q_col;
  int64_t ld_col;
  float* s_col;
  uint16_t *note_row, *note_col;  // optional notes on the scales, of each warp and tile
  int64_t row_tiles, col_tiles;
  const void* sizes;  // optional: rows fall into groups, row blocks start anew in each
  int sizes64;
  int64_t groups;
  int po2, square;
  float bound;
};

// max / bound with the conventions above; NaN and infinity go through.
__device__ __forceinline__ float block_scale(float a, float bound, int po2) {
  if (a == 0.f) a = 1.f;
  float s = __fdiv_rn(a, bound);
  if (s < 1.17549435e-38f) s = 1.17549435e-38f;
  if (po2) {
    const uint32_t b = __float_as_uint(s);
    // a normal number with a non-zero mantissa goes up to the next power of two
    if ((b & 0x7f800000u) != 0x7f800000u && (b & 0x007fffffu))
      s = __uint_as_float((b & 0x7f800000u) + 0x00800000u);
  }
  return s;
}

// Four products as four fp8 bytes: (a, b, c, d) times the factors of their pairs.
template <bool E5>
__device__ __forceinline__ uint32_t fp8_quad(float2 ab, float2 cd, float2 f_ab, float2 f_cd) {
  const float2 p = __fmul2_rn(ab, f_ab), q = __fmul2_rn(cd, f_cd);
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(p, __NV_SATFINITE, E5 ? __NV_E5M2 : __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, E5 ? __NV_E5M2 : __NV_E4M3);
  return __byte_perm(lo, hi, 0x5410);
}

// max |.| of bf16 pairs, keeping a NaN (as jnp.max does)
__device__ __forceinline__ uint32_t max_abs_bf16x2(uint32_t m, uint32_t w) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(w & 0x7fff7fffu));
  return r;
}

// The 8 x 8 elements of one thread. bf16 stays packed: 32 registers.
template <bool BF16>
struct Elems;
template <>
struct Elems<true> {
  uint32_t w[8][4];
  __device__ __forceinline__ float get(int i, int j) const {
    return (j & 1) ? bf16hi(w[i][j >> 1]) : bf16lo(w[i][j >> 1]);
  }
  __device__ __forceinline__ void zero(int i) { w[i][0] = w[i][1] = w[i][2] = w[i][3] = 0; }
  // Largest magnitudes as f32 bit patterns (a NaN ranks above infinity).
  __device__ __forceinline__ void row_maxima(uint32_t* row) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t r = w[i][0] & 0x7fff7fffu;
#pragma unroll
      for (int j = 1; j < 4; ++j) r = max_abs_bf16x2(r, w[i][j]);
      row[i] = max(r << 16, r & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void col_maxima(uint32_t* col) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t c = w[0][j] & 0x7fff7fffu;
#pragma unroll
      for (int i = 1; i < 8; ++i) c = max_abs_bf16x2(c, w[i][j]);
      col[2 * j] = c << 16;
      col[2 * j + 1] = c & 0xffff0000u;
    }
  }
  __device__ __forceinline__ void load(int i, const void* p, int64_t at) {
    const uint4 u = __ldg((const uint4*)((const unsigned short*)p + at));
    w[i][0] = u.x; w[i][1] = u.y; w[i][2] = u.z; w[i][3] = u.w;
  }
  // The same eight elements from an address that is only element aligned: aligned
  // pieces of eight bytes, shifted into place. Each piece that is read holds at least
  // one of the elements, so it lies in the tensor's memory.
  __device__ __forceinline__ void load_words(int i, const void* p, int64_t at) {
    const uintptr_t a = (uintptr_t)((const unsigned short*)p + at);
    const uint2* q = (const uint2*)(a & ~(uintptr_t)7);
    const uint2 t0 = __ldg(q), t1 = __ldg(q + 1), t2 = (a & 7) ? __ldg(q + 2) : make_uint2(0, 0);
    const bool far = a & 4;
    const uint32_t v[5] = {far ? t0.y : t0.x, far ? t1.x : t0.y, far ? t1.y : t1.x, far ? t2.x : t1.y,
                           far ? t2.y : t2.x};
    const uint32_t by = (a & 2) * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[i][j] = __funnelshift_r(v[j], v[j + 1], by);
  }
  __device__ __forceinline__ void set(int i, int j, const void* p, int64_t at) {
    const uint32_t v = __ldg((const unsigned short*)p + at);
    w[i][j >> 1] = (j & 1) ? (w[i][j >> 1] & 0xffffu) | (v << 16) : (w[i][j >> 1] & 0xffff0000u) | v;
  }
  __device__ __forceinline__ void drop(int i, int j) { w[i][j >> 1] &= (j & 1) ? 0xffffu : 0xffff0000u; }
};
template <>
struct Elems<false> {
  float v[8][8];
  __device__ __forceinline__ float get(int i, int j) const { return v[i][j]; }
  __device__ __forceinline__ void row_maxima(uint32_t* row) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      row[i] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) row[i] = max(row[i], __float_as_uint(v[i][j]) & 0x7fffffffu);
    }
  }
  __device__ __forceinline__ void col_maxima(uint32_t* col) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      col[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) col[j] = max(col[j], __float_as_uint(v[i][j]) & 0x7fffffffu);
    }
  }
  __device__ __forceinline__ void zero(int i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
  }
  __device__ __forceinline__ void load(int i, const void* p, int64_t at) {
    const float4* q = (const float4*)((const float*)p + at);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    v[i][0] = a.x; v[i][1] = a.y; v[i][2] = a.z; v[i][3] = a.w;
    v[i][4] = b.x; v[i][5] = b.y; v[i][6] = b.z; v[i][7] = b.w;
  }
  __device__ __forceinline__ void load_words(int i, const void* p, int64_t at) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = __ldg((const float*)p + at + j);
  }
  __device__ __forceinline__ void set(int i, int j, const void* p, int64_t at) {
    v[i][j] = __ldg((const float*)p + at);
  }
  __device__ __forceinline__ void drop(int i, int j) { v[i][j] = 0.f; }
};

// VEC: columns contiguous, rows start on 16-byte boundaries.
template <bool BF16, bool E5, bool VEC>
__global__ void __launch_bounds__(BQ_THREADS, BF16 ? 4 : 2) block_quantize_kernel(BqParams P) {
  __shared__ uint2 tile[QB * 16];              // [column][8-byte slot of 8 rows]
  __shared__ __align__(16) uint32_t red[BQ_THREADS / 32][QB];
  __shared__ __align__(16) float col_inv[QB];
  __shared__ int64_t place[3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c8 = tid & 15, rg = tid >> 4;
  const int64_t ct = blockIdx.x % P.col_tiles;
  const int64_t rt = blockIdx.x / P.col_tiles % P.row_tiles;  // with groups, of the padded order
  const int64_t b = blockIdx.x / P.col_tiles / P.row_tiles;

  // a product launched to follow may take the SMs that come free and fetch its
  // weights; it waits for this grid's end before it reads what is written here
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int64_t row0 = rt * QB, row_end = P.rows;
  if (P.sizes != nullptr) {
    if (warp == 0) {
      int64_t off = 0, pad = 0;
      bool found = false;
      for (int64_t g0 = 0; g0 < P.groups; g0 += 32) {
        const int64_t g = g0 + lane;
        const int64_t n = g < P.groups ? min(group_size_at(P.sizes, P.sizes64, g), P.rows) : 0;
        const int64_t end = min(off + warp_scan(n, lane), P.rows);
        int64_t start = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) start = off;
        const int64_t tiles = (end - start + QB - 1) / QB;
        const int64_t pend = pad + warp_scan(tiles, lane);
        const bool mine = rt < pend && rt >= pend - tiles;
        if (mine) {
          place[0] = start + (rt - (pend - tiles)) * QB;
          place[1] = end;
        }
        found = __any_sync(0xffffffffu, mine);
        if (found) break;
        off = __shfl_sync(0xffffffffu, end, 31);
        pad = __shfl_sync(0xffffffffu, pend, 31);
      }
      if (lane == 0) place[2] = found;
    }
    __syncthreads();
    if (!place[2]) return;
    row0 = place[0];
    row_end = place[1];
  }

  const int64_t i0 = b / P.b1, i1 = b % P.b1;
  const int64_t base = i0 * P.bs0 + i1 * P.bs1;
  const int64_t col = ct * QB + c8 * 8;
  const int64_t row = row0 + rg * 8;
  Elems<BF16> x;
  if (VEC && row0 + QB <= row_end && (ct + 1) * QB <= P.cols) {
    const int64_t at = base + row * P.rs + col;
#pragma unroll
    for (int i = 0; i < 8; ++i) x.load(i, P.x, at + i * P.rs);
  } else if (row < row_end && col + 8 <= P.cols && (VEC || P.cs == 1)) {
    // Behind the last row that one is read again and dropped: with a branch a row the
    // eight loads waited for one another (8111 x 4095, bf16, along columns: 41 us
    // with the branches, 27 us without).
    const int64_t at = base + col;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = at + min(row + i, row_end - 1) * P.rs;
      if constexpr (VEC) x.load(i, P.x, r);
      else x.load_words(i, P.x, r);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (row + i >= row_end) x.zero(i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.zero(i);
    if (row < row_end && col < P.cols) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t at = base + min(row + i, row_end - 1) * P.rs;
#pragma unroll
        for (int j = 0; j < 8; ++j) x.set(i, j, P.x, at + min(col + j, P.cols - 1) * P.cs);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (row + i >= row_end || col + j >= P.cols) x.drop(i, j);
      }
    }
  }

  const bool want_row = P.q_row != nullptr, want_col = P.q_col != nullptr;
  float inv_r[8], inv_c[8];
  if (P.square) {
    uint32_t row_max[8];
    x.row_maxima(row_max);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, row_max[i]);
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) red[0][warp] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int w = 0; w < BQ_THREADS / 32; ++w) m = max(m, red[0][w]);
    const float s = block_scale(__uint_as_float(m), P.bound, P.po2);
    const float inv = __fdiv_rn(1.f, s);
    if (tid == 0) {
      const int64_t at = (b * P.row_tiles + rt) * P.col_tiles + ct;
      if (P.s_row != nullptr) P.s_row[at] = s;
      if (P.s_col != nullptr) P.s_col[at] = s;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) inv_r[i] = inv_c[i] = inv;
  } else {
    if (want_row) {
      // Maxima over the sixteen lanes that share eight rows: each exchange halves
      // the rows a lane is in charge of, so eight shuffles do for all of them and
      // lane l ends with row (l / 2) % 8, whose one division it computes.
      uint32_t m[8];
      x.row_maxima(m);
#pragma unroll
      for (int n = 4, o = 8; n > 0; n >>= 1, o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int q = 0; q < n; ++q) {
          const uint32_t give = upper ? m[q] : m[q + n];
          const uint32_t keep = upper ? m[q + n] : m[q];
          m[q] = max(keep, __shfl_xor_sync(0xffffffffu, give, o));
        }
      }
      const uint32_t mine = max(m[0], __shfl_xor_sync(0xffffffffu, m[0], 1));
      const float s = block_scale(__uint_as_float(mine), P.bound, P.po2);
      const float inv = __fdiv_rn(1.f, s);
      const int64_t r = row + ((lane >> 1) & 7);
      if ((lane & 1) == 0 && r < row_end) P.s_row[(b * P.col_tiles + ct) * P.rows + r] = s;
      if (P.note_row != nullptr) {
        const uint16_t note = scale_note(s);
        if (lane == 0) P.note_row[(rt * P.col_tiles + ct) * 8 + warp] = note;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) inv_r[i] = __shfl_sync(0xffffffffu, inv, (lane & 16) | (i << 1));
    }
    if (want_col) {
      uint32_t m[8];
      x.col_maxima(m);
      const bool upper = lane & 16;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t give = upper ? m[q] : m[q + 4];
        const uint32_t keep = upper ? m[q + 4] : m[q];
        m[q] = max(keep, __shfl_xor_sync(0xffffffffu, give, 16));
      }
      *(uint4*)&red[warp][c8 * 8 + (upper ? 4 : 0)] = make_uint4(m[0], m[1], m[2], m[3]);
      __syncthreads();
      float scale = 0.f;
      if (tid < QB) {
        uint32_t top = 0;
#pragma unroll
        for (int w = 0; w < BQ_THREADS / 32; ++w) top = max(top, red[w][tid]);
        const float s = block_scale(__uint_as_float(top), P.bound, P.po2);
        col_inv[tid] = __fdiv_rn(1.f, s);
        if (ct * QB + tid < P.cols)
          P.s_col[(b * P.row_tiles + rt) * P.cols + ct * QB + tid] = s;
        scale = s;
      }
      if (P.note_col != nullptr) {
        const uint16_t note = scale_note(scale);
        if (lane == 0) P.note_col[(rt * P.col_tiles + ct) * 8 + warp] = note;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 v = *(const float4*)&col_inv[c8 * 8 + j];
        inv_c[j] = v.x; inv_c[j + 1] = v.y; inv_c[j + 2] = v.z; inv_c[j + 3] = v.w;
      }
    }
  }

  if (want_row && col < P.ld_row) {
    uint8_t* q = P.q_row + (b * P.rows + row) * P.ld_row + col;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (row + i < row_end) {
        const float2 f = make_float2(inv_r[i], inv_r[i]);
        const uint32_t lo = fp8_quad<E5>(make_float2(x.get(i, 0), x.get(i, 1)),
                                         make_float2(x.get(i, 2), x.get(i, 3)), f, f);
        const uint32_t hi = fp8_quad<E5>(make_float2(x.get(i, 4), x.get(i, 5)),
                                         make_float2(x.get(i, 6), x.get(i, 7)), f, f);
        *(uint2*)(q + i * P.ld_row) = make_uint2(lo, hi);
      }
    }
  }
  if (want_col) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = make_float2(inv_c[j], inv_c[j]);
      const uint32_t lo = fp8_quad<E5>(make_float2(x.get(0, j), x.get(1, j)),
                                       make_float2(x.get(2, j), x.get(3, j)), f, f);
      const uint32_t hi = fp8_quad<E5>(make_float2(x.get(4, j), x.get(5, j)),
                                       make_float2(x.get(6, j), x.get(7, j)), f, f);
      tile[(c8 * 8 + j) * 16 + (rg ^ c8)] = make_uint2(lo, hi);
    }
    __syncthreads();
    const int64_t at = rt * QB + c8 * 8;  // position along the (padded) rows
    if (at < P.ld_col) {
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int c = it * 16 + rg;
        if (ct * QB + c < P.cols)
          *(uint2*)(P.q_col + (b * P.cols + ct * QB + c) * P.ld_col + at) =
              tile[c * 16 + (c8 ^ (c >> 3))];
      }
    }
  }
}

}  // namespace aqtb200

using namespace aqtb200;

extern "C" {

int aqtb200_block_quantize(const aqtb200_block_quant_desc* d, void* stream) {
  AQT_REQUIRE(d != nullptr, AQTB200_EINVAL, "null block quantize descriptor");
  aqtb200_view v = d->x;
  AQT_REQUIRE(v.b0 >= 0 && v.b1 >= 0 && v.rows >= 0 && v.cols >= 0, AQTB200_EINVAL, "negative extent");
  AQT_REQUIRE(v.dtype == AQTB200_F32 || v.dtype == AQTB200_BF16, AQTB200_EUNSUPPORTED,
              "block quantization takes f32 or bf16 (got dtype %d)", v.dtype);
  AQT_REQUIRE(d->qdtype == AQTB200_E4M3 || d->qdtype == AQTB200_E5M2, AQTB200_EUNSUPPORTED,
              "block quantization writes e4m3 or e5m2 (got dtype %d)", d->qdtype);
  const int64_t batch = v.b0 * v.b1;
  if (batch == 0 || v.rows == 0 || v.cols == 0) return 0;
  AQT_REQUIRE(d->q_row != nullptr || d->q_col != nullptr, AQTB200_EINVAL, "no output");
  AQT_REQUIRE(d->square ? (d->scale_row != nullptr || d->scale_col != nullptr)
                        : ((d->q_row == nullptr || d->scale_row != nullptr) &&
                           (d->q_col == nullptr || d->scale_col != nullptr)),
              AQTB200_EINVAL, "an output has no place for its scales");
  AQT_REQUIRE(v.ptr != nullptr, AQTB200_EINVAL, "null input");
  AQT_REQUIRE((d->note_row == nullptr && d->note_col == nullptr) ||
                  (batch == 1 && !d->square && (((uintptr_t)d->note_row | (uintptr_t)d->note_col) & 15) == 0),
              AQTB200_EUNSUPPORTED, "notes on scales: of one matrix in blocks of 1 x 128, 16-byte aligned");
  BqParams P{};
  P.x = v.ptr;
  P.rows = v.rows; P.cols = v.cols; P.b1 = v.b1;
  P.bs0 = v.b0_stride; P.bs1 = v.b1_stride; P.rs = v.row_stride; P.cs = v.col_stride;
  P.q_row = (uint8_t*)d->q_row; P.ld_row = d->ld_row; P.s_row = d->scale_row;
  P.q_col = (uint8_t*)d->q_col; P.ld_col = d->ld_col; P.s_col = d->scale_col;
  P.note_row = (uint16_t*)d->note_row; P.note_col = (uint16_t*)d->note_col;
  P.po2 = d->po2_scale; P.square = d->square;
  P.bound = d->qdtype == AQTB200_E4M3 ? 448.f : 57344.f;
  P.col_tiles = (v.cols + QB - 1) / QB;
  P.row_tiles = (v.rows + QB - 1) / QB;
  if (d->group_sizes != nullptr) {
    AQT_REQUIRE(batch == 1 && !d->square, AQTB200_EUNSUPPORTED,
                "grouped rows: no batch and no 128 x 128 blocks");
    AQT_REQUIRE(d->groups >= 1, AQTB200_EINVAL, "grouped rows without a group");
    P.sizes = d->group_sizes; P.sizes64 = d->sizes_int64; P.groups = d->groups;
    // every group may end in a partial block
    P.row_tiles = P.rows / QB + std::min<int64_t>(d->groups, P.rows);
  }
  AQT_REQUIRE(d->q_row == nullptr ||
                  (d->ld_row % 16 == 0 && d->ld_row >= v.cols && ((uintptr_t)d->q_row & 15) == 0),
              AQTB200_EINVAL, "q_row: 16-byte aligned rows of at least `cols` bytes");
  AQT_REQUIRE(d->q_col == nullptr ||
                  (d->ld_col % 16 == 0 && ((uintptr_t)d->q_col & 15) == 0 &&
                   d->ld_col >= (d->group_sizes != nullptr ? P.row_tiles * QB : v.rows)),
              AQTB200_EINVAL, "q_col: 16-byte aligned rows of at least `rows` bytes (whole blocks when grouped)");
  AQT_REQUIRE(P.row_tiles * P.col_tiles <= (int64_t)0x7fffffff / batch, AQTB200_EUNSUPPORTED,
              "block quantization: more than 2^31 - 1 blocks");
  const int es = dtype_size(v.dtype);
  auto al = [&](int64_t s, int64_t n) { return n <= 1 || (s * es) % 16 == 0; };
  const bool vec = v.col_stride == 1 && ((uintptr_t)v.ptr & 15) == 0 && al(v.row_stride, v.rows) &&
                   al(v.b1_stride, v.b1) && al(v.b0_stride, v.b0);
  const unsigned grid = (unsigned)(P.col_tiles * P.row_tiles * batch);
  cudaStream_t st = (cudaStream_t)stream;
  const bool bf = v.dtype == AQTB200_BF16, e5 = d->qdtype == AQTB200_E5M2;
#define AQT_BQ(B, E)                                                                 \
  do {                                                                               \
    if (vec) block_quantize_kernel<B, E, true><<<grid, BQ_THREADS, 0, st>>>(P);      \
    else block_quantize_kernel<B, E, false><<<grid, BQ_THREADS, 0, st>>>(P);         \
  } while (0)
  if (bf) { if (e5) AQT_BQ(true, true); else AQT_BQ(true, false); }
  else { if (e5) AQT_BQ(false, true); else AQT_BQ(false, false); }
#undef AQT_BQ
  AQT_CUDA_OK(cudaGetLastError()); count_launch();
  return 0;
}

}  // extern "C"
