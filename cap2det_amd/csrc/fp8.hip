// 8-bit floating-point storage: the block quantiser and the product of block-scaled matrices, for one
// weight matrix or one per group of rows.
#include "products_common.h"

using namespace c2d_pr;

namespace {

// ---- quantiser --------------------------------------------------------------------------------------
//
// scale = max(max |x| / F, 2^-126), q = rne8(x / scale).  The quotient is x * r with r = 1 / scale correctly
// rounded, and one correction by its own remainder (Markstein's theorem: the quotient is then correctly
// rounded too): three operations an element where a division takes ten, and no value near a tie falls on
// another side than the true quotient's.  |x| <= F * scale up to rounding, so nothing overflows the type.

template <class T>
struct Eight { f32x4 lo, hi; };

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
}
__device__ __forceinline__ void load8(const __bf16* p, float (&v)[8]) {
  const bf16x8 a = *(const bf16x8*)p;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
}

// eight elements of a row from column c, zeros behind the last
template <class T>
__device__ __forceinline__ void load_chunk(const T* row, int c, int cols, bool wide, float (&v)[8]) {
  if (wide && c + 8 <= cols) {
    load8(row + c, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? (float)row[c + j] : 0.0f;
  }
}

__device__ __forceinline__ float largest(const float (&v)[8]) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));  // (a NaN takes no part)
  return m;
}

__device__ __forceinline__ float largest_of_16_lanes(float m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  return m;
}

template <bool E5M2>
__device__ __forceinline__ float scale_of(float m) {
  return fmaxf(m / (E5M2 ? 57344.0f : 448.0f), 0x1p-126f);
}

template <bool E5M2>
__device__ __forceinline__ u32x2 quantize8(const float (&v)[8], float scale) {
  const float r = 1.0f / scale;
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = v[j] * r;
    q[j] = fmaf(fmaf(-t, scale, v[j]), r, t);
  }
  u32x2 o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = 0;
    if constexpr (E5M2) {
      w = __builtin_amdgcn_cvt_pk_bf8_f32(q[4 * h], q[4 * h + 1], w, false);
      w = __builtin_amdgcn_cvt_pk_bf8_f32(q[4 * h + 2], q[4 * h + 3], w, true);
    } else {
      w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], w, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], w, true);
    }
    o[h] = (unsigned)w;
  }
  return o;
}

__device__ __forceinline__ void store_chunk(unsigned char* row, int c, int cols, bool wide, u32x2 q) {
  if (wide && c + 8 <= cols) {
    *(u32x2*)(row + c) = q;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < cols) row[c + j] = (unsigned char)(q[j >> 2] >> (8 * (j & 3)));
  }
}

struct QuantArgs {
  const void* x;
  long long ldx, x_batch;
  unsigned char* q;
  float* scale;
  int rows, cols, kb, per_wg;  // per_wg: rows of a workgroup (1 x 128 blocks)
  unsigned magic;              // ceil(2^32 / kb): t / kb = umulhi(t, magic) for t < 2^16
  int wide_in, wide_out;
};

// Blocks of 1 x 128: 16 lanes a block, 8 elements a lane, up to 64 blocks a workgroup, all of whose loads
// are issued before the first is used.
template <class T, bool E5M2>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a) {
  const int lane16 = threadIdx.x & 15, slot = threadIdx.x >> 4;
  const long long row0 = (long long)blockIdx.x * a.per_wg;
  const int j0 = blockIdx.y * 64, nj = min(64, a.kb - j0);
  const int rows = (int)min((long long)a.per_wg, a.rows - row0);
  const int tasks = a.kb > 64 ? nj : rows * a.kb;
  const T* x = (const T*)a.x + blockIdx.z * a.x_batch;
  float v[4][8];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int t = slot + 16 * u;
    if (t < tasks) {
      const int r = a.kb > 64 || a.kb == 1 ? (a.kb == 1 ? t : 0) : (int)__umulhi((unsigned)t, a.magic);
      const int j = a.kb > 64 ? j0 + t : t - r * a.kb;
      load_chunk(x + (row0 + r) * a.ldx, j * 128 + lane16 * 8, a.cols, a.wide_in, v[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int t = slot + 16 * u;
    if (t < tasks) {
      const int r = a.kb > 64 || a.kb == 1 ? (a.kb == 1 ? t : 0) : (int)__umulhi((unsigned)t, a.magic);
      const int j = a.kb > 64 ? j0 + t : t - r * a.kb;
      const float s = scale_of<E5M2>(largest_of_16_lanes(largest(v[u])));
      const long long row = (long long)blockIdx.z * a.rows + row0 + r;
      store_chunk(a.q + row * a.cols, j * 128 + lane16 * 8, a.cols, a.wide_out, quantize8<E5M2>(v[u], s));
      if (lane16 == 0) a.scale[row * a.kb + j] = s;
    }
  }
}

// Blocks of 128 x 128: one a workgroup, held in registers between the maximum and the division.
template <class T, bool E5M2>
__global__ __launch_bounds__(256) void quantize_square_kernel(QuantArgs a) {
  __shared__ float top[4];
  const int lane16 = threadIdx.x & 15, slot = threadIdx.x >> 4;
  const int mb = (a.rows + 127) / 128;
  const int bj = blockIdx.x % a.kb, bi = blockIdx.x / a.kb;
  const int c = bj * 128 + lane16 * 8;
  const T* x = (const T*)a.x + blockIdx.y * a.x_batch;
  float v[8][8], m = 0.0f;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int r = bi * 128 + slot + 16 * u;
    if (r < a.rows) {
      load_chunk(x + r * a.ldx, c, a.cols, a.wide_in, v[u]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[u][j] = 0.0f;
    }
  }
#pragma unroll
  for (int u = 0; u < 8; ++u) m = fmaxf(m, largest(v[u]));
  m = c2d_wave_max(m);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();
  const float s = scale_of<E5M2>(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int r = bi * 128 + slot + 16 * u;
    if (r < a.rows)
      store_chunk(a.q + ((long long)blockIdx.y * a.rows + r) * a.cols, c, a.cols, a.wide_out, quantize8<E5M2>(v[u], s));
  }
  if (threadIdx.x == 0) a.scale[((long long)blockIdx.y * mb + bi) * a.kb + bj] = s;
}

template <class T, bool E5M2>
int launch_quantize(QuantArgs a, int batch, int block_rows, hipStream_t stream) {
  if (block_rows == 1) {
    a.per_wg = a.kb >= 64 ? 1 : 64 / a.kb;
    const long long gx = ((long long)a.rows + a.per_wg - 1) / a.per_wg;
    const int gy = (a.kb + 63) / 64;
    if (gx >= (1ll << 31) || gy > 65535 || batch > 65535) return C2D_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((quantize_rows_kernel<T, E5M2>), dim3((unsigned)gx, gy, batch), dim3(256), 0, stream, a);
  } else {
    const long long gx = ((long long)a.rows + 127) / 128 * a.kb;
    if (gx >= (1ll << 31) || batch > 65535) return C2D_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((quantize_square_kernel<T, E5M2>), dim3((unsigned)gx, batch), dim3(256), 0, stream, a);
  }
  return c2d_launch_status();
}

}  // namespace

extern "C" int c2dp_fp8_quantize(const void* x, int x_type, long long ldx, long long x_batch, void* q, int q_type,
                                 float* scale, int batch, int rows, int cols, int block_rows, void* stream) {
  C2D_CHECK_ARG(x_type == C2DP_F32 || x_type == C2DP_BF16);
  C2D_CHECK_ARG(q_type == C2DP_E4M3 || q_type == C2DP_E5M2);
  C2D_CHECK_ARG(batch >= 0 && rows >= 0 && cols >= 0 && ldx >= cols && (block_rows == 1 || block_rows == 128));
  if (batch == 0 || rows == 0 || cols == 0) return C2D_OK;
  C2D_CHECK_ARG(x && q && scale);
  QuantArgs a;
  a.x = x;
  a.ldx = ldx;
  a.x_batch = x_batch;
  a.q = (unsigned char*)q;
  a.scale = scale;
  a.rows = rows;
  a.cols = cols;
  a.kb = (int)(((long long)cols + 127) / 128);
  a.per_wg = 0;
  a.magic = (unsigned)((0x100000000ull + a.kb - 1) / a.kb);
  const int es = x_type == C2DP_F32 ? 4 : 2;
  a.wide_in = aligned16(x, ldx * es) && (batch == 1 || x_batch * es % 16 == 0);
  a.wide_out = cols % 8 == 0 && ((unsigned long long)q & 7) == 0;
  const hipStream_t s = (hipStream_t)stream;
  if (es == 4)
    return q_type == C2DP_E5M2 ? launch_quantize<float, true>(a, batch, block_rows, s)
                               : launch_quantize<float, false>(a, batch, block_rows, s);
  return q_type == C2DP_E5M2 ? launch_quantize<__bf16, true>(a, batch, block_rows, s)
                             : launch_quantize<__bf16, false>(a, batch, block_rows, s);
}

// ---- product ----------------------------------------------------------------------------------------
//
// y = act(sum_c a_scale[.][c] b_scale[.][c] (a_c . b_c) + bias), c the blocks of 128 k.  A stage of the
// operand tiles is one block c: two v_mfma_f32_32x32x64_f8f6f4 from zero, then one multiply-add per sum with
// the block's scale.  A lane's sums lie in ONE row of the result (products_common.h), so that
// the scale is one number per lane and tile.

namespace {

struct Fp8Args {
  const char* a;
  long long lda;
  const float* a_scale;
  const char* b;
  const float* b_scale;
  const int* offsets;
  const float* bias;
  char* y;
  long long ldy;
  int groups, rows, n, k, kb, nb;
  int ntiles, wide, clear, relu;
};

// 32 rows from r0, 64 k of step s: chunks 4 s + 2 lh, + 1
__device__ __forceinline__ i32x8 fp8_frag(const char* t, int r0, int s) {
  const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
  const char* p = t + (r0 + li) * 128;
  const int x = (li >> 1) & 7;
  const i32x4 lo = *(const i32x4*)(p + (((4 * s + 2 * lh) ^ x) << 4));
  const i32x4 hi = *(const i32x4*)(p + (((4 * s + 2 * lh + 1) ^ x) << 4));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <bool E5M2>
__device__ __forceinline__ f32x16 fp8_mfma(i32x8 b, i32x8 a, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, c, 0, E5M2 ? 1 : 0, 0, 0, 0, 0);
}

template <bool E5M2, int WM, int WN, int MT, int NT, bool VEC, bool OUT16>
__global__ __launch_bounds__(WM * WN * 64) void fp8_tile_kernel(Fp8Args a) {
  constexpr int BM = WM * MT * 32, BN = WN * NT * 32, NTH = WM * WN * 64;
  typedef Tile<1, false, BM, NTH, VEC> TA;
  typedef Tile<1, false, BN, NTH, VEC> TB;
  constexpr int STAGE = TA::BYTES + TB::BYTES;
  static_assert(NT * 32 <= 128, "a wave's columns share a block of b");
  __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
  typedef typename std::conditional<OUT16, __bf16, float>::type out_t;
  const Place p = place_tile<BM>(a.offsets, a.groups, a.rows, a.ntiles, blockIdx.x, gridDim.x);
  if (!p.live) {
    if (a.clear) clear_rest(p, (out_t*)a.y, a.ldy, a.rows, a.n, NTH);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
  const int n0 = p.nt * BN;
  TA ta;
  TB tb;
  ta.begin(a.a + (long long)p.m0 * a.lda, a.lda, p.hi - p.m0, a.k);
  tb.begin(a.b + ((long long)p.e * a.n + n0) * a.k, a.k, a.n - n0, a.k);
  // scales: one row each for this lane's MT rows, one block of columns for the wave
  const float* as[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    as[i] = a.a_scale + (long long)min(p.m0 + (wm * MT + i) * 32 + li, p.hi - 1) * a.kb;
  const float* const bs = a.b_scale + ((long long)p.e * a.nb + min((n0 + wn * NT * 32) >> 7, a.nb - 1)) * a.kb;

  f32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  float scale[MT];
  if (a.kb > 0) {
    ta.issue(smem, 0);
    tb.issue(smem + TA::BYTES, 0);
#pragma unroll
    for (int i = 0; i < MT; ++i) scale[i] = as[i][0] * bs[0];
  }
  for (int it = 0; it < a.kb; ++it) {
    char* const now = smem + (it & 1) * STAGE;
    char* const next = smem + (~it & 1) * STAGE;
    float s_now[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) s_now[i] = scale[i];
    stage_barrier();
    if (it + 1 < a.kb) {
      ta.issue(next, it + 1);
      tb.issue(next + TA::BYTES, it + 1);
#pragma unroll
      for (int i = 0; i < MT; ++i) scale[i] = as[i][it + 1] * bs[it + 1];
    }
    const char* const sa = now + wm * MT * 32 * 128;
    const char* const sb = now + TA::BYTES + wn * NT * 32 * 128;
    i32x8 fb[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) { fb[j][0] = fp8_frag(sb, j * 32, 0); fb[j][1] = fp8_frag(sb, j * 32, 1); }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const i32x8 f0 = fp8_frag(sa, i * 32, 0), f1 = fp8_frag(sa, i * 32, 1);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        f32x16 z;
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = 0.0f;
        z = fp8_mfma<E5M2>(fb[j][0], f0, z);
        z = fp8_mfma<E5M2>(fb[j][1], f1, z);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = fmaf(z[r], s_now[i], acc[i][j][r]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = n0 + (wn * NT + j) * 32;
    float add[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int c = n + 8 * (r >> 2) + 4 * lh + (r & 3);
      add[r] = a.bias && c < a.n ? a.bias[(long long)p.e * a.n + c] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = p.m0 + (wm * MT + i) * 32 + li;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float v = acc[i][j][r] + add[r];
        acc[i][j][r] = a.relu && v < 0.0f ? 0.0f : v;
      }
      store_tile<OUT16>(acc[i][j], m < p.hi && n < a.n ? (char*)((out_t*)a.y + m * a.ldy + n) : nullptr, a.n - n, a.wide);
    }
  }
}

template <bool E5M2, bool VEC, bool OUT16>
int launch_fp8(Fp8Args a, hipStream_t stream) {
  constexpr int BM = 128, BN = 128;
  a.ntiles = (a.n + BN - 1) / BN;
  const unsigned grid = place_grid(BM, a.groups, a.offsets != nullptr, a.rows, a.ntiles);
  if (!grid) return C2D_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((fp8_tile_kernel<E5M2, 2, 2, 2, 2, VEC, OUT16>), dim3(grid), dim3(256), 0, stream, a);
  return c2d_launch_status();
}

}  // namespace

extern "C" unsigned long long c2dp_fp8_matmul_workspace_bytes(int groups, int rows, int n, int k) {
  (void)groups; (void)rows; (void)n; (void)k;
  return 0;
}

extern "C" int c2dp_fp8_matmul(const void* a_, int a_type, long long lda, const float* a_scale, const void* b,
                               const float* b_scale, const int32_t* offsets, int groups, const float* bias, int relu,
                               void* y, int y_type, long long ldy, int rows, int n, int k, int clear_rest,
                               void* workspace, unsigned long long workspace_bytes, void* stream) {
  C2D_CHECK_ARG(a_type == C2DP_E4M3 || a_type == C2DP_E5M2);
  C2D_CHECK_ARG(y_type == C2DP_F32 || y_type == C2DP_BF16);
  C2D_CHECK_ARG(groups > 0 && (offsets || groups == 1) && rows >= 0 && n >= 0 && k >= 0 && lda >= k && ldy >= n);
  if (rows == 0 || n == 0) return C2D_OK;
  C2D_CHECK_ARG(y && (k == 0 || (a_ && b && a_scale && b_scale)));
  if (lda > C2DP_MAX_PITCH || k > C2DP_MAX_PITCH) return C2D_ERR_UNSUPPORTED;
  (void)workspace; (void)workspace_bytes;
  Fp8Args a;
  a.a = (const char*)a_;
  a.lda = lda;
  a.a_scale = a_scale;
  a.b = (const char*)b;
  a.b_scale = b_scale;
  a.offsets = offsets;
  a.bias = bias;
  a.y = (char*)y;
  a.ldy = ldy;
  a.groups = groups;
  a.rows = rows;
  a.n = n;
  a.k = k;
  a.kb = (k + 127) / 128;
  a.nb = (n + 127) / 128;
  a.wide = aligned16(y, ldy * (y_type == C2DP_BF16 ? 2 : 4));
  a.clear = clear_rest;
  a.relu = relu;
  const bool vec = aligned16(a_, lda) && aligned16(b, k);
  const bool wide16 = y_type == C2DP_BF16;
  const hipStream_t s = (hipStream_t)stream;
  if (a_type == C2DP_E5M2) {
    if (wide16) return vec ? launch_fp8<true, true, true>(a, s) : launch_fp8<true, false, true>(a, s);
    return vec ? launch_fp8<true, true, false>(a, s) : launch_fp8<true, false, false>(a, s);
  }
  if (wide16) return vec ? launch_fp8<false, true, true>(a, s) : launch_fp8<false, false, true>(a, s);
  return vec ? launch_fp8<false, true, false>(a, s) : launch_fp8<false, false, false>(a, s);
}
