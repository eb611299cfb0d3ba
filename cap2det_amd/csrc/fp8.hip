// 8-bit floating-point storage: the block quantiser and the product of block-scaled matrices, for one
// weight matrix or one per group of rows.
#include "products_few.h"

using namespace c2d_pr;

namespace {

// ---- quantiser --------------------------------------------------------------------------------------
//
// s = max(max |x| / F, 2^-126), scale = s as fp32, q = rne8(x / s), rounded once: x / scale as fp32 lies on another side of
// a tie than x / s in about one of a million values, which is then a whole step off.  |x| <= F s, so nothing
// overflows the type.

// (any address)
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  f32x4 a, b;
  __builtin_memcpy(&a, p, 16);
  __builtin_memcpy(&b, p + 4, 16);
#pragma unroll
  for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
}
__device__ __forceinline__ void load8(const __bf16* p, float (&v)[8]) {
  bf16x8 a;
  __builtin_memcpy(&a, p, 16);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
}

// eight elements of a row from column c, zeros behind the last
template <class T>
__device__ __forceinline__ void load_chunk(const T* row, int c, int cols, float (&v)[8]) {
  if (c + 8 <= cols) {
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
constexpr float LARGEST = E5M2 ? 57344.0f : 448.0f;  // F = 7 * 2^i

template <bool E5M2>
__device__ __forceinline__ float scale_of(float m) {
  return fmaxf(m / LARGEST<E5M2>, 0x1p-126f);
}

template <bool E5M2>
__device__ __forceinline__ u32x2 to_8_bits(const float (&q)[8]) {
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

// x / s rounded so that its rounding to 8 bits is that of the true quotient.  The quotient is t + c, t = x r and c its
// correction: the remainder x - t s, exact (one fused multiply-add), by r, and what the scale's rounding makes (rho).
// Their sum's own rounding leaves e, known to 2^-44 of the quotient: where there is one, the result is the odd one of
// the two fp32 numbers around the quotient, which lies on the same side of every tie as the quotient does.
template <bool E5M2>
__device__ __forceinline__ void quotients(const float (&v)[8], float m, float scale, float (&q)[8]) {
#pragma clang fp contract(off)  // (t is the rounded product in all of its uses)
  const float up = m < 0x1p-40f ? 0x1p80f : 1.0f;  // (no remainder is a denormal number)
  const float s = scale * up, r = 1.0f / s, top = m * up;
  const float rho = scale > 0x1p-126f ? fmaf(-s, LARGEST<E5M2>, top) / top : 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = v[j] * up, t = x * r;
    const float c = fmaf(-t, rho, fmaf(-t, s, x) * r);
    const float sum = t + c, e = c - (sum - t);
    int bits = __float_as_int(sum);
    if (fabsf(e) > 0x1p-40f * fabsf(sum) && !(bits & 1)) bits += (bits ^ __float_as_int(e)) < 0 ? -1 : 1;
    q[j] = __int_as_float(bits);
  }
}

// m: the block's largest |x|.
// bf16: a quotient is a tie, or 2^-13 of it or more away from one: X and M being whole numbers below 256, 7 X 2^i and
// T M differ by one or more, T < 32.  x * (1 / s) is within 2^-22 of it: rounded to 21 bits it is on the tie, or on its side.
// fp32: x by 1 / s made smaller and larger by 2^-21 are on either side of the quotient.  Where both round to the same
// it does too; where not, in one of some 10^5 random values, the quotient is made with care.
template <class T, bool E5M2>
__device__ __forceinline__ u32x2 quantize8(const float (&v)[8], float m, float scale) {
  const float r = scale < __builtin_inff() ? 1.0f / scale : __builtin_nanf("");  // (an infinity makes NaNs of its block)
  float q[8];
  if constexpr (std::is_same<T, __bf16>::value) {
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = __int_as_float((__float_as_int(v[j] * r) + 4) & ~7);
    return to_8_bits<E5M2>(q);
  } else {
    const float below = r * (1.0f - 0x1p-21f), above = r * (1.0f + 0x1p-21f);
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = v[j] * below;
    const u32x2 o = to_8_bits<E5M2>(q);
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = v[j] * above;
    const u32x2 p = to_8_bits<E5M2>(q);
    if (o[0] == p[0] && o[1] == p[1]) return o;
    quotients<E5M2>(v, m, scale, q);
    return to_8_bits<E5M2>(q);
  }
}

__device__ __forceinline__ void store_chunk(unsigned char* row, int c, int cols, u32x2 q) {
  if (c + 8 <= cols) {
    store_at((char*)row + c, q);
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
  int rows, cols, kb;
  int span, per_wg;            // 1 x 128 blocks, and rows, of a workgroup
  int row_wg, col_wg, batch0;  // where this launch begins: workgroups along the rows and the columns, matrix of the stack
  unsigned magic;              // ceil(2^32 / kb): t / kb = umulhi(t, magic) for t < 2^16
};

// Blocks of 1 x 128: 16 lanes a block, 8 elements a lane, `span` blocks a workgroup (64; 32 or 16 where that many would
// leave CUs without work), all of whose loads are issued before the first is used.  What bounds it is memory: 32768 x
// 8192 bf16 in 147 us in a replayed graph and 150-174 launched one by one (5.5 and 4.6-5.4 TB/s of twice as much read as
// written, where a copy reaches 5.15).
template <class T, bool E5M2>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a) {
  const int lane16 = threadIdx.x & 15, slot = threadIdx.x >> 4;
  const long long row0 = (long long)(a.row_wg + blockIdx.x) * a.per_wg, matrix = a.batch0 + blockIdx.z;
  const bool wide = a.kb > a.span;  // a row is several workgroups'
  const int j0 = (a.col_wg + blockIdx.y) * a.span, nj = min(a.span, a.kb - j0);
  const int rows = (int)min((long long)a.per_wg, a.rows - row0);
  const int tasks = wide ? nj : rows * a.kb;
  const T* x = (const T*)a.x + matrix * a.x_batch;
  float v[4][8];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int t = slot + 16 * u;
    if (t < tasks) {
      const int r = wide ? 0 : a.kb == 1 ? t : (int)__umulhi((unsigned)t, a.magic);
      const int j = wide ? j0 + t : t - r * a.kb;
      load_chunk(x + (row0 + r) * a.ldx, j * 128 + lane16 * 8, a.cols, v[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int t = slot + 16 * u;
    if (t < tasks) {
      const int r = wide ? 0 : a.kb == 1 ? t : (int)__umulhi((unsigned)t, a.magic);
      const int j = wide ? j0 + t : t - r * a.kb;
      const float m = largest_of_16_lanes(largest(v[u])), s = scale_of<E5M2>(m);
      const long long row = matrix * a.rows + row0 + r;
      store_chunk(a.q + row * a.cols, j * 128 + lane16 * 8, a.cols, quantize8<T, E5M2>(v[u], m, s));
      if (lane16 == 0) a.scale[row * a.kb + j] = s;
    }
  }
}

// Blocks of 128 x 128: one a workgroup, held in registers between the maximum and the division, U chunks of 8
// elements a thread (8; 2 where the blocks are fewer than CUs: 300 x 300 fp32 3.7 us, with 8 6.5).
template <class T, bool E5M2, int U>
__global__ __launch_bounds__(2048 / U) void quantize_square_kernel(QuantArgs a) {
  constexpr int STEP = 128 / U, WAVES = 32 / U;
  __shared__ float top[WAVES];
  const int lane16 = threadIdx.x & 15, slot = threadIdx.x >> 4;
  const int mb = (a.rows + 127) / 128;
  const int bj = blockIdx.x % a.kb, bi = blockIdx.x / a.kb;
  const int c = bj * 128 + lane16 * 8;
  const long long matrix = a.batch0 + blockIdx.y;
  const T* x = (const T*)a.x + matrix * a.x_batch;
  float v[U][8], m = 0.0f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = bi * 128 + slot + STEP * u;
    if (r < a.rows) {
      load_chunk(x + r * a.ldx, c, a.cols, v[u]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[u][j] = 0.0f;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) m = fmaxf(m, largest(v[u]));
  m = c2d_wave_max(m);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) m = fmaxf(m, top[w]);
  const float s = scale_of<E5M2>(m);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = bi * 128 + slot + STEP * u;
    if (r < a.rows)
      store_chunk(a.q + (matrix * a.rows + r) * a.cols, c, a.cols, quantize8<T, E5M2>(v[u], m, s));
  }
  if (threadIdx.x == 0) a.scale[(matrix * mb + bi) * a.kb + bj] = s;
}

// A launch holds fewer than 2^32 threads along x and 2^16 workgroups along y and z: what is larger goes in several.
template <class T, bool E5M2>
int launch_quantize(QuantArgs a, int batch, int block_rows, hipStream_t stream) {
  constexpr long long X = 1 << 22, YZ = 65535;
  auto least = [](long long n, long long most) { return (unsigned)(n < most ? n : most); };
  if (block_rows == 1) {
    const double blocks = (double)batch * a.rows * a.kb;
    a.span = blocks >= 64 * 512 ? 64 : blocks >= 32 * 512 ? 32 : 16;
    a.per_wg = a.kb >= a.span ? 1 : a.span / a.kb;
    const long long gx = ((long long)a.rows + a.per_wg - 1) / a.per_wg, gy = (a.kb + a.span - 1) / a.span;
    for (long long z = 0; z < batch; z += YZ)
      for (long long y = 0; y < gy; y += YZ)
        for (long long x = 0; x < gx; x += X) {
          a.row_wg = (int)x;
          a.col_wg = (int)y;
          a.batch0 = (int)z;
          hipLaunchKernelGGL((quantize_rows_kernel<T, E5M2>), dim3(least(gx - x, X), least(gy - y, YZ), least(batch - z, YZ)),
                             dim3(256), 0, stream, a);
          if (c2d_launch_status() != C2D_OK) return C2D_ERR_LAUNCH;
        }
    return C2D_OK;
  }
  const long long gx = ((long long)a.rows + 127) / 128 * a.kb;
  if (gx >= (1ll << 24)) return C2D_ERR_UNSUPPORTED;  // (415 GB and more of one bf16 matrix and its values)
  for (long long z = 0; z < batch; z += YZ) {
    a.batch0 = (int)z;
    const dim3 grid((unsigned)gx, least(batch - z, YZ));
    if (gx * batch < c2d_available_cus())
      hipLaunchKernelGGL((quantize_square_kernel<T, E5M2, 2>), grid, dim3(1024), 0, stream, a);
    else
      hipLaunchKernelGGL((quantize_square_kernel<T, E5M2, 8>), grid, dim3(256), 0, stream, a);
    if (c2d_launch_status() != C2D_OK) return C2D_ERR_LAUNCH;
  }
  return C2D_OK;
}

}  // namespace

extern "C" int c2dp_fp8_quantize(const void* x, int x_type, long long ldx, long long x_batch, void* q, int q_type,
                                 float* scale, int batch, int rows, int cols, int block_rows, void* stream) {
  C2D_CHECK_ARG(x_type == C2DP_F32 || x_type == C2DP_BF16);
  C2D_CHECK_ARG(q_type == C2DP_E4M3 || q_type == C2DP_E5M2);
  C2D_CHECK_ARG(batch >= 0 && rows >= 0 && cols >= 0 && ldx >= cols && (block_rows == 1 || block_rows == 128));
  if (batch == 0 || rows == 0 || cols == 0) return C2D_OK;
  C2D_CHECK_ARG(x && q && scale);
  if (!sizes_fit(batch, rows, cols)) return C2D_ERR_UNSUPPORTED;
  QuantArgs a;
  a.x = x;
  a.ldx = ldx;
  a.x_batch = x_batch;
  a.q = (unsigned char*)q;
  a.scale = scale;
  a.rows = rows;
  a.cols = cols;
  a.kb = (int)(((long long)cols + 127) / 128);
  a.span = a.per_wg = a.row_wg = a.col_wg = a.batch0 = 0;
  a.magic = (unsigned)((0x100000000ull + a.kb - 1) / a.kb);
  const int es = x_type == C2DP_F32 ? 4 : 2;
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
// operand tiles is one block c: its products are summed from zero, then one multiply-add per sum with the
// block's scale.  A lane's sums lie in ONE row of the result (products_common.h), so that the scale is one
// number per lane and tile.
//
// The 8-bit matrix instructions (every shape of them) add the products of 8 consecutive k with each cut off, towards zero, at
// 2^-13 of 2^e, e the largest sum of two factors' exponents among the products that are not zero, a denormal factor's
// exponent being its type's least; those sums are added in fp32 (measured, from products beside larger ones that cancel:
// 2^-13 of a larger one in the same 8 is kept and 2^-14 lost, in another 8 2^-23).  A product of two normal values
// has 6 bits behind its point or fewer: one whose exponents are up to 7 below the largest loses nothing.  That is
// 1.4e-5 of a block's sum for normal values, and 7 * 2^-13 of the largest product of each 8 at most, where
// the operands' own rounding is 2^-4 of each value: a bf16 result, which is rounded to 2^-8, takes them.  For an fp32 result
// the fragments are widened to bf16, which holds every 8-bit value exactly, and go through the bf16 matrix instructions, whose
// sums are fp32 (2e-7; 2^-23 of any larger product is kept), at half the rate.

namespace {

// 32 rows from r0 of a stage: chunks 2 c + lh, c = C0 .. C1 - 1, of a lane's row
template <int C0, int C1>
__device__ __forceinline__ void fp8_load(const char* t, int r0, i32x4 (&f)[4]) {
  const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
  const char* p = t + (r0 + li) * 128;
  const int x = (li >> 1) & 7;
#pragma unroll
  for (int c = C0; c < C1; ++c) f[c] = *(const i32x4*)(p + (((2 * c + lh) ^ x) << 4));
}

// half a stage's products (64 k) of 32 columns and 32 rows, added to z
template <bool E5M2, bool WIDE>
__device__ __forceinline__ f32x16 fp8_half(const i32x4 (&b)[4], const i32x4 (&a)[4], int h, f32x16 z) {
  if constexpr (WIDE) {
#pragma unroll
    for (int c = 2 * h; c < 2 * h + 2; ++c) {
      z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen8<false>(b[c][0], b[c][1]), widen8<E5M2>(a[c][0], a[c][1]), z, 0, 0, 0);
      z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen8<false>(b[c][2], b[c][3]), widen8<E5M2>(a[c][2], a[c][3]), z, 0, 0, 0);
    }
    return z;
  } else {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
        __builtin_shufflevector(b[2 * h], b[2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7),
        __builtin_shufflevector(a[2 * h], a[2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7), z, 0, E5M2 ? 1 : 0, 0, 0, 0, 0);
  }
}

// The stages of A go round D buffers, those of B round D + 1: while a stage is multiplied, the next of A and
// the next two of B are on their way (D = 2; five buffers are what the LDS holds of 256 x 256 tiles).  Within a
// stage the loads are issued between the matrix instructions of its first tiles, and a tile's scaling runs under
// the matrix instructions of the next: 8192^3 in 493-515 us in a replayed graph, 517-537 launched one by one (2180 and 2090
// TFLOP/s; in the first 10 ms of such a load up to 655), where the library's product with one scale for the whole matrix reaches
// 2680-2790; with the loads in front and the scaling behind its own products 652.  The
// matrix pipe is busy 55 % of that time, LDS 22 %: the wait at the stages' barriers is what is left.
//
// KG > 1: KG groups of WM x WN waves share the tile, group g taking the stages g, g + KG, ..; their sums are
// joined through LDS, in the groups' order.  A stage of a small tile is a chain of waits (barrier, LDS read, two
// matrix instructions, scaling) of 0.5 us whatever its size (64 x 64 tiles): where there is a workgroup per CU
// or less, KG chains run side by side (256 x 4096 x 4096: 17.6 us, with two groups 13.6, with four 14.6).
template <bool E5M2, int WM, int WN, int MT, int NT, int KG, int D, bool VEC>
struct Fp8Tiles {
  static constexpr int BM = WM * MT * 32, BN = WN * NT * 32, NTH = WM * WN * 64, DA = D, DB = D + 1, TILES = MT * NT;
  typedef Tile<1, false, BM, NTH, VEC> TA;
  typedef Tile<1, false, BN, NTH, VEC> TB;
  static constexpr int PASSES = TA::LOADS + TB::LOADS;
  static constexpr int RING = DA * TA::BYTES + DB * TB::BYTES;
  static_assert(128 % (NT * 32) == 0, "a wave's columns share a block of b");
  static_assert(KG == 1 || (KG - 1) * NTH * 64 <= KG * RING, "the sums are joined a tile at a time in the ring's LDS");
};

// A row tile (`p`) of BM rows or less.
template <bool E5M2, int WM, int WN, int MT, int NT, int KG, int D, bool VEC, bool OUT16>
__device__ __forceinline__ void fp8_tile(const FewArgs& a, const Place& p, char* smem, int group, int tid) {
  typedef Fp8Tiles<E5M2, WM, WN, MT, NT, KG, D, VEC> C;
  constexpr int BN = C::BN, NTH = C::NTH, DA = C::DA, DB = C::DB, TILES = C::TILES, PASSES = C::PASSES, RING = C::RING;
  typedef typename C::TA TA;
  typedef typename C::TB TB;
  typedef typename std::conditional<OUT16, __bf16, float>::type out_t;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
  const int n0 = p.nt * BN;
  char* const ring_a = smem + group * RING;
  char* const ring_b = ring_a + DA * TA::BYTES;
  TA ta;
  TB tb;
  ta.begin(a.a + (long long)p.m0 * a.lda, a.lda, p.hi - p.m0, a.k, tid);
  tb.begin(a.b + p.e * a.b_group + n0 * a.ldb, a.ldb, a.n - n0, a.k, tid);
  // scales: one row each for this lane's MT rows, one block of columns for the wave
  const float* const as = a.a_scale + (long long)p.m0 * a.kb;
  unsigned as_at[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) as_at[i] = (unsigned)(min((wm * MT + i) * 32 + li, p.hi - 1 - p.m0) * a.kb);
  typedef __attribute__((address_space(4))) const float scalar_float;
  const scalar_float* const bs = (const scalar_float*)(unsigned long long)(
      a.b_scale + ((long long)p.e * a.nb + min((n0 + wn * NT * 32) >> 7, a.nb - 1)) * a.kb);

  f32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  const int rounds = (a.kb + KG - 1) / KG;
  float row_scale[MT], col_scale;
  auto load_scales = [&](int st) {
    const int c = min(st, a.kb - 1);
    col_scale = bs[c];
#pragma unroll
    for (int i = 0; i < MT; ++i) row_scale[i] = as[as_at[i] + (unsigned)c];
  };
  if (rounds > 0) {
    load_scales(group);
    tb.issue(ring_b, group);
#pragma unroll
    for (int d = 0; d < D - 1; ++d) {
      ta.issue(ring_a + d * TA::BYTES, d * KG + group);
      tb.issue(ring_b + (d + 1) * TB::BYTES, (d + 1) * KG + group);
    }
  }
  int now_a = 0, now_b = 0, next_a = DA - 1, next_b = DB - 1;
  for (int it = 0; it < rounds; ++it) {
    // (behind this stage's A have been issued: B of the next, and D - 2 whole stages)
    stage_barrier<VEC, TB::LOADS + (D - 2) * PASSES>();
    float scale[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i)  // (a group's stage behind the last is zeros, which no scale may make a NaN)
      scale[i] = KG > 1 && it * KG + group >= a.kb ? 0.0f : row_scale[i] * col_scale;
    load_scales((it + 1) * KG + group);  // in front of the loads to LDS
    const int st_a = (it + DA - 1) * KG + group, st_b = (it + DB - 1) * KG + group;
    const typename TA::Stage ga = ta.at(st_a);
    const typename TB::Stage gb = tb.at(st_b);
    const char* const sa = ring_a + now_a * TA::BYTES;
    const char* const sb = ring_b + now_b * TB::BYTES;
    i32x4 fa[MT][4], fb[4];
    fp8_load<0, 4>(sb, wn * NT * 32, fb);
#pragma unroll
    for (int i = 0; i < MT; ++i) fp8_load<0, 4>(sa, (wm * MT + i) * 32, fa[i]);
    f32x16 z[2], zero;
#pragma unroll
    for (int r = 0; r < 16; ++r) zero[r] = 0.0f;
    // tiles in the order (j, i), j the slow one; u: the tile whose products are taken while t is scaled
#pragma unroll
    for (int u = 0; u <= TILES; ++u) {
      const int t = u - 1, i = u % MT, j = u / MT;
      constexpr int PER = (2 * PASSES + TILES - 1) / TILES;  // passes a tile, in the first half of the tiles
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (u < TILES) {
          z[u & 1] = fp8_half<E5M2, !OUT16>(fb, fa[i], h, h ? z[u & 1] : zero);
          // the last use of this half of the column fragment: the next one's takes its registers
          if (i == MT - 1 && j + 1 < NT) {
            __builtin_amdgcn_sched_barrier(0);
            if (h == 0) fp8_load<0, 2>(sb, (wn * NT + j + 1) * 32, fb);
            else fp8_load<2, 4>(sb, (wn * NT + j + 1) * 32, fb);
          }
        }
        if (t >= 0) {
#pragma unroll
          for (int r = 8 * h; r < 8 * h + 8; ++r) acc[t % MT][t / MT][r] = fmaf(z[t & 1][r], scale[t % MT], acc[t % MT][t / MT][r]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int q = u * PER; q < (u + 1) * PER && q < PASSES; ++q) {
        if (q < TA::LOADS) ta.pass(ring_a + next_a * TA::BYTES, ga, st_a, q);
        else tb.pass(ring_b + next_b * TB::BYTES, gb, st_b, q - TA::LOADS);
      }
    }
    now_a = now_a + 1 == DA ? 0 : now_a + 1;
    next_a = next_a + 1 == DA ? 0 : next_a + 1;
    now_b = now_b + 1 == DB ? 0 : now_b + 1;
    next_b = next_b + 1 == DB ? 0 : next_b + 1;
  }
  drain_loads();
  if constexpr (KG > 1) {
    join_groups<KG, NTH>((float*)smem, group, tid, acc);
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float add[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int c = n0 + (wn * NT + j) * 32 + 8 * (r >> 2) + 4 * lh + (r & 3);
      add[r] = a.bias && c < a.n ? a.bias[(long long)p.e * a.n + c] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float v = acc[i][j][r] + add[r];
        acc[i][j][r] = a.relu && v < 0.0f ? 0.0f : v;
      }
  }
  __syncthreads();
  if (group > 0) return;
  typedef Store<OUT16, NT> S;
  static_assert(NTH / 64 * S::BYTES <= RING, "the result goes out through the ring's LDS");
  const int m = p.m0 + wm * MT * 32, n = n0 + wn * NT * 32;
  S::run(acc, smem + wave * S::BYTES, (char*)((out_t*)a.y + m * a.ldy + n), a.ldy * (long long)sizeof(out_t), p.hi - m, a.n - n);
}

// A group's last tile is on average half full.  Half of it or less is multiplied as a tile of half the height.
template <bool E5M2, int WM, int WN, int MT, int NT, int KG, int D, bool VEC, bool OUT16>
__global__ __launch_bounds__(WM * WN * KG * 64, 2) void fp8_tile_kernel(FewArgs a) {
  typedef Fp8Tiles<E5M2, WM, WN, MT, NT, KG, D, VEC> C;
  __shared__ __attribute__((aligned(1024))) char smem[KG * C::RING];
  typedef typename std::conditional<OUT16, __bf16, float>::type out_t;
  const Place p = place_tile<C::BM, (MT > 1)>(a.offsets, a.groups, a.rows, a.ntiles, workgroup(), workgroups(), a.slots);
  if (!p.live) {
    if (a.clear) clear_rest(p, (out_t*)a.y, a.ldy, a.rows, a.n, C::NTH * KG);
    return;
  }
  const int group = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / C::NTH), tid = threadIdx.x - group * C::NTH;
  if constexpr (MT > 1) {
    if (p.hi - p.m0 <= C::BM / 2) {
      fp8_tile<E5M2, WM, WN, MT / 2, NT, KG, D, VEC, OUT16>(a, p, smem, group, tid);
      return;
    }
  }
  fp8_tile<E5M2, WM, WN, MT, NT, KG, D, VEC, OUT16>(a, p, smem, group, tid);
}

template <bool E5M2, int WM, int WN, int MT, int NT, int KG, int D, bool VEC, bool OUT16>
int launch_tiles(FewArgs a, hipStream_t stream) {
  constexpr int BM = WM * MT * 32, BN = WN * NT * 32;
  a.ntiles = (a.n + BN - 1) / BN;
  a.slots = slots_per_xcd(KG * Fp8Tiles<E5M2, WM, WN, MT, NT, KG, D, VEC>::RING);
  const unsigned grid = place_grid(BM, a.groups, a.offsets != nullptr, a.rows, a.ntiles, MT > 1 ? a.slots / 2 : 0);
  if (!grid) return C2D_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((fp8_tile_kernel<E5M2, WM, WN, MT, NT, KG, D, VEC, OUT16>), grid_of(grid), dim3(WM * WN * KG * 64), 0, stream, a);
  return c2d_launch_status();
}

template <bool E5M2, bool VEC, bool OUT16>
int launch_fp8(const FewArgs& a, hipStream_t stream) {
  constexpr int KIND = OUT16 ? FP8 : FP8_WIDE;
  switch (fp8_shape(a.rows, a.n, a.k, a.groups, a.offsets != nullptr, OUT16, VEC, c2d_available_cus())) {
    case T16: return launch_few<KIND, E5M2, 1, 1, 8, VEC, OUT16>(a, stream);
    case T16W: return launch_few<KIND, E5M2, 1, 2, 2, VEC, OUT16>(a, stream);
    case T32: return launch_few<KIND, E5M2, 2, 2, 8, VEC, OUT16>(a, stream);
    case T64: return launch_tiles<E5M2, 2, 2, 1, 1, 2, 4, VEC, OUT16>(a, stream);
    case T256:
      if constexpr (OUT16 && VEC) return launch_tiles<E5M2, 4, 2, 2, 4, 1, 2, true, true>(a, stream);
    default: return launch_tiles<E5M2, 2, 2, 2, 2, 1, 2, VEC, OUT16>(a, stream);
  }
}

}  // namespace

extern "C" int c2dp_fp8_matmul(const void* a_, int a_type, long long lda, const float* a_scale, const void* b,
                               const float* b_scale, const int32_t* offsets, int groups, const float* bias, int relu,
                               void* y, int y_type, long long ldy, int rows, int n, int k, int clear_rest,
                               void* stream) {
  C2D_CHECK_ARG(a_type == C2DP_E4M3 || a_type == C2DP_E5M2);
  C2D_CHECK_ARG(y_type == C2DP_F32 || y_type == C2DP_BF16);
  C2D_CHECK_ARG(groups > 0 && (offsets || groups == 1) && rows >= 0 && n >= 0 && k >= 0 && lda >= k && ldy >= n);
  if (rows == 0 || n == 0) return C2D_OK;
  C2D_CHECK_ARG(y && (k == 0 || (a_ && b && a_scale && b_scale)));
  if (!groups_fit(groups) || !sizes_fit(rows, n, k) || lda > C2DP_MAX_PITCH || k > C2DP_MAX_PITCH) return C2D_ERR_UNSUPPORTED;
  FewArgs a;
  a.a = (const char*)a_;
  a.lda = lda;
  a.a_scale = a_scale;
  a.b = (const char*)b;
  a.ldb = k;
  a.b_group = (long long)n * k;
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
