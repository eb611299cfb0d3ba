// Products of few rows or few tiles: D[m][n] = sum_k A[m][k] * B[n][k], both with the contraction contiguous,
// without LDS staging.
//
// A workgroup makes a tile of 16 MT rows by 16 NT columns; its KW waves take every KW-th segment of 128 bytes
// of the contraction and add their sums through LDS at the end.  A wave loads fragments straight into
// registers: 16 rows by 64 bytes an instruction, one segment ahead of the one it multiplies.  What bounds such a
// call is the weights' way from HBM and the latency of a chain of loads; splitting the contraction over
// the waves of a workgroup makes that chain 1 / KW as long and fills the chip where there are few column
// tiles, with no second pass over partial sums in memory.
#pragma once
#include "products_common.h"

namespace c2d_pr {
namespace {

// What is multiplied: 8-bit operands on the 8-bit matrix instructions, 8-bit operands widened to bf16 (exact;
// see fp8.hip), bf16, fp32.
enum Kind { FP8 = 0, FP8_WIDE = 1, BF16 = 2, F32 = 3 };
constexpr int elem_size(int kind) { return kind == BF16 ? 2 : kind == F32 ? 4 : 1; }

template <bool E5M2>
__device__ __forceinline__ bf16x2 widen2(int w, bool high) {
  if constexpr (E5M2)
    return high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, false);
  else
    return high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
}
// eight 8-bit values as bf16
template <bool E5M2>
__device__ __forceinline__ bf16x8 widen8(int lo, int hi) {
  const bf16x2 a = widen2<E5M2>(lo, false), b = widen2<E5M2>(lo, true), c = widen2<E5M2>(hi, false), d = widen2<E5M2>(hi, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 16 columns (first operand) by 16 rows, the two 16-byte chunks that a lane holds of a segment.
template <int KIND, bool E5M2>
__device__ __forceinline__ f32x4 mul_segment(const u32x4 (&b)[2], const u32x4 (&a)[2], f32x4 c) {
  if constexpr (KIND == FP8) {
    const i32x8 fb = __builtin_shufflevector(__builtin_bit_cast(i32x4, b[0]), __builtin_bit_cast(i32x4, b[1]), 0, 1, 2, 3, 4, 5, 6, 7);
    const i32x8 fa = __builtin_shufflevector(__builtin_bit_cast(i32x4, a[0]), __builtin_bit_cast(i32x4, a[1]), 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb, fa, c, 0, E5M2 ? 1 : 0, 0, 0, 0, 0);
  } else if constexpr (KIND == FP8_WIDE) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8<false>(b[h][0], b[h][1]), widen8<E5M2>(a[h][0], a[h][1]), c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8<false>(b[h][2], b[h][3]), widen8<E5M2>(a[h][2], a[h][3]), c, 0, 0, 0);
    }
    return c;
  } else if constexpr (KIND == BF16) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b[h]), __builtin_bit_cast(bf16x8, a[h]), c, 0, 0, 0);
    return c;
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 fb = __builtin_bit_cast(f32x4, b[h]), fa = __builtin_bit_cast(f32x4, a[h]);
#pragma unroll
      for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[q], fa[q], c, 0, 0, 0);
    }
    return c;
  }
}

struct FewArgs {
  const char* a;
  long long lda;                 // bytes
  const char* b;
  long long ldb, b_group;        // bytes
  const float *a_scale, *b_scale, *bias;
  const int* offsets;
  char* y;
  long long ldy;                 // elements
  int groups, rows, n, k, kb, nb;
  int ntiles, slots, clear, relu;
};

// One 16-byte chunk of a segment; zeros behind the contraction's end.
template <bool VEC, int ES>
__device__ __forceinline__ u32x4 few_load(__amdgpu_buffer_rsrc_t rs, const char* row, unsigned off, int at, int bytes) {
  if constexpr (VEC) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(at < bytes ? off + at : OUTSIDE), 0, 0);
    return __builtin_bit_cast(u32x4, v);
  } else {
    unsigned char v[16];
    if (at + 16 <= bytes) {
      __builtin_memcpy(v, row + at, 16);
    } else
#pragma unroll
    for (int j = 0; j < 16; j += ES) {
      const bool in = at + j < bytes;
      if constexpr (ES == 1) {
        v[j] = in ? *(const unsigned char*)(row + at + j) : 0;
      } else if constexpr (ES == 2) {
        const unsigned short e = in ? *(const unsigned short*)(row + at + j) : 0;
        __builtin_memcpy(v + j, &e, 2);
      } else {
        const unsigned e = in ? *(const unsigned*)(row + at + j) : 0;
        __builtin_memcpy(v + j, &e, 4);
      }
    }
    u32x4 o;
    __builtin_memcpy(&o, v, 16);
    return o;
  }
}

template <int KIND, bool E5M2, int MT, int NT, int KW, bool VEC, bool OUT16>
__global__ __launch_bounds__(KW * 64) void few_rows_kernel(FewArgs p) {
  constexpr int ES = elem_size(KIND), BM = 16 * MT, BN = 16 * NT;
  constexpr bool SCALED = KIND == FP8 || KIND == FP8_WIDE;
  typedef typename std::conditional<OUT16, __bf16, float>::type out_t;
  constexpr int PITCH = BN + 4;  // floats; 16-byte aligned rows, rows four banks apart
  __shared__ __attribute__((aligned(16))) float part[KW][BM][PITCH];
  const Place pl = place_tile<BM, false>(p.offsets, p.groups, p.rows, p.ntiles, workgroup(), workgroups(), 1);
  if (!pl.live) {
    if (p.clear) clear_rest(pl, (out_t*)p.y, p.ldy, p.rows, p.n, KW * 64);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int l16 = lane & 15, q = lane >> 4;
  const int n0 = pl.nt * BN, bytes = p.k * ES;
  const int segments = (bytes + 127) >> 7;
  const char* const a0 = p.a + (long long)pl.m0 * p.lda;
  const char* const b0 = p.b + pl.e * p.b_group + n0 * p.ldb;
  const int a_rows = min(BM, pl.hi - pl.m0), b_rows = min(BN, p.n - n0);
  const __amdgpu_buffer_rsrc_t ra = buffer_of(a0, (a_rows - 1) * p.lda + bytes), rb = buffer_of(b0, (b_rows - 1) * p.ldb + bytes);
  unsigned a_off[MT], b_off[NT];
  const float* as[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = min(16 * i + l16, a_rows - 1);
    a_off[i] = (unsigned)(r * (int)p.lda);
    if (SCALED) as[i] = p.a_scale + (long long)(pl.m0 + r) * p.kb;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) b_off[j] = (unsigned)(min(16 * j + l16, b_rows - 1) * (int)p.ldb);
  const float* const bs = SCALED ? p.b_scale + ((long long)pl.e * p.nb + (n0 >> 7)) * p.kb : nullptr;

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  struct Segment { u32x4 a[MT][2], b[NT][2]; float s[MT], sb; };
  auto load = [&](Segment& g, int c) {
    const int at = (c << 7) + (q << 4);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) g.b[j][h] = few_load<VEC, ES>(rb, b0 + b_off[j], b_off[j], at + 64 * h, bytes);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) g.a[i][h] = few_load<VEC, ES>(ra, a0 + a_off[i], a_off[i], at + 64 * h, bytes);
    if constexpr (SCALED) {
      g.sb = bs[c];
#pragma unroll
      for (int i = 0; i < MT; ++i) g.s[i] = as[i][c];
    }
  };
  auto multiply = [&](const Segment& g) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if constexpr (SCALED) {
          const f32x4 z = mul_segment<KIND, E5M2>(g.b[j], g.a[i], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
          const float s = g.s[i] * g.sb;
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(z[r], s, acc[i][j][r]);
        } else {
          acc[i][j] = mul_segment<KIND, E5M2>(g.b[j], g.a[i], acc[i][j]);
        }
      }
  };
  // (U segments in flight while U are multiplied: more where a segment is small)
  constexpr int U = MT == 1 ? 2 : 1;
  Segment g[2][U];
  int c = wave;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c + u * KW < segments) load(g[0][u], c + u * KW);
  for (; c < segments; c += 2 * U * KW) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int now = c + h * U * KW, next = now + U * KW;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (next + u * KW < segments) load(g[h ^ 1][u], next + u * KW);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (now + u * KW < segments) multiply(g[h][u]);
    }
  }

  // a lane holds row 16 i + l16, columns 16 j + 4 q + 0..3
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) *(f32x4*)&part[wave][16 * i + l16][16 * j + 4 * q] = acc[i][j];
  __syncthreads();
  // the sums in the waves' order; BN / 4 lanes a row, four columns each
  for (int t = threadIdx.x; t < BM * (BN / 4); t += KW * 64) {
    const int m = t / (BN / 4), col = (t % (BN / 4)) * 4;
    if (m >= a_rows) break;
    f32x4 v = *(const f32x4*)&part[0][m][col];
#pragma unroll
    for (int w = 1; w < KW; ++w) v += *(const f32x4*)&part[w][m][col];
    const int n = n0 + col;
    if (p.bias) {
      const float* const bias = p.bias + (long long)pl.e * p.n + n;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += n + r < p.n ? bias[r] : 0.0f;
    }
    if (p.relu) {
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = v[r] < 0.0f ? 0.0f : v[r];
    }
    out_t* const y = (out_t*)p.y + (long long)(pl.m0 + m) * p.ldy + n;
    if (n + 4 <= p.n) {
      if constexpr (OUT16) store_at((char*)y, u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])});
      else store_at((char*)y, v);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < p.n) y[r] = (out_t)v[r];
    }
  }
}

template <int KIND, bool E5M2, int MT, int NT, int KW, bool VEC, bool OUT16>
int launch_few(FewArgs p, hipStream_t stream) {
  p.ntiles = (p.n + 16 * NT - 1) / (16 * NT);
  const unsigned grid = place_grid(16 * MT, p.groups, p.offsets != nullptr, p.rows, p.ntiles, 0);
  if (!grid) return C2D_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((few_rows_kernel<KIND, E5M2, MT, NT, KW, VEC, OUT16>), grid_of(grid), dim3(KW * 64), 0, stream, p);
  return c2d_launch_status();
}

}  // namespace
}  // namespace c2d_pr
