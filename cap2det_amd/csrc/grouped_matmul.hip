// Matrix products grouped by expert: the rows of x sorted by group, one weight matrix per group, the groups'
// lengths on the device.  Forward, input gradient and weight gradient, bf16 and fp32 operands, fp32 sums.
#include "products_common.h"

using namespace c2d_pr;
#ifndef XWM
#define XWM 2
#define XWN 2
#define XMT 2
#define XNT 2
#define XD 2
#endif

namespace {

struct RowsArgs {             // forward and input gradient: one row of the result per row of A
  const char* a;
  long long lda;              // bytes
  const char* w;
  long long ldw, w_group;     // bytes
  const int* offsets;
  char* y;
  long long ldy;              // elements
  int groups, rows, n, k;     // n: result columns, k: contraction
  int ntiles, clear;
};

struct WgradArgs {
  const char *dy, *x;
  long long lddy, ldx;        // bytes
  const int* offsets;
  float* dw;                  // [groups][n][k], or [splits][groups][n][k]
  int groups, rows, n, k;
  int ntiles, ktiles, splits, accumulate;
};

// A ring of D buffers, each a stage of A and B: while one is multiplied the next D - 1 are on their way.  One
// barrier per stage.  D[m][n], this wave's MT x NT tiles of 32 x 32.
template <int ES, bool TRA, bool TRB, int WM, int WN, int MT, int NT, int D, bool VEC>
struct Core {
  static constexpr int BM = WM * MT * 32, BN = WN * NT * 32, NTH = WM * WN * 64;
  typedef Tile<ES, TRA, BM, NTH, VEC> TA;
  typedef Tile<ES, TRB, BN, NTH, VEC> TB;
  static constexpr int STAGE = TA::BYTES + TB::BYTES;
  static constexpr int KST = TA::KST;

  // fragment of 32 rows (TR: columns) from `r0`, k-step s, for a lane
  template <bool TR, int R>
  static __device__ __forceinline__ auto frag(const char* t, int r0, int s) {
    const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
    if constexpr (ES == 2) {
      if constexpr (!TR) {
        return *(const bf16x8*)(t + (r0 + li) * 128 + (((2 * s + lh) ^ ((li >> 1) & 7)) << 4));
      } else {
        // rows 16 s + 8 lh + (0..3, 4..7): the transposed read hands lane l column l & 31 of them
        const int tq = (lane & 15) >> 2, tp = lane & 3, tg = (lane >> 4) & 1;
        const char* p = t + (16 * s + 8 * lh + tq) * (R * 2) + (((r0 >> 5) ^ tq) << 6) + 32 * tg + 8 * tp;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * R * 2));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    } else {
      // four k of this lane's half: 4 (2 s + lh) + 0..3, one v_mfma_f32_32x32x2_f32 each
      if constexpr (!TR) {
        return *(const f32x4*)(t + (r0 + li) * 128 + (((2 * s + lh) ^ ((li >> 1) & 7)) << 4));
      } else {
        const char* p = t + 4 * (2 * s + lh) * (R * 4) + (r0 + li) * 4;
        return f32x4{*(const float*)p, *(const float*)(p + R * 4), *(const float*)(p + 2 * R * 4),
                     *(const float*)(p + 3 * R * 4)};
      }
    }
  }
  typedef typename std::conditional<ES == 2, bf16x8, f32x4>::type frag_t;

  static __device__ __forceinline__ void load(const char* sa, const char* sb, int wm, int wn, int s, frag_t (&fa)[MT], frag_t (&fb)[NT]) {
#pragma unroll
    for (int j = 0; j < NT; ++j) fb[j] = frag<TRB, BN>(sb, (wn * NT + j) * 32, s);
#pragma unroll
    for (int i = 0; i < MT; ++i) fa[i] = frag<TRA, BM>(sa, (wm * MT + i) * 32, s);
  }

  static __device__ __forceinline__ void stage(const char* sa, const char* sb, int wm, int wn, f32x16 (&acc)[MT][NT]) {
    frag_t fa[2][MT], fb[2][NT];
    load(sa, sb, wm, wn, 0, fa[0], fb[0]);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s < 3) load(sa, sb, wm, wn, s + 1, fa[(s + 1) & 1], fb[(s + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (ES == 2) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[s & 1][j], fa[s & 1][i], acc[i][j], 0, 0, 0);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[s & 1][j][q], fa[s & 1][i][q], acc[i][j], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  static __device__ __forceinline__ void run(TA& ta, TB& tb, int first, int stages, char* smem, int wm, int wn, f32x16 (&acc)[MT][NT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
      if (d < stages) {
        ta.issue(smem + d * STAGE, first + d);
        tb.issue(smem + d * STAGE + TA::BYTES, first + d);
      }
    int now = 0, next = D - 1;
    for (int it = 0; it < stages; ++it) {
      if (it + D - 1 <= stages) stage_barrier<VEC, (D - 2) * (TA::LOADS + TB::LOADS)>();
      else stage_barrier<VEC, 0>();
      if (it + D - 1 < stages) {
        ta.issue(smem + next * STAGE, first + it + D - 1);
        tb.issue(smem + next * STAGE + TA::BYTES, first + it + D - 1);
      }
      stage(smem + now * STAGE, smem + now * STAGE + TA::BYTES, wm, wn, acc);
      now = now + 1 == D ? 0 : now + 1;
      next = next + 1 == D ? 0 : next + 1;
    }
  }
};

// y = x . w^T (TRB false: w [n][k], the contraction along its rows) or dx = dy . w (TRB: across them).
template <int ES, bool TRB, int WM, int WN, int MT, int NT, int D, bool VEC, bool OUT16>
__global__ __launch_bounds__(WM * WN * 64, 2) void grouped_rows_kernel(RowsArgs a) {
  typedef Core<ES, false, TRB, WM, WN, MT, NT, D, VEC> C;
  __shared__ __attribute__((aligned(1024))) char smem[D * C::STAGE];
  typedef typename std::conditional<OUT16, __bf16, float>::type out_t;
  const Place p = place_tile<C::BM>(a.offsets, a.groups, a.rows, a.ntiles, blockIdx.x, gridDim.x);
  if (!p.live) {
    if (a.clear) clear_rest(p, (out_t*)a.y, a.ldy, a.rows, a.n, C::NTH);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int n0 = p.nt * C::BN;
  typename C::TA ta;
  typename C::TB tb;
  ta.begin(a.a + (long long)p.m0 * a.lda, a.lda, p.hi - p.m0, a.k);
  tb.begin(a.w + p.e * a.w_group + (TRB ? (long long)n0 * ES : n0 * a.ldw), a.ldw, a.n - n0, a.k);
  f32x16 acc[MT][NT];
  C::run(ta, tb, 0, (a.k + C::KST - 1) / C::KST, smem, wm, wn, acc);
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = p.m0 + (wm * MT + i) * 32 + (threadIdx.x & 31);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = n0 + (wn * NT + j) * 32;
      store_tile<OUT16>(acc[i][j], m < p.hi && n < a.n ? (char*)((out_t*)a.y + m * a.ldy + n) : nullptr, a.n - n);
    }
  }
}

// dw_e = dy_e^T . x_e.  Workgroup: group, tile of dw, and a share of the group's rows (whole stages).
template <int ES, int WM, int WN, int MT, int NT, int D, bool VEC>
__global__ __launch_bounds__(WM * WN * 64, 2) void grouped_wgrad_kernel(WgradArgs a) {
  typedef Core<ES, true, true, WM, WN, MT, NT, D, VEC> C;
  __shared__ __attribute__((aligned(1024))) char smem[D * C::STAGE];
  const int tiles = a.ntiles * a.ktiles;
  const int e = blockIdx.x / (tiles * a.splits), at = blockIdx.x % (tiles * a.splits);
  const int split = at / tiles, nt = at % tiles / a.ktiles, kt = at % a.ktiles;
  const Span g = group_span(a.offsets, a.groups, a.rows, e);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int n0 = nt * C::BM, k0 = kt * C::BN;
  const int all = (g.hi - g.lo + C::KST - 1) / C::KST;
  const int first = (int)((long long)all * split / a.splits), last = (int)((long long)all * (split + 1) / a.splits);
  typename C::TA ta;
  typename C::TB tb;
  ta.begin(a.dy + g.lo * a.lddy + (long long)n0 * ES, a.lddy, a.n - n0, g.hi - g.lo);
  tb.begin(a.x + g.lo * a.ldx + (long long)k0 * ES, a.ldx, a.k - k0, g.hi - g.lo);
  f32x16 acc[MT][NT];
  C::run(ta, tb, first, last - first, smem, wm, wn, acc);
  float* const dw = a.dw + ((long long)split * a.groups + e) * a.n * a.k;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int n = n0 + (wm * MT + i) * 32 + (threadIdx.x & 31);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int k = k0 + (wn * NT + j) * 32;
      float* const row = n < a.n && k < a.k ? dw + (long long)n * a.k + k : nullptr;
      if (a.accumulate && row) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int c = 8 * (r >> 2) + 4 * ((threadIdx.x >> 5) & 1) + (r & 3);
          if (k + c < a.k) acc[i][j][r] += row[c];
        }
      }
      store_tile<false>(acc[i][j], (char*)row, a.k - k);
    }
  }
}

bool fits(long long pitch_bytes) { return pitch_bytes > 0 && pitch_bytes <= C2DP_MAX_PITCH; }

template <int ES, bool TRB, bool VEC, bool OUT16>
int launch_rows(RowsArgs a, hipStream_t stream) {
  constexpr int WM = XWM, WN = XWN, MT = XMT, NT = XNT, D = XD;
  constexpr int BM = WM * MT * 32, BN = WN * NT * 32;
  a.ntiles = (a.n + BN - 1) / BN;
  const unsigned grid = place_grid(BM, a.groups, true, a.rows, a.ntiles);
  if (!grid) return C2D_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((grouped_rows_kernel<ES, TRB, WM, WN, MT, NT, D, VEC, OUT16>), dim3(grid), dim3(WM * WN * 64), 0, stream, a);
  return c2d_launch_status();
}

template <bool TRB>
int rows_product(const void* x, int x_type, long long ldx, const void* w, const int32_t* offsets, int groups, void* y,
                 int y_type, long long ldy, int rows, int n, int k, int contraction, int clear, void* stream) {
  // n: result columns, contraction: columns of x; w [groups][..][k] of the caller's n and k
  C2D_CHECK_ARG(groups > 0 && rows >= 0 && n >= 0 && contraction >= 0 && ldx >= contraction && ldy >= n);
  C2D_CHECK_ARG(x_type == C2DP_F32 || x_type == C2DP_BF16);
  C2D_CHECK_ARG(y_type == x_type || (x_type == C2DP_BF16 && y_type == C2DP_F32));
  if (rows == 0 || n == 0) return C2D_OK;
  C2D_CHECK_ARG(offsets && y && (contraction == 0 || (x && w)));
  const int es = x_type == C2DP_BF16 ? 2 : 4, ys = y_type == C2DP_BF16 ? 2 : 4;
  if ((long long)(contraction > 0 ? ldx : 1) * es > C2DP_MAX_PITCH || (long long)(k > 0 ? k : 1) * es > C2DP_MAX_PITCH)
    return C2D_ERR_UNSUPPORTED;
  RowsArgs a;
  a.a = (const char*)x;
  a.lda = ldx * es;
  a.w = (const char*)w;
  a.ldw = (long long)k * es;
  a.w_group = (long long)n * contraction * es;
  a.offsets = offsets;
  a.y = (char*)y;
  a.ldy = ldy;
  a.groups = groups;
  a.rows = rows;
  a.n = n;
  a.k = contraction;
  a.clear = clear;
  const hipStream_t s = (hipStream_t)stream;
  // (16-byte loads: the contraction's last chunk is whole; across it, a row of w is whole chunks)
  const bool vec = aligned16(x, a.lda) && aligned16(w, a.ldw) && (long long)contraction * es % 16 == 0;
  if (es == 4) return vec ? launch_rows<4, TRB, true, false>(a, s) : launch_rows<4, TRB, false, false>(a, s);
  if (ys == 4) return vec ? launch_rows<2, TRB, true, false>(a, s) : launch_rows<2, TRB, false, false>(a, s);
  return vec ? launch_rows<2, TRB, true, true>(a, s) : launch_rows<2, TRB, false, true>(a, s);
}

}  // namespace

extern "C" int c2dp_version(void) { return C2DP_ABI_VERSION; }

extern "C" int c2dp_grouped_matmul(const void* x, int x_type, long long ldx, const void* w, const int32_t* offsets,
                                   int groups, void* y, int y_type, long long ldy, int rows, int n, int k,
                                   int clear_rest, void* stream) {
  return rows_product<false>(x, x_type, ldx, w, offsets, groups, y, y_type, ldy, rows, n, k, k, clear_rest, stream);
}

extern "C" int c2dp_grouped_matmul_dgrad(const void* dy, int dy_type, long long lddy, const void* w,
                                         const int32_t* offsets, int groups, void* dx, int dx_type, long long lddx,
                                         int rows, int n, int k, int clear_rest, void* stream) {
  return rows_product<true>(dy, dy_type, lddy, w, offsets, groups, dx, dx_type, lddx, rows, k, k, n, clear_rest, stream);
}

extern "C" unsigned long long c2dp_grouped_matmul_wgrad_workspace_bytes(int groups, int rows, int n, int k) {
  (void)groups; (void)rows; (void)n; (void)k;
  return 0;
}

namespace {
template <int ES, bool VEC>
int launch_wgrad(WgradArgs a, hipStream_t stream) {
  constexpr int WM = XWM, WN = XWN, MT = XMT, NT = XNT, D = XD;
  constexpr int BM = WM * MT * 32, BN = WN * NT * 32;
  a.ntiles = (a.n + BM - 1) / BM;
  a.ktiles = (a.k + BN - 1) / BN;
  a.splits = 1;
  const long long grid = (long long)a.groups * a.ntiles * a.ktiles * a.splits;
  if (grid >= (1ll << 30)) return C2D_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((grouped_wgrad_kernel<ES, WM, WN, MT, NT, D, VEC>), dim3((unsigned)grid), dim3(WM * WN * 64), 0, stream, a);
  return c2d_launch_status();
}
}  // namespace

extern "C" int c2dp_grouped_matmul_wgrad(const void* x, int x_type, long long ldx, const void* dy, long long lddy,
                                         const int32_t* offsets, int groups, float* dw, int rows, int n, int k,
                                         int accumulate, void* workspace, unsigned long long workspace_bytes,
                                         void* stream) {
  C2D_CHECK_ARG(groups > 0 && rows >= 0 && n >= 0 && k >= 0 && ldx >= k && lddy >= n);
  C2D_CHECK_ARG(x_type == C2DP_F32 || x_type == C2DP_BF16);
  if (n == 0 || k == 0) return C2D_OK;
  C2D_CHECK_ARG(offsets && dw && (rows == 0 || (x && dy)));
  const int es = x_type == C2DP_BF16 ? 2 : 4;
  if (!fits(ldx * es) || !fits(lddy * es)) return C2D_ERR_UNSUPPORTED;
  (void)workspace; (void)workspace_bytes;
  WgradArgs a;
  a.dy = (const char*)dy;
  a.x = (const char*)x;
  a.lddy = lddy * es;
  a.ldx = ldx * es;
  a.offsets = offsets;
  a.dw = dw;
  a.groups = groups;
  a.rows = rows;
  a.n = n;
  a.k = k;
  a.accumulate = accumulate;
  const bool vec = aligned16(x, a.ldx) && aligned16(dy, a.lddy) && n * es % 16 == 0 && k * es % 16 == 0;
  const hipStream_t s = (hipStream_t)stream;
  if (es == 4) return vec ? launch_wgrad<4, true>(a, s) : launch_wgrad<4, false>(a, s);
  return vec ? launch_wgrad<2, true>(a, s) : launch_wgrad<2, false>(a, s);
}
