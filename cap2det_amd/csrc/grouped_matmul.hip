// Matrix products grouped by expert: the rows of x sorted by group, one weight matrix per group, the groups'
// lengths on the device.  Forward, input gradient and weight gradient, bf16 and fp32 operands, fp32 sums.
#include "products_few.h"

using namespace c2d_pr;

namespace {

struct WgradArgs {
  const char *dy, *x;
  long long lddy, ldx;        // bytes
  const int* offsets;
  float* dw;                  // [groups][n][k], or [splits][groups][n][k]
  int groups, rows, n, k;
  int ntiles, ktiles, splits, accumulate;
};

// The stages of A go round D buffers, those of B round D + 1: while a stage is multiplied, the next of A and
// the next two of B are on their way (D = 2; five buffers are what the LDS holds of 256 x 256 tiles, and a load takes
// longer than a stage).  B are the weights, which come from memory, each group's own, where rows come from L2
// for all but one of their column tiles (8192^3: 851 us, with the third buffer A's 874; its input gradient 870, 906;
// on other cards of the kind 851-881 and 870-925).
// One barrier per stage; the loads are issued between the matrix instructions of its first half, since a burst
// of them behind the barrier holds up every wave of the workgroup.
// KG > 1: KG groups of WM x WN waves share the tile, group g taking the stages g, g + KG, ..
template <int ES, bool TRA, bool TRB, int WM, int WN, int MT, int NT, int KG, int D, bool VEC>
struct Core {
  static constexpr int BM = WM * MT * 32, BN = WN * NT * 32, NTH = WM * WN * 64, DA = D, DB = D + 1;
  typedef Tile<ES, TRA, BM, NTH, VEC, TRA || TRB> TA;
  typedef Tile<ES, TRB, BN, NTH, VEC, TRA || TRB> TB;
  static constexpr int RING = DA * TA::BYTES + DB * TB::BYTES;
  static constexpr int PASSES = TA::LOADS + TB::LOADS;
  static constexpr int KST = TA::KST;
  static_assert(KG == 1 || (KG - 1) * NTH * 64 <= KG * RING, "the sums are joined a tile at a time in the ring's LDS");

  // fragment of 32 rows (TR: columns) from `r0`, k-step s, for a lane
  template <class T, bool TR, int R>
  static __device__ __forceinline__ auto frag(const char* t, int r0, int s) {
    const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
    if constexpr (ES == 2) {
      if constexpr (!TR) {
        return *(const bf16x8*)(t + (r0 + li) * 128 + (((2 * s + lh) ^ ((li >> 1) & 7)) << 4));
      } else {
        // rows 16 s + 8 lh + (0..3, 4..7): the transposed read hands lane l column l & 31 of them
        const int tq = (lane & 15) >> 2, tp = lane & 3, tg = (lane >> 4) & 1;
        const char* p = t + (16 * s + 8 * lh + tq) * (R * 2) + (((r0 >> 5) ^ (T::swizzle(tq) >> 2)) << 6) + 32 * tg + 8 * tp;
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
    for (int j = 0; j < NT; ++j) fb[j] = frag<TB, TRB, BN>(sb, (wn * NT + j) * 32, s);
#pragma unroll
    for (int i = 0; i < MT; ++i) fa[i] = frag<TA, TRA, BM>(sa, (wm * MT + i) * 32, s);
  }

  // Stages first .. first + stages - 1.
  static __device__ __forceinline__ void run(const TA& ta, const TB& tb, int first, int stages, char* smem, int group, int wm,
                                             int wn, f32x16 (&acc)[MT][NT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    if (stages <= 0) return;
    char* const ring_a = smem + group * RING;
    char* const ring_b = ring_a + DA * TA::BYTES;
    const int rounds = (stages + KG - 1) / KG;
    // (a stage behind the last reads zeros: the operands end there)
    tb.issue(ring_b, first + group);
#pragma unroll
    for (int d = 0; d < D - 1; ++d) {
      ta.issue(ring_a + d * TA::BYTES, first + d * KG + group);
      tb.issue(ring_b + (d + 1) * TB::BYTES, first + (d + 1) * KG + group);
    }
    int now_a = 0, now_b = 0, next_a = DA - 1, next_b = DB - 1;
    for (int it = 0; it < rounds; ++it) {
      // (behind this stage's A have been issued: B of the next, and D - 2 whole stages)
      stage_barrier<VEC, TB::LOADS + (D - 2) * PASSES>();
      const int st_a = first + (it + DA - 1) * KG + group, st_b = first + (it + DB - 1) * KG + group;
      const typename TA::Stage ga = ta.at(st_a);
      const typename TB::Stage gb = tb.at(st_b);
      const char* const sa = ring_a + now_a * TA::BYTES;
      const char* const sb = ring_b + now_b * TB::BYTES;
      auto pass = [&](int q) {
        if (q < TA::LOADS) ta.pass(ring_a + next_a * TA::BYTES, ga, st_a, q);
        else tb.pass(ring_b + next_b * TB::BYTES, gb, st_b, q - TA::LOADS);
      };
      constexpr int QS = ES == 2 ? 1 : 4, SLOTS = 4 * QS * MT * NT;  // matrix instructions of a stage
      constexpr int PER = (2 * PASSES + SLOTS - 1) / SLOTS, EVERY = PER > 1 ? 1 : SLOTS / (2 * PASSES);
      frag_t fa[2][MT], fb[2][NT];
      load(sa, sb, wm, wn, 0, fa[0], fb[0]);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (s < 3) load(sa, sb, wm, wn, s + 1, fa[(s + 1) & 1], fb[(s + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < QS; ++q)
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              if constexpr (ES == 2)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[s & 1][j], fa[s & 1][i], acc[i][j], 0, 0, 0);
              else
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[s & 1][j][q], fa[s & 1][i][q], acc[i][j], 0, 0, 0);
              const int slot = ((s * QS + q) * MT + i) * NT + j;
              if (slot % EVERY == 0) {
#pragma unroll
                for (int u = slot / EVERY * PER; u < (slot / EVERY + 1) * PER && u < PASSES; ++u) pass(u);
                if (slot / EVERY * PER < PASSES) __builtin_amdgcn_sched_barrier(0);
              }
            }
        __builtin_amdgcn_sched_barrier(0);
      }
      now_a = now_a + 1 == DA ? 0 : now_a + 1;
      next_a = next_a + 1 == DA ? 0 : next_a + 1;
      now_b = now_b + 1 == DB ? 0 : now_b + 1;
      next_b = next_b + 1 == DB ? 0 : next_b + 1;
    }
    drain_loads();
    if constexpr (KG > 1) join_groups<KG, NTH>((float*)smem, group, threadIdx.x - group * NTH, acc);
  }
};

// y = x . w^T (TRB false: w [n][k], the contraction along its rows) or dx = dy . w (TRB: across them).
// A row tile (`p`) of C's height or less.
template <class C, bool TRB, int ES, int WN, int MT, int NT, bool OUT16>
__device__ __forceinline__ void rows_tile(const FewArgs& a, const Place& p, char* smem, int group, int tid) {
  typedef typename std::conditional<OUT16, __bf16, float>::type out_t;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int n0 = p.nt * C::BN;
  typename C::TA ta;
  typename C::TB tb;
  ta.begin(a.a + (long long)p.m0 * a.lda, a.lda, p.hi - p.m0, a.k, tid);
  tb.begin(a.b + p.e * a.b_group + (TRB ? (long long)n0 * ES : n0 * a.ldb), a.ldb, a.n - n0, a.k, tid);
  f32x16 acc[MT][NT];
  C::run(ta, tb, 0, (a.k + C::KST - 1) / C::KST, smem, group, wm, wn, acc);
  __syncthreads();
  if (group > 0) return;
  typedef Store<OUT16, NT> S;
  static_assert(C::NTH / 64 * S::BYTES <= C::RING, "the result goes out through the ring's LDS");
  const int m = p.m0 + wm * MT * 32, n = n0 + wn * NT * 32;
  S::run(acc, smem + wave * S::BYTES, (char*)((out_t*)a.y + m * a.ldy + n), a.ldy * (long long)sizeof(out_t), p.hi - m, a.n - n);
}

// A group's last tile is on average half full.  Half of it or less is multiplied as a tile of half the height.
template <int ES, bool TRB, int WM, int WN, int MT, int NT, int KG, int D, bool VEC, bool OUT16>
__global__ __launch_bounds__(WM * WN * KG * 64, 2) void grouped_rows_kernel(FewArgs a) {
  typedef Core<ES, false, TRB, WM, WN, MT, NT, KG, D, VEC> C;
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
      rows_tile<Core<ES, false, TRB, WM, WN, MT / 2, NT, KG, D, VEC>, TRB, ES, WN, MT / 2, NT, OUT16>(a, p, smem, group, tid);
      return;
    }
  }
  rows_tile<C, TRB, ES, WN, MT, NT, OUT16>(a, p, smem, group, tid);
}

// dw_e = dy_e^T . x_e.  Workgroup: group, tile of dw, and a share of the group's rows (whole stages).
template <int ES, int WM, int WN, int MT, int NT, int KG, int D, bool VEC>
__global__ __launch_bounds__(WM * WN * KG * 64, 2) void grouped_wgrad_kernel(WgradArgs a) {
  typedef Core<ES, true, true, WM, WN, MT, NT, KG, D, VEC> C;
  __shared__ __attribute__((aligned(1024))) char smem[KG * C::RING];
  // Workgroups go round the 8 XCDs: of every 256 tiles XCD x takes the x-th eighth, so that a group's rows come through
  // the L2 of an XCD or two instead of all eight, and every XCD meets long groups and short ones (32 groups of
  // about 512 x 2048 x 2048: 242 us, on other cards to 262; tiles in their order 252, 576 MB fetched of 134; an eighth of all tiles 271.  One
  // group of 16384 x 2048 x 2048: 138 us, in their order 165).
  const int tiles = a.ntiles * a.ktiles, total = tiles * a.splits * a.groups;
  const unsigned wg = workgroup();
  const int xcd = wg & 7, window = wg >> 8 << 8, at_xcd = wg >> 3 & 31;
  const int here = min(256, total - window), share = (here + 7) >> 3;
  if (at_xcd >= share || xcd * share + at_xcd >= here) return;
  const int idx = window + xcd * share + at_xcd;
  const int e = idx / (tiles * a.splits), at = idx % (tiles * a.splits);
  const int split = at / tiles, nt = at % tiles / a.ktiles, kt = at % a.ktiles;
  const Span g = group_span(a.offsets, a.groups, a.rows, e);
  const int group = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / C::NTH), tid = threadIdx.x - group * C::NTH;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int n0 = nt * C::BM, k0 = kt * C::BN;
  const int all = (g.hi - g.lo + C::KST - 1) / C::KST;
  const int first = (int)((long long)all * split / a.splits), last = (int)((long long)all * (split + 1) / a.splits);
  typename C::TA ta;
  typename C::TB tb;
  // (the share's end is the operands' end)
  const int end = min(g.hi - g.lo, last * C::KST);
  ta.begin(a.dy + g.lo * a.lddy + (long long)n0 * ES, a.lddy, a.n - n0, end, tid);
  tb.begin(a.x + g.lo * a.ldx + (long long)k0 * ES, a.ldx, a.k - k0, end, tid);
  f32x16 acc[MT][NT];
  C::run(ta, tb, first, last - first, smem, group, wm, wn, acc);
  __syncthreads();
  if (group > 0) return;
  typedef Store<false, NT> S;
  static_assert(C::NTH / 64 * S::BYTES <= C::RING, "the result goes out through the ring's LDS");
  const int n = n0 + wm * MT * 32, k = k0 + wn * NT * 32;
  float* const dw = a.dw + ((long long)split * a.groups + e) * a.n * a.k + (long long)n * a.k + k;
  S::run(acc, smem + wave * S::BYTES, (char*)dw, a.k * 4ll, a.n - n, a.k - k, a.accumulate);
}

// dw (+)= the sum of the shares' tiles, in their order.  What dw holds is added last, as by a workgroup that made the whole
// gradient: added first, shares below half a step of a large dw would go one by one.
__global__ __launch_bounds__(256) void join_shares_kernel(const float* __restrict__ parts, float* __restrict__ dw, long long count,
                                                          int splits, int accumulate) {
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < count; i += (long long)gridDim.x * 1024) {
    if (i + 4 <= count) {
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f}, p;
      for (int s = 0; s < splits; ++s) {
        __builtin_memcpy(&p, parts + s * count + i, 16);
        v += p;
      }
      if (accumulate) {
        __builtin_memcpy(&p, dw + i, 16);
        v += p;
      }
      store_at((char*)(dw + i), v);
    } else {
      for (long long j = i; j < count; ++j) {
        float v = 0.0f;
        for (int s = 0; s < splits; ++s) v += parts[s * count + j];
        dw[j] = accumulate ? v + dw[j] : v;
      }
    }
  }
}

// ---- launches (products_choice.h says which) ---------------------------------------------------------

template <int ES, bool TRB, int WM, int WN, int MT, int NT, int KG, int D, bool VEC, bool OUT16>
int launch_tiles(FewArgs a, hipStream_t stream) {
  constexpr int BM = WM * MT * 32, BN = WN * NT * 32;
  a.ntiles = (a.n + BN - 1) / BN;
  a.slots = slots_per_xcd(KG * Core<ES, false, TRB, WM, WN, MT, NT, KG, D, VEC>::RING);
  const unsigned grid = place_grid(BM, a.groups, true, a.rows, a.ntiles, MT > 1 ? a.slots / 2 : 0);
  if (!grid) return C2D_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((grouped_rows_kernel<ES, TRB, WM, WN, MT, NT, KG, D, VEC, OUT16>), grid_of(grid), dim3(WM * WN * KG * 64), 0, stream, a);
  return c2d_launch_status();
}

template <int ES, bool TRB, bool VEC, bool OUT16>
int launch_rows(const FewArgs& a, hipStream_t stream) {
  const Shape shape = rows_shape(a.rows, a.n, a.k, a.groups, ES, !TRB, VEC, c2d_available_cus());
  if constexpr (ES == 2 && VEC) {
    if (shape == T256) return launch_tiles<ES, TRB, 2, 4, 4, 2, 1, 2, true, OUT16>(a, stream);
    if (shape == T128W) return launch_tiles<ES, TRB, 2, 4, 2, 2, 1, 2, true, OUT16>(a, stream);
  }
  if constexpr (!TRB) {
    if (ES == 2 && shape == T16W) return launch_few<BF16, false, 1, 2, 2, VEC, OUT16>(a, stream);
    if (shape == T16) return launch_few<ES == 2 ? BF16 : F32, false, 1, 1, 8, VEC, OUT16>(a, stream);
    if (shape == T32) return launch_few<ES == 2 ? BF16 : F32, false, 2, 2, 8, VEC, OUT16>(a, stream);
  }
  if (shape == T128) return launch_tiles<ES, TRB, 2, 2, 2, 2, 1, 2, VEC, OUT16>(a, stream);
  return launch_tiles<ES, TRB, 2, 2, 1, 1, 2, 4, VEC, OUT16>(a, stream);
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
  if (!groups_fit(groups) || !sizes_fit(rows, n, k)) return C2D_ERR_UNSUPPORTED;
  if ((long long)(contraction > 0 ? ldx : 1) * es > C2DP_MAX_PITCH || (long long)(k > 0 ? k : 1) * es > C2DP_MAX_PITCH)
    return C2D_ERR_UNSUPPORTED;
  FewArgs a = {};
  a.a = (const char*)x;
  a.lda = ldx * es;
  a.b = (const char*)w;
  a.ldb = (long long)k * es;
  a.b_group = (long long)n * contraction * es;
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
  const bool vec = aligned16(x, a.lda) && aligned16(w, a.ldb) && (long long)contraction * es % 16 == 0;
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

extern "C" unsigned long long c2dp_grouped_matmul_wgrad_workspace_bytes(int groups, int rows, int n, int k, int x_type) {
  if (groups <= 0 || rows <= 0 || n <= 0 || k <= 0 || (x_type != C2DP_F32 && x_type != C2DP_BF16)) return 0;
  const int splits = wgrad_plan(groups, rows, n, k, x_type == C2DP_BF16 ? 2 : 4).splits;
  return splits > 1 ? 4ull * splits * groups * n * k : 0;
}

namespace {
template <int ES, int WM, int WN, int MT, int NT, int KG, int D, bool VEC>
int launch_wgrad(WgradArgs a, hipStream_t stream) {
  a.ntiles = (a.n + WM * MT * 32 - 1) / (WM * MT * 32);
  a.ktiles = (a.k + WN * NT * 32 - 1) / (WN * NT * 32);
  const long long grid = (long long)a.groups * a.ntiles * a.ktiles * a.splits;
  if (grid >= (1ll << 30)) return C2D_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((grouped_wgrad_kernel<ES, WM, WN, MT, NT, KG, D, VEC>), grid_of((grid + 255) / 256 * 256), dim3(WM * WN * KG * 64), 0, stream, a);
  return c2d_launch_status();
}

template <int ES, bool VEC>
int launch_wgrad_side(const WgradArgs& a, int side, hipStream_t stream) {
  if constexpr (ES == 2 && VEC) {
    if (side == 256) return launch_wgrad<2, 4, 2, 2, 4, 1, 2, true>(a, stream);
  }
  if (side >= 128) return launch_wgrad<ES, 2, 2, 2, 2, 1, 2, VEC>(a, stream);
  return launch_wgrad<ES, 2, 2, 1, 1, 2, 4, VEC>(a, stream);
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
  if (!groups_fit(groups) || !sizes_fit(rows, n, k) || ldx * es > C2DP_MAX_PITCH || lddy * es > C2DP_MAX_PITCH) return C2D_ERR_UNSUPPORTED;
  const unsigned long long need = c2dp_grouped_matmul_wgrad_workspace_bytes(groups, rows, n, k, x_type);
  if (workspace_bytes < need || (need && !workspace)) return C2D_ERR_WORKSPACE;
  C2D_CHECK_ARG(((unsigned long long)workspace & 15) == 0);
  const WgradPlan plan = wgrad_plan(groups, rows, n, k, es);
  WgradArgs a;
  a.dy = (const char*)dy;
  a.x = (const char*)x;
  a.lddy = lddy * es;
  a.ldx = ldx * es;
  a.offsets = offsets;
  a.splits = need ? plan.splits : 1;
  a.dw = need ? (float*)workspace : dw;
  a.groups = groups;
  a.rows = rows;
  a.n = n;
  a.k = k;
  a.accumulate = need ? 0 : accumulate;
  const bool vec = aligned16(x, a.ldx) && aligned16(dy, a.lddy) && n * es % 16 == 0 && k * es % 16 == 0;
  const hipStream_t s = (hipStream_t)stream;
  const int status = es == 4 ? (vec ? launch_wgrad_side<4, true>(a, plan.side, s) : launch_wgrad_side<4, false>(a, plan.side, s))
                             : (vec ? launch_wgrad_side<2, true>(a, plan.side, s) : launch_wgrad_side<2, false>(a, plan.side, s));
  if (status != C2D_OK || !need) return status;
  const long long count = (long long)groups * n * k;
  const long long blocks = (count + 1023) / 1024;
  hipLaunchKernelGGL(join_shares_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, (const float*)workspace, dw,
                     count, a.splits, accumulate);
  return c2d_launch_status();
}
