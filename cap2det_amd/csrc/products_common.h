// What the grouped and 8-bit matrix products share: where a workgroup's tile lies among ragged groups, the
// staging of operand tiles in LDS, the fragments read from it and the store of a result tile.  gfx950 only.
//
// Every product here is  D[m][n] = sum_k A[m][k] * B[n][k]  over operands that lie either with the
// contraction contiguous (A[m][k] at m * ld + k) or across it (A[m][k] at k * ld + m, "TR"):
//   forward         A = x  [row][k]   B = w [n][k]
//   input gradient  A = dy [row][n]   B = w, contracted over its rows (TR)
//   weight gradient A = dy, B = x, both contracted over their rows (TR, TR)
// A stage holds 128 bytes of the contraction of every operand row: 128 8-bit, 64 bf16 or 32 fp32 elements.
// MFMAs take B as their first operand, so that a lane's registers run along n, which is contiguous in
// every result: 16-byte stores, and one activation scale per lane in the 8-bit product.
#pragma once
#include "c2d_common.h"
#include "../../include/cap2det_products.h"
#include "products_choice.h"
#include "products_place.h"
#include <type_traits>

namespace c2d_pr {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

constexpr unsigned OUTSIDE = 0x7FFFFF00u;  // an offset behind every buffer: the load returns zeros

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, long long bytes) {
  const unsigned long long u = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)u);
  const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)(u >> 32));
  const unsigned nb = __builtin_amdgcn_readfirstlane(
      (unsigned)(bytes < 0 ? 0 : bytes < (long long)OUTSIDE ? bytes : (long long)OUTSIDE));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((unsigned long long)hi << 32) | lo), (short)0, (int)nb,
                                           0x00020000);
}

// The same as the four words of a buffer resource.
__device__ __forceinline__ i32x4 buffer_words(const void* p, long long bytes) {
  const unsigned long long u = (unsigned long long)p;
  return i32x4{__builtin_amdgcn_readfirstlane((int)(unsigned)u), __builtin_amdgcn_readfirstlane((int)(unsigned)(u >> 32) & 0xffff),
               __builtin_amdgcn_readfirstlane((int)(bytes < 0 ? 0 : bytes < (long long)OUTSIDE ? bytes : (long long)OUTSIDE)),
               0x00020000};
}

// ---- ragged groups ------------------------------------------------------------------------------

// Running sums / maxima (of numbers from 0) over the lanes of a wave: four steps within 16 lanes and two across them, as
// operands of the vector instructions (DPP).  As shuffles through LDS they were most of a workgroup's start.
template <class Op>
__device__ __forceinline__ int lane_scan(int v, Op op) {
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));  // row_shr:1
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));  // row_shr:2
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));  // row_shr:4
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));  // row_shr:8
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));  // row_bcast:15, into rows 1 and 3
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));  // row_bcast:31, into rows 2 and 3
  return v;
}
__device__ __forceinline__ int lane_prefix_sum(int v) {
  return lane_scan(v, [](int a, int b) { return a + b; });
}

// The spans of groups base .. base + 63, one per lane (empty behind the last group); `carry`: the
// largest boundary so far, updated.
__device__ __forceinline__ Span lane_span(const int* __restrict__ offsets, int groups, int rows, int base,
                                          int* carry) {
  const int i = base + (int)(threadIdx.x & 63);
  int lo = max(0, min(rows, offsets[min(i, groups)]));
  const int next = max(0, min(rows, offsets[min(i + 1, groups)]));
  lo = max(lane_scan(lo, [](int a, int b) { return max(a, b); }), *carry);
  const int hi = max(lo, next);
  *carry = __builtin_amdgcn_readlane(hi, 63);
  return {lo, i < groups ? hi : lo};
}

// One group's span (all waves, any lane).
__device__ __forceinline__ Span group_span(const int* __restrict__ offsets, int groups, int rows, int e) {
  int carry = 0;
  for (int base = 0;; base += 64) {
    const Span s = lane_span(offsets, groups, rows, base, &carry);
    if (e < base + 64)
      return {__builtin_amdgcn_readlane(s.lo, e - base), __builtin_amdgcn_readlane(s.hi, e - base)};
  }
}

// Workgroups by number.  A launch holds fewer than 2^32 threads along x, 2^23 workgroups of 512: more than 2^22 go along y, in
// rows of 2^22, which keeps their way round the XCDs.
inline dim3 grid_of(long long workgroups) {
  constexpr long long ROW = 1 << 22;
  return workgroups <= ROW ? dim3((unsigned)workgroups) : dim3((unsigned)ROW, (unsigned)((workgroups + ROW - 1) / ROW));
}
__device__ __forceinline__ unsigned workgroup() { return blockIdx.y * gridDim.x + blockIdx.x; }
__device__ __forceinline__ unsigned workgroups() { return gridDim.y * gridDim.x; }

// Tile of workgroup `bid` (products_place.h).  The host cannot know how many row tiles the groups make; it launches the
// largest number, rows / BM + groups, and each wave counts them here: one or two loads and two dozen lane shuffles
// for 64 groups.
template <int BM, bool HALVES>
__device__ __forceinline__ Place place_tile(const int* __restrict__ offsets, int groups, int rows, int ntiles,
                                            unsigned bid, unsigned nbid, int slots) {
  Place p;
  int carry = 0, full = 0, half = 0;  // row tiles of all groups
  Span s = {0, rows};
  int upto_full = 0, upto_half = 0;
  if (!offsets) {
    full = (rows + BM - 1) / BM;
    p.begin = 0;
    p.end = rows;
  } else {
    for (int base = 0; base < groups; base += 64) {
      s = lane_span(offsets, groups, rows, base, &carry);
      if (base == 0) p.begin = __builtin_amdgcn_readlane(s.lo, 0);
      upto_full = lane_prefix_sum(full_tiles_of<BM, HALVES>(s.hi - s.lo));
      full += __builtin_amdgcn_readlane(upto_full, 63);
      if (HALVES) {
        upto_half = lane_prefix_sum(half_tiles_of<BM, HALVES>(s.hi - s.lo));
        half += __builtin_amdgcn_readlane(upto_half, 63);
      }
    }
    p.end = carry;
  }
  const Pick t = pick_tile<HALVES>(p, full, half, ntiles, bid, nbid, slots);
  if (!p.live) return p;
  if (!offsets) {
    p.e = 0; p.lo = 0; p.hi = rows;
    tile_rows<BM>(p, t, 0, full);
    return p;
  }
  int before = 0;
  if (groups > 64) carry = 0;
  for (int base = 0; base < groups; base += 64) {
    if (groups > 64) {
      s = lane_span(offsets, groups, rows, base, &carry);
      upto_full = lane_prefix_sum(full_tiles_of<BM, HALVES>(s.hi - s.lo));
      if (HALVES) upto_half = lane_prefix_sum(half_tiles_of<BM, HALVES>(s.hi - s.lo));
    }
    const int upto = t.small ? upto_half : upto_full;
    const unsigned long long has = __ballot(before + upto > t.mt);
    if (has) {
      const int l = __builtin_ctzll(has);
      p.e = base + l;
      p.lo = __builtin_amdgcn_readlane(s.lo, l);
      p.hi = __builtin_amdgcn_readlane(s.hi, l);
      const int mine = full_tiles_of<BM, HALVES>(p.hi - p.lo);
      tile_rows<BM>(p, t, before + __builtin_amdgcn_readlane(upto, l) - mine, mine);
      return p;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  p.live = false;  // (offsets that somebody changed since they were counted: no tile, rather than a search without end)
  return p;
}

// Rows in no group := 0, by the workgroups that have no tile.
template <class T>
__device__ __forceinline__ void clear_rest(const Place& p, T* y, long long ldy, int rows, int n, int threads) {
  if (p.spare < 0) return;
  const int rest = rows - (p.end - p.begin);
  for (long long i = p.spare; i < rest; i += p.spares) {
    const long long row = i < p.begin ? i : p.end + (i - p.begin);
    for (int c = threadIdx.x; c < n; c += threads) y[row * ldy + c] = (T)0.0f;
  }
}

// ---- staging --------------------------------------------------------------------------------------

// One operand's tile of R rows (or, TR, R columns) by 128 bytes of the contraction, staged by NTH threads.
//
// LDS image, contraction contiguous: 128-byte rows, 16-byte chunk c of row r at c ^ ((r >> 1) & 7).  A
// ds_read_b128 takes one chunk of 16 consecutive rows at a time; the XOR puts those on 16 different
// 16-byte slots of the 256-byte bank period.  TR: 128 / ES rows of R * ES bytes as they lie in memory;
// bf16 moves 64-byte granule g of row r to g ^ (r & 3) (R = 64, two granules a row: g ^ (r >> 1 & 1)), so that
// the four rows of a transposed read (ds_read_b64_tr_b16) lie on four bank groups.  The image of a load to LDS is lane-linear: the XOR is
// applied to the address that a lane fetches from.
//
// VEC: loads go to LDS directly (buffer_load ... lds, 16 bytes a lane), and lie outside their buffer, which
// returns zeros, behind the operand's last row and behind the contraction's end.  Not VEC (a pitch, a
// pointer or a length that 16-byte loads to LDS do not fit): loads to registers, with their own bounds.
//
// UNSEEN: the load to LDS is written as an instruction that the compiler does not look into.  It waits for
// every such load that it knows of before each transposed LDS read, which is the whole latency of the next stage
// at every step of 16 k (input gradient 8192^3 in 256 x 256 tiles: 1054 us, unseen 921, with the loads between the matrix
// instructions as they are now 870-925; in 128 x 128 tiles 1341, 1113);
// stage_barrier waits for what is needed.
template <int ES, bool TR, int R, int NTH, bool VEC, bool UNSEEN = false>
struct Tile {
  static constexpr int BYTES = R * 128;
  static constexpr int LOADS = BYTES / (NTH * 16);
  static constexpr int EPC = 16 / ES;
  static constexpr int KST = 128 / ES;               // contraction elements per stage
  static constexpr int CPR = TR ? R * ES / 16 : 8;   // chunks per staged row
  static constexpr int RPP = NTH / CPR;              // staged rows per pass
  static_assert(LOADS * NTH * 16 == BYTES, "tile vs workgroup");
  static_assert(NTH % CPR == 0 && (RPP % 16 == 0 || (TR && RPP % 4 == 0)), "the XOR is the same in every pass");

  const char* base;
  long long ld;          // bytes
  int across, len;       // rows (TR: columns) from base that exist; contraction elements
  int tid, row, chunk;   // thread among the NTH, its staged row and source chunk of the first pass
  int wave;              // (of the wave)
  unsigned off;          // its offset; pass i lies i * RPP rows behind it

  __device__ __forceinline__ void begin(const void* p, long long ld_bytes, int across_, int len_, int tid_ = threadIdx.x) {
    tid = tid_;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    base = (const char*)p;
    ld = ld_bytes;
    across = min(across_, R);
    len = len_;
    row = tid / CPR;
    const int pos = tid % CPR;
    chunk = pos ^ swizzle(row);
    off = (unsigned)(row * (int)ld + chunk * 16);
  }

  // what is XORed to the chunk's number in staged row r
  static __device__ __forceinline__ int swizzle(int r) {
    if (!TR) return (r >> 1) & 7;
    if (ES != 2) return 0;
    return CPR == 8 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
  }

  // Where stage `st` begins, for the passes that follow: (TR) the buffer, else the lane's offset.
  struct Stage { const char* base; long long bytes; unsigned off; int k0; };
  __device__ __forceinline__ Stage at(int st) const {
    Stage g;
    if constexpr (TR) {
      const long long k0 = (long long)st * KST, left = len - k0;
      g.base = base + k0 * ld;
      g.bytes = left > 0 && across > 0 ? (min(left, (long long)KST) - 1) * ld + (long long)across * ES : 0;
      g.off = off;
      g.k0 = 0;
    } else {
      g.base = base;
      g.bytes = across > 0 ? (long long)(across - 1) * ld + (long long)len * ES : 0;
      g.k0 = st * 128;
      g.off = st * KST + chunk * EPC < len ? off : OUTSIDE;
    }
    return g;
  }
  // Pass i of stage `st` into LDS at `to`.  (The bound of a buffer holds for lane offset + scalar offset.)
  __device__ __forceinline__ void pass(char* to, const Stage& g, int st, int i) const {
    if constexpr (VEC) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is reserved, and named as overwritten all the same)
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass refuses 16 bytes here, and with that drops some kernels' stubs)
      const int soff = __builtin_amdgcn_readfirstlane(g.k0 + i * RPP * (int)ld);
      char* const lds = to + i * NTH * 16 + wave * 1024;
      if constexpr (UNSEEN) {
        // The low half of an LDS pointer is its offset.  A scalar register that a vector instruction wrote (readfirstlane)
        // may be read by a load five wait states later, which the compiler sees to for loads that it knows: s_mov's
        // one and s_nop's four (input gradient of 8 groups of 512 x 1024 x 1024: 18.7 us, without them 18.2).
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                     :: "s"(__builtin_amdgcn_readfirstlane((int)(unsigned long long)lds)), "v"(g.off),
                        "s"(buffer_words(g.base, g.bytes)), "s"(soff) : "memory", "m0");
      } else {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer_of(g.base, g.bytes), (lds_void*)lds, 16, (int)g.off, soff, 0, 0);
      }
#endif
#pragma clang diagnostic pop
    } else {
      typedef typename std::conditional<ES == 1, unsigned char,
                                        typename std::conditional<ES == 2, unsigned short, unsigned>::type>::type elem_t;
      typedef elem_t chunk_t __attribute__((ext_vector_type(EPC)));
      const int r = row + i * RPP;
      const long long k = TR ? (long long)st * KST + r : (long long)st * KST + chunk * EPC;
      const int a = TR ? chunk * EPC : r;
      const char* const p = base + (TR ? k * ld + (long long)a * ES : a * ld + k * ES);
      const long long left = k >= len || a >= across ? 0 : TR ? across - a : len - k;  // elements that exist
      chunk_t v;
      if (left >= EPC) {
        __builtin_memcpy(&v, p, 16);
      } else {
#pragma unroll
        for (int j = 0; j < EPC; ++j) v[j] = j < left ? ((const elem_t*)p)[j] : (elem_t)0;
      }
      *(chunk_t*)(to + i * NTH * 16 + tid * 16) = v;
    }
  }
  __device__ __forceinline__ void issue(char* to, int st) const {
    const Stage g = at(st);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) pass(to, g, st, i);
  }
};

// All but the last `later` of this wave's loads to LDS have landed and its LDS reads and writes are done; then
// the same of every wave.  (Not VEC: what a thread staged itself it has written by then.)
template <bool VEC, int later>
__device__ __forceinline__ void stage_barrier() {
  static_assert(later <= 63, "a six-bit counter");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(VEC ? later : 0) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// No load to LDS is on its way any more: before the LDS is another workgroup's.
__device__ __forceinline__ void drain_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Adds the sums of KG groups of NTH threads that made the same tile, in the groups' order; group 0 has them then.
// `sums`: (KG - 1) * NTH * 64 bytes that nobody else uses any more.
template <int KG, int NTH, int MT, int NT>
__device__ __forceinline__ void join_groups(float* sums, int group, int tid, f32x16 (&acc)[MT][NT]) {
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      __syncthreads();
      if (group > 0) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(f32x4*)&sums[(((group - 1) * 4 + g) * NTH + tid) * 4] =
              f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
      }
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int o = 0; o < KG - 1; ++o)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 v = *(const f32x4*)&sums[((o * 4 + g) * NTH + tid) * 4];
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][4 * g + r] += v[r];
          }
      }
    }
}

// ---- result -----------------------------------------------------------------------------------------

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
  bf16x2 v;
  v[0] = (__bf16)a;
  v[1] = (__bf16)b;
  return __builtin_bit_cast(unsigned, v);
}

// 16 (8) bytes wherever they lie: global memory takes them at any address.
template <class V>
__device__ __forceinline__ void store_at(char* p, V v) { __builtin_memcpy(p, &v, sizeof(V)); }

// LDS writes of a wave's lanes before it, reads of others after it (they happen in the program's order: this holds the
// compiler to it).
__device__ __forceinline__ void lanes_in_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A wave's MT x NT result tiles of 32 x 32: lane l holds row m = l & 31, register r column 8 (r >> 2) + 4 (l >> 5) +
// (r & 3).  They go to memory through LDS, 32 rows at a time, so that a store writes whole rows of the wave's
// columns, 16 bytes a lane: straight from the registers an instruction would write 32 bytes of each of 32
// rows (weight gradient of 32 groups of 2048 x 2048: 246 us, straight 277).
//   lds   LDS that nobody else uses any more, STORE_BYTES a wave
//   y     the wave's first row and column of the result, pitch ldy bytes; `rows`, `cols`: how many exist
//   add   the result is added to what is there (fp32)
template <bool BF16, int NT>
struct Store {
  static constexpr int ES = BF16 ? 2 : 4, ROW = NT * 32 * ES, PITCH = ROW + 16, BYTES = 32 * PITCH;
  static constexpr int LANES = ROW / 16, STEP = 64 / LANES;  // lanes a row, rows an instruction

  template <int MT>
  static __device__ __forceinline__ void run(const f32x16 (&acc)[MT][NT], char* lds, char* y, long long ldy, int rows, int cols,
                                             bool add = false) {
    const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
    const int col = (lane % LANES) * (16 / ES);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (i * 32 >= rows) break;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          char* const to = lds + li * PITCH + (j * 32 + 8 * g + 4 * lh) * ES;
          const f32x16& v = acc[i][j];
          if constexpr (BF16) *(u32x2*)to = u32x2{pack_bf16(v[4 * g], v[4 * g + 1]), pack_bf16(v[4 * g + 2], v[4 * g + 3])};
          else *(f32x4*)to = f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
        }
      lanes_in_order();
#pragma unroll
      for (int t = 0; t < 32 / STEP; ++t) {
        const int r = t * STEP + lane / LANES, m = i * 32 + r;
        u32x4 v = *(const u32x4*)(lds + r * PITCH + col * ES);
        if (m < rows && col < cols) {
          char* const to = y + m * ldy + (long long)col * ES;
          if (col + 16 / ES <= cols) {
            if (!BF16 && add) {
              f32x4 old;
              __builtin_memcpy(&old, to, 16);
              v = __builtin_bit_cast(u32x4, __builtin_bit_cast(f32x4, v) + old);
            }
            store_at(to, v);
          } else {
#pragma unroll
            for (int e = 0; e < 16 / ES; ++e)
              if (col + e < cols) {
                if constexpr (BF16) ((unsigned short*)to)[e] = (unsigned short)(v[e >> 1] >> (16 * (e & 1)));
                else ((float*)to)[e] = __uint_as_float(v[e]) + (add ? ((const float*)to)[e] : 0.0f);
              }
          }
        }
      }
      lanes_in_order();
    }
  }
};

// Workgroups with this much LDS that an XCD of this process holds at a time.
inline int slots_per_xcd(int lds_bytes) {
  const int n = c2d_available_cus() / 8 * (160 * 1024 / lds_bytes);
  return n > 0 ? n : 1;
}

inline bool sizes_fit(int a, int b, int c) { return a <= C2DP_MAX_SIZE && b <= C2DP_MAX_SIZE && c <= C2DP_MAX_SIZE; }

// Every workgroup looks through the offsets for its tile: 65536 groups of one row, 64 x 64, take 35 ms (input gradient 69), 4096
// 0.16 ms, 2^20 would take many seconds.
inline bool groups_fit(int groups) { return groups <= C2DP_MAX_GROUPS; }

inline bool aligned16(const void* p, long long pitch_bytes) {
  return ((unsigned long long)p & 15) == 0 && (pitch_bytes & 15) == 0;
}

}  // namespace
}  // namespace c2d_pr
