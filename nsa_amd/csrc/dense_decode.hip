// Dense decode attention: the one new token of every sequence attends all cached tokens (or the last `window`
// of them), contiguous or paged cache, the same layouts as the sparse decode step:
//   q [B][Hq][Dk]; keys row-major [page][64][Hkv][Dk] (or [B][ctx_cap][Hkv][Dk]); values key-contiguous
//   [page][Hkv][Dv][64] (or [B][Hkv][Dv][ctx_cap]); ctx_lens [B] = tokens including the current one
//   s_j = scale * <q_h, k_j> over the visible j, m = max s_j, l = sum exp(s_j - m)
//   out_h = sum exp(s_j - m) v_j / l,  lse_h = m + ln l;  nothing visible: out = 0, lse = -inf
//
// Bound by reading K and V once: the matrix instructions of a 32-key chunk take about a tenth of the time its
// bytes need (128 / 128 channels, 16 heads), so one wavefront simply loads its fragments straight from memory
// into the operand registers, with no LDS in the loop: the next chunk's keys are on their way during the softmax and the
// second product, its values from there on.
//
// Work split: a (sequence, kv head) with few others beside it would leave most of the 256 CUs idle, and a ragged
// batch would wait for its longest sequence.  So the pages of ALL sequences are cut into runs ("units") of the same
// number of pages C, and a workgroup takes one unit of one kv head.  C follows from ctx_lens on the device, every
// wavefront computes the same plan from them, so that a captured graph stays right as the sequences grow; the host
// only fixes an upper bound of the number of units.  A sequence of more than one unit leaves one partial softmax
// state (fp32) per unit, and a second kernel joins them; the others are finished by the first kernel.
#include <type_traits>

#include "decode_common.h"

namespace nsa {

constexpr int kDenseWaves = 4;         // wavefronts of a workgroup that shares a sequence with others
constexpr int kDenseWholeWaves = 8;    // and of one that takes a whole (short) sequence
constexpr int kDenseWholePages = 16;
constexpr int kDenseMinPages = 2;      // fewest pages per unit: one 32-key chunk for each wavefront

struct DenseSpan { int n, lo, first, pages; };   // tokens, first visible token, its page, pages to read

__device__ __forceinline__ DenseSpan dense_span(int len, int cap, int window) {
  DenseSpan s;
  s.n = min(max(len, 0), cap);
  s.lo = window > 0 ? max(0, s.n - window) : 0;
  s.first = s.lo >> 6;
  s.pages = ((s.n + 63) >> 6) - s.first;
  return s;
}
// Sum over the wavefront, in every lane: rotations inside the 16-lane rows, then the two row exchanges.
__device__ __forceinline__ int wave_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x128, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x124, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x122, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x121, 0xF, 0xF, true);
  auto r = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
  x = (int)(r[0] + r[1]);
  r = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
  return (int)(r[0] + r[1]);
}
// Inclusive prefix sum over the wavefront: shifts inside the rows, then the last lane of row 0 and 2 added to the row
// behind it, and that of row 1 to rows 2 and 3.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
  return x;
}
__device__ __forceinline__ int dense_units_of(int pages, int C) { return max(1, (int)((unsigned)(pages + C - 1) / (unsigned)C)); }
// Pages per unit: the pages of all sequences over the units aimed at, and more where the sequences' last, shorter units
// would make a second round of workgroups: each step takes C up by the excess, and by a 16th at least after the third,
// until the units are no more than aimed at, which they are at one per sequence.  (32 / 4 heads of 128 bf16, us, with the
// first C, after three steps and after all of them: 28 x 8192 tokens 143, 100, 100; 33 x 8192 171, 190, 155; 38 x 32768 747,
// 1150, 583; 37 sequences of 0 to 16001 184, 139, 140; 50 of 0 to 8192 131, 114, 121.)  sum_b max(1, ceil(pages_b / C)) is at
// most units + batch for the first C already, which is what the grid and the workspace hold.
__device__ __forceinline__ int dense_unit_pages(const DenseDecodeArgs& a) {
  const int lane = __lane_id();
  if (a.batch == 1) {
    const unsigned pages = dense_span(a.ctx_lens[0], a.ctx_cap, a.window).pages;
    return max(kDenseMinPages, (int)((pages + a.units - 1) / (unsigned)a.units));
  }
  int total = 0, mine = 0;
  for (int b = lane; b < a.batch; b += 64) {
    mine = dense_span(a.ctx_lens[b], a.ctx_cap, a.window).pages;
    total += mine;
  }
  total = wave_sum(total);
  const unsigned aim = (unsigned)a.units;
  int C = max(kDenseMinPages, (int)(((unsigned)total + aim - 1) / aim));
  if (a.batch > 64 || a.batch >= a.units) return C;
#pragma unroll 1
  for (int step = 0;; ++step) {
    const unsigned got = wave_sum(lane < a.batch ? dense_units_of(mine, C) : 0);
    if (got <= aim) break;
    C = max(C + (step < 3 ? 1 : 1 + C / 16), (int)(((uint64_t)C * got + aim - 1) / aim));
  }
  return C;
}

// How far below the running maximum the reference of the exponentials is put.  In 32 bits and bfloat16 it goes 2^8 above, by
// which the maximum may then grow before the sums are rescaled, so that no probability passes 1 and the sums end where those
// of the formula do (with probabilities of up to 2^8 values of 2^119 overflowed).  float16 ends at 2^-24 and its values at
// 2^16: with probabilities of up to 2^(7 + 8) it keeps what lies 2^-31 below the maximum, which thousands of such keys add up
// to (one key that takes nearly all the weight, 1000 others at 2^-26 each: 1/8 of their sum was lost without).
template <typename T> constexpr float kDenseBelow = -kMaxSlackLog2;
template <> constexpr float kDenseBelow<f16_t> = 7.0f;

// A 16-bit value that is no number or infinite, by its bits (the library is compiled with the promise that no NaN occurs).
template <typename T> constexpr unsigned kExpMask16 = 0x7f80u;
template <> constexpr unsigned kExpMask16<f16_t> = 0x7c00u;
template <typename T>
__device__ __forceinline__ bool odd16(T x) { return (__builtin_bit_cast(uint16_t, x) & kExpMask16<T>) == kExpMask16<T>; }

// Fragments of one 32-key chunk and the two products on them.  Visible keys of the chunk [cb, cb + 32) are lo..n-1.
// Whatever a page holds outside them (rows of a sequence that had the page before, infinities, NaN) must not reach the
// sums: their scores are replaced, and their values too, since 0 * inf is NaN.
template <typename T, int DK, int NT>
__device__ __forceinline__ void dense_scores(const vec8_t<T> (&k0)[DK / 32], const vec8_t<T> (&k1)[DK / 32],
                                             const vec8_t<T> (&q)[NT][DK / 32], float (&s)[NT][8]) {
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    f32x4_t s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < DK / 32; ++kk) {
      s0 = mma16(k0[kk], q[j][kk], s0);
      s1 = mma16(k1[kk], q[j][kk], s1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) { s[j][i] = s0[i]; s[j][4 + i] = s1[i]; }
  }
}
// ODD: among the values there are infinities or NaN, which the split probabilities would turn into NaN (infinity times a
// rest of 0, or of the other sign).  The keys are gone through twice then: with the finite values alone (`finite`), and with
// the others alone, each with weight 1 unless its probability is 0.
template <bool ODD, typename T, int DK, int DV, int NT>
__device__ __forceinline__ void dense_values(DecState<T, DK, DV> (&st)[NT], vec8_t<T> (&v)[DV / 16],
                                             const float (&s)[NT][8], int cb, int lo, int n, float c, int g, bool finite) {
  const bool whole = cb >= lo && cb + 32 <= n;
  if (!whole) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = cb + 8 * g + i;
      if (key < lo || key >= n) {
#pragma unroll
        for (int t = 0; t < DV / 16; ++t) v[t][i] = (T)0.0f;
      }
    }
  }
  if constexpr (ODD) {
#pragma unroll
    for (int t = 0; t < DV / 16; ++t)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (odd16<T>(v[t][i]) == finite) v[t][i] = (T)0.0f;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float p[8];
    float mx = kNegInf;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = cb + 8 * g + i;
      const float x = s[j][i] * c;
      mx = fmaxf(mx, whole || (key >= lo && key < n) ? x : kNegInf);
    }
    // The reference of the exponentials follows the maximum only when that has grown by more than 2^8 (the first chunk, and
    // hardly ever again): probabilities stay within 1 (float16: 2^15), and the sums are not rescaled at every chunk.
    mx = colgroup_max(mx);
    constexpr float below = kDenseBelow<T>;
    if (__any(mx > st[j].m + (kMaxSlackLog2 + below))) {
      const float m_new = fmaxf(st[j].m, mx - below);
      const float alpha = fast_exp2(st[j].m - (m_new == kNegInf ? 0.f : m_new));
      st[j].m = m_new;
      st[j].l *= alpha;
#pragma unroll
      for (int t = 0; t < DV / 16; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) st[j].o[t][i] *= alpha;
    }
    const float mref = st[j].m == kNegInf ? 0.f : st[j].m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = cb + 8 * g + i;
      const float x = fast_exp2(fmaf(s[j][i], c, -mref));
      p[i] = whole || (key >= lo && key < n) ? x : 0.f;
      if (ODD && !finite) p[i] = p[i] == 0.f ? 0.f : 1.f;
      sum += p[i];
    }
    if (!ODD || finite) st[j].l += sum;
    // The second product takes 16-bit probabilities: a rounded one and what the rounding left, each with its own matrix
    // instructions (the loads are the bound), so that only the rounding of the result remains.
    const vec8_t<T> pb = pack8<T>(p);
    vec8_t<T> rest = zero8<T>();
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) rest[i] = (T)(p[i] - (float)pb[i]);
    }
#pragma unroll
    for (int t = 0; t < DV / 16; ++t) {
      st[j].o[t] = mma16(v[t], pb, st[j].o[t]);
      if constexpr (sizeof(T) == 2) {
        if (!ODD || finite) st[j].o[t] = mma16(v[t], rest, st[j].o[t]);
      }
    }
  }
}

// Registers (32-bit, per lane) of one chunk's fragments, of the queries and sums of NT head tiles, and what else there is.
template <typename T, int DK, int DV, int NT> constexpr int kDenseRegs =
    (2 * (DK / 32) + DV / 16) * 2 * (int)sizeof(T) + NT * ((DK / 32) * 2 * (int)sizeof(T) + DV / 4) + 48;
// Wavefronts per SIMD that the register file (512) then holds, of W of a workgroup at least.  The count is short by what a
// second tile needs besides: 64 / 64 with two tiles and 32 / 32 with four (16-bit) come out at four wavefronts and spill 39
// to 73 registers, and fp32 192 / 128 at the eight wavefronts of a whole sequence, which need two per SIMD, spills 40.
template <typename T, int DK, int DV, int NT, int W> constexpr int kDenseOccupancy =
    kDenseRegs<T, DK, DV, NT> <= 128 ? 4 : kDenseRegs<T, DK, DV, NT> <= 168 ? 3 :
    kDenseRegs<T, DK, DV, NT> <= 256 || W > 4 ? 2 : 1;

// NT: 16-head tiles of the GQA group that share the loaded keys and values.  grid: unit * (hkv * head blocks) + those
template <typename T, int DK, int DV, int NT, int W>
__global__ void __launch_bounds__(W * 64, (kDenseOccupancy<T, DK, DV, NT, W>))
dense_decode_kernel(const DenseDecodeArgs a) {
  constexpr int kPitch = DV + 4;
  __shared__ float plane[W][16][kPitch];
  __shared__ float ml[W][16][2];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g = lane >> 4;
  const int G = a.hq / a.hkv, blocks = (G + 16 * NT - 1) / (16 * NT);
  const int per = a.hkv * blocks;
  const int unit = blockIdx.x / per, hb = blockIdx.x % per;
  const int h = hb / blocks, row0 = (hb % blocks) * 16 * NT;

  // the plan: which sequence this unit belongs to, and which of its units it is
  int b = a.part == nullptr ? unit : -1, idx = 0, count = 1, before = 0;
  const int C = a.part == nullptr ? (a.ctx_cap + 63) / 64 : dense_unit_pages(a);
  for (int b0 = 0; b0 < a.batch && b < 0; b0 += 64) {
    const int mine = b0 + lane;
    const int nu = mine < a.batch ? dense_units_of(dense_span(a.ctx_lens[mine], a.ctx_cap, a.window).pages, C) : 0;
    const int incl = wave_scan(nu);
    const int run = __builtin_amdgcn_readlane(incl, 63);
    if (unit < before + run) {
      const unsigned long long hit = __ballot(before + incl > unit);
      const int at = __ffsll((long long)hit) - 1;
      b = b0 + at;
      count = __builtin_amdgcn_readlane(nu, at);
      idx = unit - before - (__builtin_amdgcn_readlane(incl, at) - count);
    }
    before += run;
  }
  if (b < 0) return;                                   // the bound on the number of units is not always reached
  const DenseSpan sp = dense_span(a.ctx_lens[b], a.ctx_cap, a.window);
  const int p0 = sp.first + idx * C, p1 = min(sp.first + sp.pages, p0 + C);

  DecState<T, DK, DV> st[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) dec_reset(st[j]);

  // one run over this wavefront's chunks of the unit
  auto stream = [&](auto odd, bool finite, int lane) {
    constexpr bool kOdd = decltype(odd)::value;
    const int n16 = lane & 15, g = lane >> 4;
    const T* kbase = reinterpret_cast<const T*>(a.k) + (long)h * DK + 8 * g;
    const T* vbase = reinterpret_cast<const T*>(a.v);
    const long krow = (long)a.hkv * DK;
    const bool paged = a.block_table != nullptr;
    const long vrow = paged ? 64 : a.ctx_cap;
    const int32_t* table = paged ? a.block_table + (long)b * a.max_pages : nullptr;

    vec8_t<T> q[NT][DK / 32];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int head = h * G + min(row0 + 16 * j + n16, G - 1);
      const T* qp = reinterpret_cast<const T*>(a.q) + ((long)b * a.hq + head) * DK + 8 * g;
#pragma unroll
      for (int kk = 0; kk < DK / 32; ++kk) q[j][kk] = load8(qp + 32 * kk);
    }
    const float c = a.scale * kLog2e;

    // chunk i of this wavefront covers keys 64 p0 + 32 (w + W i) ..; 64 page ids at a time sit in the lanes
    int ids_at = p0, ids = 0;
    if (paged && p0 + lane < p1) ids = table[p0 + lane];
    auto page_of = [&](int cb) -> int {
      const int p = cb >> 6;
      if (p - ids_at >= 64) {
        ids_at = p;
        ids = p + lane < p1 ? table[p + lane] : 0;
      }
      // an id outside the pool would fault: read page 0 instead (the caller's table is wrong)
      const int id = __builtin_amdgcn_readlane(ids, p - ids_at);
      return (unsigned)id < (unsigned)a.num_pages ? id : 0;
    };
    vec8_t<T> k0[DK / 32], k1[DK / 32], v[DV / 16];
    auto load_keys = [&](int cb, int id) {
      const T* kp = kbase + (paged ? (long)id * 64 + (cb & 63) : (long)b * a.ctx_cap + cb) * krow;
      const T* k0p = kp + chunk_key_of_row(0, n16) * krow;
      const T* k1p = kp + chunk_key_of_row(1, n16) * krow;
#pragma unroll
      for (int kk = 0; kk < DK / 32; ++kk) { k0[kk] = load8(k0p + 32 * kk); k1[kk] = load8(k1p + 32 * kk); }
    };
    auto load_values = [&](int cb, int id) {
      const T* vp = vbase + ((long)(paged ? id : b) * a.hkv + h) * DV * vrow + (paged ? (cb & 63) : cb) + (long)n16 * vrow + 8 * g;
#pragma unroll
      for (int t = 0; t < DV / 16; ++t) v[t] = load8(vp + 16 * t * vrow);
    };
    // the next chunk's keys are requested as soon as the scores have used this one's, its values after the second
    // product: one set of registers, and loads of this wavefront are always in flight
    const int end = min(p1 * 64, sp.n);
    int cb = p0 * 64 + 32 * w;
    if (cb >= end) return;
    int id = paged ? page_of(cb) : 0;
    load_keys(cb, id);
    load_values(cb, id);
    while (true) {
      float s[NT][8];
      dense_scores<T, DK, NT>(k0, k1, q, s);
      const int next = cb + 32 * W;
      if (next < end) {
        id = paged ? page_of(next) : 0;
        if (!kOdd) load_keys(next, id);
      }
      dense_values<kOdd, T, DK, DV, NT>(st, v, s, cb, sp.lo, sp.n, c, g, finite);
      if (next >= end) break;
      if (kOdd) load_keys(next, id);         // it has no registers to spare
      load_values(next, id);
      cb = next;
    }
  };
  stream(std::false_type(), true, lane);
  if constexpr (sizeof(T) == 2) {
    // once something is infinite or no number, the sums stay so: only then the unit is read again
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int t = 0; t < DV / 16; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(st[j].o[t][i]) << 1);
    if (__any(top >= 0xff000000u)) {
#pragma unroll
      for (int j = 0; j < NT; ++j) dec_reset(st[j]);
#pragma unroll 1
      for (int pass = 0; pass < 2; ++pass) {
        int again = lane;
        asm volatile("" : "+v"(again));      // what follows from it is worked out anew, not kept in registers all along
        stream(std::true_type(), pass == 0, again);
      }
    }
  }

  // join the wavefronts, 16 heads at a time
  const long slot = (long)unit * per + hb;
  const int rows = min(G - row0, 16 * NT);
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    if (j > 0) __syncthreads();
    const float l = colgroup_sum(st[j].l);
    if (g == 0) { ml[w][n16][0] = st[j].m; ml[w][n16][1] = l; }
    __syncthreads();
    float M = kNegInf;
#pragma unroll
    for (int x = 0; x < W; ++x) M = fmaxf(M, ml[x][n16][0]);
    const float own = fast_exp2(st[j].m - (M == kNegInf ? 0.f : M));
#pragma unroll
    for (int t = 0; t < DV / 16; ++t) {
      f32x4_t o = st[j].o[t];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= own;
      *reinterpret_cast<f32x4_t*>(&plane[w][n16][16 * t + 4 * g]) = o;
    }
    __syncthreads();
    for (int item = threadIdx.x; item < 16 * (DV / 4); item += W * 64) {
      const int r = item / (DV / 4), d = 4 * (item % (DV / 4));
      if (16 * j + r >= rows) break;
      float Mr = kNegInf, L = 0.f;
#pragma unroll
      for (int x = 0; x < W; ++x) Mr = fmaxf(Mr, ml[x][r][0]);
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < W; ++x) {
        L += ml[x][r][1] * fast_exp2(ml[x][r][0] - (Mr == kNegInf ? 0.f : Mr));
        o += *reinterpret_cast<const f32x4_t*>(&plane[x][r][d]);
      }
      if (count > 1) {
        float* po = a.part + (slot * (16 * NT) + 16 * j + r) * DV + d;
        *reinterpret_cast<f32x4_t*>(po) = o;
        if (d == 0) {
          float* pm = a.part_ml + (slot * (16 * NT) + 16 * j + r) * 2;
          pm[0] = Mr;
          pm[1] = L;
        }
      } else {
        const float inv = L == 0.f ? 0.f : 1.0f / L;     // not L > 0: a NaN among the scores has to come through
        const long row = (long)b * a.hq + h * G + row0 + 16 * j + r;
        T* dst = reinterpret_cast<T*>(a.out) + row * DV + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[i] = (T)(o[i] * inv);
        if (a.lse != nullptr && d == 0) a.lse[row] = L == 0.f ? kNegInf : (Mr + __log2f(L)) * (1.0f / kLog2e);
      }
    }
  }
}

// One (sequence, query head) per workgroup: joins the partial states of the sequence's units.
template <typename T, int DV>
__global__ void __launch_bounds__(256)
dense_decode_join_kernel(const DenseDecodeArgs a, int rows_per_slot, int blocks) {
  constexpr int kLanes = DV / 4, kGroups = 256 / kLanes;
  __shared__ float acc[kGroups][DV];
  __shared__ float red[kGroups][2];
  const int b = blockIdx.x / a.hq, head = blockIdx.x % a.hq;
  const int lane = threadIdx.x & 63;
  const int C = dense_unit_pages(a);
  int u0 = 0;
  for (int x = lane; x < b; x += 64) u0 += dense_units_of(dense_span(a.ctx_lens[x], a.ctx_cap, a.window).pages, C);
  u0 = wave_sum(u0);
  const int count = dense_units_of(dense_span(a.ctx_lens[b], a.ctx_cap, a.window).pages, C);
  // more units than there is room for: only if another stream changed the lengths between the two kernels
  if (count <= 1 || u0 + count > a.units + a.batch) return;
  const int G = a.hq / a.hkv, h = head / G, r = head % G;
  const int per = a.hkv * blocks, hb = h * blocks + r / rows_per_slot;
  const long step = (long)per * rows_per_slot;
  const long first = ((long)u0 * per + hb) * rows_per_slot + r % rows_per_slot;
  // every kLanes threads run over their own units, eight at a time so that the loads of a round travel together
  const int x = threadIdx.x % kLanes, y = threadIdx.x / kLanes;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float m = kNegInf, l = 0.f;
  for (int u = y; u < count; u += 8 * kGroups) {
    float um[8], ul[8];
    f32x4_t uo[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const long at = first + min(u + k * kGroups, count - 1) * step;
      um[k] = a.part_ml[at * 2];
      ul[k] = a.part_ml[at * 2 + 1];
      uo[k] = *reinterpret_cast<const f32x4_t*>(a.part + at * DV + 4 * x);
    }
    float mx = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (u + k * kGroups >= count) {                      // the last unit once more: infinity times a weight of 0 is NaN
        um[k] = kNegInf;
        uo[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
      mx = fmaxf(mx, um[k]);
    }
    const float ref = mx == kNegInf ? 0.f : mx;
    const float alpha = fast_exp2(m - ref);
    m = mx;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= alpha;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float wgt = fast_exp2(um[k] - ref);
      l = fmaf(ul[k], wgt, l);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(uo[k][i], wgt, o[i]);
    }
  }
  *reinterpret_cast<f32x4_t*>(&acc[y][4 * x]) = o;
  if (x == 0) { red[y][0] = m; red[y][1] = l; }
  __syncthreads();
  if (threadIdx.x >= DV) return;
  float M = kNegInf, sum = 0.f, L = 0.f;
#pragma unroll
  for (int k = 0; k < kGroups; ++k) M = fmaxf(M, red[k][0]);
  const float ref = M == kNegInf ? 0.f : M;
#pragma unroll
  for (int k = 0; k < kGroups; ++k) {
    const float wgt = fast_exp2(red[k][0] - ref);
    sum = fmaf(acc[k][threadIdx.x], wgt, sum);
    L = fmaf(red[k][1], wgt, L);
  }
  const long row = (long)b * a.hq + head;
  reinterpret_cast<T*>(a.out)[row * DV + threadIdx.x] = (T)(L == 0.f ? 0.f : sum / L);
  if (a.lse != nullptr && threadIdx.x == 0) a.lse[row] = L == 0.f ? kNegInf : (M + __log2f(L)) * (1.0f / kLog2e);
}

// 16-head tiles that share one pass over the keys: the whole group up to 64 heads (32 in fp32, whose fragments take
// twice the registers); larger groups read the keys once per block.  Four tiles leave one wavefront per SIMD and join in
// four rounds, so where there are few pages blocks of two are faster, although both read them (64 / 1 heads of 128 bf16,
// four tiles against two: 2 sequences of 8192 tokens 20.8 and 14.9 us, 2 of 32768 27.4 and 23.5, 16 of 32768 91 and 94;
// 192 / 128: 22.4 and 15.9, 29.8 and 25.5, 97 and 115).
static int dense_tiles(const DenseDecodeArgs& a, long pages) {
  const int G = a.hq / a.hkv;
  if (G <= 16) return 1;
  return G <= 32 || a.dtype == 1 || pages * a.hkv <= 1024 ? 2 : 4;
}

DensePlan dense_decode_plan(const DenseDecodeArgs& a) {
  DensePlan p;
  const int G = a.hq / a.hkv;
  const int cap_pages = (a.ctx_cap + 63) / 64;
  const int span = a.window > 0 ? (int)min((long)cap_pages, ((long)a.window + 62) / 64 + 1) : cap_pages;
  p.tiles = dense_tiles(a, (long)a.batch * span);
  p.blocks = (G + 16 * p.tiles - 1) / (16 * p.tiles);
  const long per = (long)a.hkv * p.blocks;
  // One workgroup per CU where its four wavefronts keep 64 KB of loads in flight, more where a chunk is smaller: few long
  // streams reach more of the memory's rate than many (64 sequences of 32768 tokens, 128 / 128 bf16: 722 us with 256
  // workgroups, 767 with 512, 791 with 768; 16 of them at 64 / 64: 108, 102, 105 us)
  const long in_flight = 32L * kDenseWaves * (a.dk + a.dv) * (a.dtype == 1 ? 4 : 2);
  const long workgroups = 256 * min(4L, max(1L, 65536 / in_flight));
  // With more sequences than that they come in several rounds anyway; a third of a sequence per unit keeps the last round
  // short (32 / 4 heads of 128 bf16, one unit per sequence against three: 65 sequences of 8192 323 and 247 us, 100 of up
  // to 8192 213 and 187, 200 of up to 4096 220 and 207; 128 of 4096, which are two rounds to the dot, 200 and 222).
  const long aim = a.batch > workgroups / per ? 3L * a.batch : workgroups / per;
  p.units = (int)max(1L, min(aim, (long)a.batch * span));
  // A short capacity is not worth a second launch: 8 wavefronts take the whole sequence.  16 / 4 heads, split against
  // whole, us: one sequence of 512 tokens, 64 / 64 bf16 9.0, 6.7, of 1024 8.8, 10.3; 128 / 128 bf16
  // 256 tokens 9.7, 6.7, 512 9.7, 10.3; 64 / 64 fp32 256 tokens 10.1, 6.9, 512 10.1, 11.8.  64 sequences fill the card
  // without a split: 1024 tokens, 128 / 128 bf16 27.0, 23.4, fp32 54.6, 52.2.
  const long span_bytes = 64L * span * (a.dk + a.dv) * (a.dtype == 1 ? 4 : 2);
  p.whole = p.tiles == 1 && (span_bytes <= 200 << 10 || (span <= kDenseWholePages && (long)a.batch * a.hkv >= 256));
  p.split = !p.whole && span > kDenseMinPages;         // otherwise every sequence is one unit
  if (!p.split) p.units = a.batch;
  p.slots = ((long)p.units + a.batch) * per;
  p.rows = 16 * p.tiles;
  return p;
}

long dense_decode_workspace_bytes(const DenseDecodeArgs& a) {
  const DensePlan p = dense_decode_plan(a);
  return p.split ? p.slots * p.rows * (long)(a.dv + 2) * (long)sizeof(float) : 0;
}

// The head dims that launch_dense builds.
bool dense_decode_dims_ok(int dk, int dv) {
  return (dk == dv && (dk == 32 || dk == 64 || dk == 128)) || (dk == 192 && dv == 128);
}

template <typename T, int DK, int DV, int NT>
static int launch_dense_n(const DenseDecodeArgs& a, const DensePlan& p, hipStream_t st) {
  const long units = p.split ? (long)p.units + a.batch : a.batch;
  const long wgs = units * a.hkv * p.blocks;
  if (wgs > 0x7fffffffL || (long)a.batch * a.hq > 0x7fffffffL) return -5;
  if constexpr (NT == 1) {
    if (p.whole) {
      hipLaunchKernelGGL((dense_decode_kernel<T, DK, DV, NT, kDenseWholeWaves>), dim3((unsigned)wgs),
                         dim3(kDenseWholeWaves * 64), 0, st, a);
      return 0;
    }
  }
  hipLaunchKernelGGL((dense_decode_kernel<T, DK, DV, NT, kDenseWaves>), dim3((unsigned)wgs), dim3(kDenseWaves * 64), 0, st, a);
  if (p.split)
    hipLaunchKernelGGL((dense_decode_join_kernel<T, DV>), dim3((unsigned)(a.batch * a.hq)), dim3(256), 0, st, a, p.rows,
                       p.blocks);
  return 0;
}

template <typename T, int DK, int DV>
static int launch_dense_t(const DenseDecodeArgs& a, const DensePlan& p, hipStream_t st) {
  if (p.tiles == 1) return launch_dense_n<T, DK, DV, 1>(a, p, st);
  if (p.tiles == 2) return launch_dense_n<T, DK, DV, 2>(a, p, st);
  if constexpr (sizeof(T) == 2) return launch_dense_n<T, DK, DV, 4>(a, p, st);
  return -2;
}

template <typename T>
static int launch_dense(const DenseDecodeArgs& a, const DensePlan& p, hipStream_t st) {
  switch (a.dk * 1000 + a.dv) {
    case 32032: return launch_dense_t<T, 32, 32>(a, p, st);
    case 64064: return launch_dense_t<T, 64, 64>(a, p, st);
    case 128128: return launch_dense_t<T, 128, 128>(a, p, st);
    case 192128: return launch_dense_t<T, 192, 128>(a, p, st);
    default: return -2;
  }
}

int launch_dense_decode(DenseDecodeArgs a, void* workspace, hipStream_t st) {
  const DensePlan p = dense_decode_plan(a);
  a.units = p.units;
  a.part = p.split ? reinterpret_cast<float*>(workspace) : nullptr;      // null: every sequence is one unit
  a.part_ml = p.split ? a.part + p.slots * p.rows * a.dv : nullptr;
  if (a.dtype == 0) return launch_dense<bf16_t>(a, p, st);
  if (a.dtype == 2) return launch_dense<f16_t>(a, p, st);
  return launch_dense<float>(a, p, st);
}

}  // namespace nsa
