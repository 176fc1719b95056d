// Dense decode attention: the one new token of every sequence attends all cached tokens (or the last `window`
// of them), contiguous or paged cache, the same layouts as the sparse decode step:
//   q [B][Hq][Dk]; keys row-major [page][64][Hkv][Dk] (or [B][ctx_cap][Hkv][Dk]); values key-contiguous
//   [page][Hkv][Dv][64] (or [B][Hkv][Dv][ctx_cap]); ctx_lens [B] = tokens including the current one
//   s_j = scale * <q_h, k_j> over the visible j, m = max s_j, l = sum exp(s_j - m)
//   out_h = sum exp(s_j - m) v_j / l,  lse_h = m + ln l;  nothing visible: out = 0, lse = -inf
//
// Bound by reading K and V once: the matrix instructions of a 32-key chunk take about a tenth of the time its
// bytes need (128 / 128 channels, 16 heads), so one wavefront simply loads its fragments straight from memory
// into the operand registers, two chunks ahead of the products, with no LDS in the loop.
//
// Work split: a (sequence, kv head) with few others beside it would leave most of the 256 CUs idle, and a ragged
// batch would wait for its longest sequence.  So the pages of ALL sequences are cut into runs ("units") of the same
// number of pages C, and a workgroup takes one unit of one kv head.  C follows from ctx_lens on the device, every
// wavefront computes the same plan from them, so that a captured graph stays right as the sequences grow; the host
// only fixes an upper bound of the number of units.  A sequence of more than one unit leaves one partial softmax
// state (fp32) per unit, and a second kernel joins them; the others are finished by the first kernel.
#include "decode_common.h"

namespace nsa {

constexpr int kDenseWaves = 4;
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
__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
  return x;
}
// Pages per unit: the pages of all sequences over the units aimed at.  sum_b max(1, ceil(pages_b / C)) is then at most
// units + batch, which is what the grid and the workspace hold.
__device__ __forceinline__ int dense_unit_pages(const DenseDecodeArgs& a) {
  int total = 0;
  for (int b = __lane_id(); b < a.batch; b += 64) total += dense_span(a.ctx_lens[b], a.ctx_cap, a.window).pages;
  total = wave_sum(total);
  return max(kDenseMinPages, (int)(((unsigned)total + a.units - 1) / (unsigned)a.units));
}
__device__ __forceinline__ int dense_units_of(int pages, int C) { return max(1, (int)((unsigned)(pages + C - 1) / (unsigned)C)); }

// Visible keys of the chunk [cb, cb + 32) are lo..n-1.  Whatever a page holds outside them (rows of a sequence that
// had the page before, infinities, NaN) must not reach the sums: their scores are replaced, and their values too,
// since 0 * inf is NaN.
template <typename T, int DK, int DV, int NT>
__device__ __forceinline__ void dense_attend(DecState<T, DK, DV> (&st)[NT], ChunkFrags<T, DK, DV>& f,
                                             const vec8_t<T> (&q)[NT][DK / 32], int cb, int lo, int n, float c, int g) {
  const bool whole = cb >= lo && cb + 32 <= n;
  if (!whole) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = cb + 8 * g + i;
      if (key < lo || key >= n) {
#pragma unroll
        for (int t = 0; t < DV / 16; ++t) f.v[t][i] = (T)0.0f;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    f32x4_t s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < DK / 32; ++kk) {
      s0 = mma16(f.k0[kk], q[j][kk], s0);
      s1 = mma16(f.k1[kk], q[j][kk], s1);
    }
    float s[8], p[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) { s[i] = s0[i]; s[4 + i] = s1[i]; }
    float mx = kNegInf;
    if (whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, s[i] * c);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = cb + 8 * g + i;
        const bool seen = key >= lo && key < n;
        mx = fmaxf(mx, seen ? s[i] * c : kNegInf);
      }
    }
    const float m_new = fmaxf(st[j].m, colgroup_max(mx));
    const float mref = m_new == kNegInf ? 0.f : m_new;
    const float alpha = fast_exp2(st[j].m - mref);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = cb + 8 * g + i;
      p[i] = fast_exp2(fmaf(s[i], c, -mref));
      if (!whole && (key < lo || key >= n)) p[i] = 0.f;
      sum += p[i];
    }
    st[j].l = st[j].l * alpha + sum;
    st[j].m = m_new;
    // probabilities are rounded to the tensors' type for the second product (at most 2^-9 of each at bf16, the
    // denominator keeps fp32); the sums stay in fp32
    const vec8_t<T> pb = pack8<T>(p);
#pragma unroll
    for (int t = 0; t < DV / 16; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) st[j].o[t][i] *= alpha;
      st[j].o[t] = mma16(f.v[t], pb, st[j].o[t]);
    }
  }
}

// Registers (32-bit, per lane) of one chunk's fragments, and of the queries and sums of NT head tiles.
template <typename T, int DK, int DV> constexpr int kDenseFragRegs = (2 * (DK / 32) + DV / 16) * 2 * (int)sizeof(T);
template <typename T, int DK, int DV, int NT> constexpr int kDenseTileRegs = NT * ((DK / 32) * 2 * (int)sizeof(T) + DV / 4);
// A second chunk in flight while one is worked on, where the register file (512 per lane) holds both.
template <typename T, int DK, int DV, int NT> constexpr bool kDenseAhead =
    2 * kDenseFragRegs<T, DK, DV> + kDenseTileRegs<T, DK, DV, NT> <= 384;
// Two wavefronts per SIMD where 256 registers hold that.
template <typename T, int DK, int DV, int NT> constexpr int kDenseOccupancy =
    2 * kDenseFragRegs<T, DK, DV> + kDenseTileRegs<T, DK, DV, NT> <= 192 ? 2 : 1;

// NT: 16-head tiles of the GQA group that share the loaded keys and values.  grid: unit * (hkv * head blocks) + those
template <typename T, int DK, int DV, int NT>
__global__ void __launch_bounds__(kDenseWaves * 64, (kDenseOccupancy<T, DK, DV, NT>))
dense_decode_kernel(const DenseDecodeArgs a) {
  constexpr int kPitch = DV + 4;
  __shared__ float plane[kDenseWaves][16][kPitch];
  __shared__ float ml[kDenseWaves][16][2];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g = lane >> 4;
  const int G = a.hq / a.hkv, blocks = (G + 16 * NT - 1) / (16 * NT);
  const int per = a.hkv * blocks;
  const int unit = blockIdx.x / per, hb = blockIdx.x % per;
  const int h = hb / blocks, row0 = (hb % blocks) * 16 * NT;

  // the plan: which sequence this unit belongs to, and which of its units it is
  const int C = dense_unit_pages(a);
  int b = -1, idx = 0, count = 0, before = 0;
  for (int b0 = 0; b0 < a.batch && b < 0; b0 += 64) {
    const int mine = b0 + lane;
    const int nu = mine < a.batch ? dense_units_of(dense_span(a.ctx_lens[mine], a.ctx_cap, a.window).pages, C) : 0;
    int incl = nu;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(incl, d);
      if (lane >= d) incl += up;
    }
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
  DecState<T, DK, DV> st[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) dec_reset(st[j]);
  const float c = a.scale * kLog2e;

  // chunk i of this wavefront covers keys 64 p0 + 32 (w + 4 i) ..; 64 page ids at a time sit in the lanes
  int ids_at = p0, ids = 0;
  if (paged && p0 + lane < p1) ids = table[p0 + lane];
  ChunkFrags<T, DK, DV> f[kDenseAhead<T, DK, DV, NT> ? 2 : 1];
  auto issue = [&](ChunkFrags<T, DK, DV>& fr, int cb) {
    const int p = cb >> 6;
    const T *kp, *vp;
    if (paged) {
      if (p - ids_at >= 64) {
        ids_at = p;
        ids = p + lane < p1 ? table[p + lane] : 0;
      }
      // an id outside the pool would fault: read page 0 instead (the caller's table is wrong)
      int id = __builtin_amdgcn_readlane(ids, p - ids_at);
      id = (unsigned)id < (unsigned)a.num_pages ? id : 0;
      kp = kbase + ((long)id * 64 + (cb & 63)) * krow;
      vp = vbase + ((long)id * a.hkv + h) * DV * 64 + (cb & 63);
    } else {
      kp = kbase + ((long)b * a.ctx_cap + cb) * krow;
      vp = vbase + ((long)b * a.hkv + h) * DV * vrow + cb;
    }
    const T* k0p = kp + chunk_key_of_row(0, n16) * krow;
    const T* k1p = kp + chunk_key_of_row(1, n16) * krow;
#pragma unroll
    for (int kk = 0; kk < DK / 32; ++kk) { fr.k0[kk] = load8(k0p + 32 * kk); fr.k1[kk] = load8(k1p + 32 * kk); }
    vp += (long)n16 * vrow + 8 * g;
#pragma unroll
    for (int t = 0; t < DV / 16; ++t) fr.v[t] = load8(vp + 16 * t * vrow);
  };
  const int end = min(p1 * 64, sp.n);
  int cb = p0 * 64 + 32 * w;
  if constexpr (kDenseAhead<T, DK, DV, NT>) {
    if (cb < end) issue(f[0], cb);
    while (cb < end) {
      const int c1 = cb + 32 * kDenseWaves, c2 = c1 + 32 * kDenseWaves;
      if (c1 < end) issue(f[1], c1);
      dense_attend<T, DK, DV, NT>(st, f[0], q, cb, sp.lo, sp.n, c, g);
      if (c2 < end) issue(f[0], c2);
      if (c1 < end) dense_attend<T, DK, DV, NT>(st, f[1], q, c1, sp.lo, sp.n, c, g);
      cb = c2;
    }
  } else {
    for (; cb < end; cb += 32 * kDenseWaves) {
      issue(f[0], cb);
      dense_attend<T, DK, DV, NT>(st, f[0], q, cb, sp.lo, sp.n, c, g);
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
    for (int x = 0; x < kDenseWaves; ++x) M = fmaxf(M, ml[x][n16][0]);
    const float own = M == kNegInf ? 0.f : fast_exp2(st[j].m - M);
#pragma unroll
    for (int t = 0; t < DV / 16; ++t) {
      f32x4_t o = st[j].o[t];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= own;
      *reinterpret_cast<f32x4_t*>(&plane[w][n16][16 * t + 4 * g]) = o;
    }
    __syncthreads();
    for (int item = threadIdx.x; item < 16 * (DV / 4); item += kDenseWaves * 64) {
      const int r = item / (DV / 4), d = 4 * (item % (DV / 4));
      if (16 * j + r >= rows) break;
      float Mr = kNegInf, L = 0.f;
#pragma unroll
      for (int x = 0; x < kDenseWaves; ++x) Mr = fmaxf(Mr, ml[x][r][0]);
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < kDenseWaves; ++x) {
        if (Mr != kNegInf) L += ml[x][r][1] * fast_exp2(ml[x][r][0] - Mr);
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
        const float inv = L > 0.f ? 1.0f / L : 0.f;
        const long row = (long)b * a.hq + h * G + row0 + 16 * j + r;
        T* dst = reinterpret_cast<T*>(a.out) + row * DV + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[i] = (T)(o[i] * inv);
        if (a.lse != nullptr && d == 0) a.lse[row] = L > 0.f ? (Mr + __log2f(L)) * (1.0f / kLog2e) : kNegInf;
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
  __shared__ float red[kGroups];
  const int b = blockIdx.x / a.hq, head = blockIdx.x % a.hq;
  const int lane = threadIdx.x & 63;
  const int C = dense_unit_pages(a);
  int u0 = 0;
  for (int x = lane; x < b; x += 64) u0 += dense_units_of(dense_span(a.ctx_lens[x], a.ctx_cap, a.window).pages, C);
  u0 = wave_sum(u0);
  const int count = dense_units_of(dense_span(a.ctx_lens[b], a.ctx_cap, a.window).pages, C);
  if (count <= 1) return;
  const int G = a.hq / a.hkv, h = head / G, r = head % G;
  const int per = a.hkv * blocks, hb = h * blocks + r / rows_per_slot;
  const long step = (long)per * rows_per_slot;
  const long first = ((long)u0 * per + hb) * rows_per_slot + r % rows_per_slot;
  float M = kNegInf;
  for (int u = lane; u < count; u += 64) M = fmaxf(M, a.part_ml[(first + u * step) * 2]);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
  const int x = threadIdx.x % kLanes, y = threadIdx.x / kLanes;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float L = 0.f;
  for (int u = y; u < count; u += kGroups) {
    const long at = first + u * step;
    const float wgt = M == kNegInf ? 0.f : fast_exp2(a.part_ml[at * 2] - M);
    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(a.part + at * DV + 4 * x);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fmaf(v[i], wgt, o[i]);
    L = fmaf(a.part_ml[at * 2 + 1], wgt, L);
  }
  *reinterpret_cast<f32x4_t*>(&acc[y][4 * x]) = o;
  if (x == 0) red[y] = L;
  __syncthreads();
  if (threadIdx.x >= DV) return;
  float sum = 0.f, l = 0.f;
#pragma unroll
  for (int k = 0; k < kGroups; ++k) { sum += acc[k][threadIdx.x]; l += red[k]; }
  const long row = (long)b * a.hq + head;
  reinterpret_cast<T*>(a.out)[row * DV + threadIdx.x] = (T)(l > 0.f ? sum / l : 0.f);
  if (a.lse != nullptr && threadIdx.x == 0) a.lse[row] = l > 0.f ? (M + __log2f(l)) * (1.0f / kLog2e) : kNegInf;
}

// 16-head tiles that share one pass over the keys: the whole group up to 64 heads (32 in fp32, whose fragments take
// twice the registers); larger groups read the keys once per block.
static int dense_tiles(const DenseDecodeArgs& a) {
  const int G = a.hq / a.hkv;
  if (G <= 16) return 1;
  return G <= 32 || a.dtype == 1 ? 2 : 4;
}

DensePlan dense_decode_plan(const DenseDecodeArgs& a) {
  DensePlan p;
  const int G = a.hq / a.hkv;
  p.tiles = dense_tiles(a);
  p.blocks = (G + 16 * p.tiles - 1) / (16 * p.tiles);
  const long per = (long)a.hkv * p.blocks;
  const int cap_pages = (a.ctx_cap + 63) / 64;
  const int span = a.window > 0 ? (int)min((long)cap_pages, ((long)a.window + 62) / 64 + 1) : cap_pages;
  constexpr long kWorkgroups = 1024;
  p.units = (int)max(1L, min(kWorkgroups / per, (long)a.batch * span));
  p.split = span > kDenseMinPages;         // otherwise every sequence is one unit
  p.slots = ((long)p.units + a.batch) * per;
  p.rows = 16 * p.tiles;
  return p;
}

long dense_decode_workspace_bytes(const DenseDecodeArgs& a) {
  const DensePlan p = dense_decode_plan(a);
  return p.split ? p.slots * p.rows * (long)(a.dv + 2) * (long)sizeof(float) : 0;
}

template <typename T, int DK, int DV, int NT>
static int launch_dense_n(const DenseDecodeArgs& a, const DensePlan& p, hipStream_t st) {
  const long units = p.split ? (long)p.units + a.batch : a.batch;
  const long wgs = units * a.hkv * p.blocks;
  if (wgs > 0x7fffffffL || (long)a.batch * a.hq > 0x7fffffffL) return -5;
  hipLaunchKernelGGL((dense_decode_kernel<T, DK, DV, NT>), dim3((unsigned)wgs), dim3(kDenseWaves * 64), 0, st, a);
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
  a.part = reinterpret_cast<float*>(workspace);
  a.part_ml = p.split ? a.part + p.slots * p.rows * a.dv : nullptr;
  if (a.dtype == 0) return launch_dense<bf16_t>(a, p, st);
  if (a.dtype == 2) return launch_dense<f16_t>(a, p, st);
  return launch_dense<float>(a, p, st);
}

}  // namespace nsa
