// The split / rotary step of qkv_rope.hip with positions on up to four axes (time, height and width of a picture's or
// film's tokens): channel pair i of a rotary head turns by pos[axis(i)][t] * inv_freq[i].
//   q_out[t][h] = R(t) q[t][h],  R = rotations by the angles, on channels [rope_off, rope_off + rope_dim); k likewise
//   pack: the reverse gather with the inverse rotation, which is the transpose, i.e. the gradient
// The angle of a far position is thousands of turns, so it is formed in 64 bits, in turns, and only what is left after
// the whole turns is rounded to 32 (a product in fp32 is 2e-3 rad off at position 32768).
//
// Bound by HBM: every element is read once and written once.  An item is 8 channels of one token; a workgroup takes
// 256 U consecutive items, across the ends of tokens, so that short rows fill it as well as long ones, with the loads of
// all U in flight before the first rotation.  The sines of the tokens it touches are computed once, into LDS, while they
// travel.
#include "common.h"
#include "kernels.h"

namespace nsa {

constexpr int kRopeItems = 8;      // U of a large call

template <typename T, bool PACK, int U>
__global__ void __launch_bounds__(256)
rope_axes_kernel(const RopeAxesArgs a) {
  extern __shared__ float2 turn[];                       // [token of the workgroup][pair]: cosine, sine
  const QkvRopeArgs& r = a.base;
  const int pq = r.hq * r.dk / 8, pk = r.hkv * r.dk / 8, pv = r.hkv * r.dv / 8;
  const int ng = r.gates != nullptr ? 3 * r.hq : 0;
  const unsigned ppt = a.pieces;
  const long first = (long)blockIdx.x * (256 * U);
  const long t0 = a.small ? (long)((unsigned)first / ppt) : first / (long)ppt;
  const unsigned r0 = (unsigned)(first - t0 * ppt);
  const int half = r.rope_dim / 2;

  // where item u of this thread reads and writes: 0 nothing, 1 copy, 2 rotate, 3 gate logits
  int kind[U], chan[U], tok[U];
  const T* src[U];
  T* dst[U];
  vec8_t<T> x[U], xp[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned at = r0 + 256 * u + threadIdx.x;
    tok[u] = (int)__umulhi(at, a.magic);                 // at / ppt, exact: at * ppt < 2^32
    const int p = (int)(at - tok[u] * ppt);
    const long t = t0 + tok[u];
    kind[u] = 0; chan[u] = 0;
    src[u] = nullptr; dst[u] = nullptr;
    x[u] = zero8<T>(); xp[u] = zero8<T>();
    if (t >= r.total) continue;
    T* prow = reinterpret_cast<T*>(r.packed) + t * r.ld;
    if (p < pq + pk + pv) {
      T* split;
      int c, dim, poff;
      bool rot = true;
      if (p < pq) { split = reinterpret_cast<T*>(r.q) + t * r.hq * r.dk; c = 8 * p; dim = r.dk; poff = r.q_off; }
      else if (p < pq + pk) { split = reinterpret_cast<T*>(r.k) + t * r.hkv * r.dk; c = 8 * (p - pq); dim = r.dk; poff = r.k_off; }
      else { split = reinterpret_cast<T*>(r.v) + t * r.hkv * r.dv; c = 8 * (p - pq - pk); dim = r.dv; poff = r.v_off; rot = false; }
      src[u] = PACK ? split + c : prow + poff + c;
      dst[u] = PACK ? prow + poff + c : split + c;
      x[u] = load8(src[u]);
      chan[u] = c % dim - r.rope_off;                    // first rotary channel of this piece (multiple of 8)
      kind[u] = rot && chan[u] >= 0 && chan[u] < r.rope_dim ? 2 : 1;
      if (kind[u] == 2 && !r.interleaved) xp[u] = load8(src[u] + (chan[u] < half ? half : -half));
    } else {
      kind[u] = 3;
      chan[u] = 8 * (p - pq - pk - pv);
    }
  }

  const int tokens = (int)__umulhi(r0 + 256 * U - 1, a.magic) + 1;
  for (int i = threadIdx.x; i < tokens * half; i += 256) {
    const int k = i / half, pair = i - k * half;
    const long t = t0 + k;
    if (t < r.total) {
      const int axis = (a.pair_axis[pair >> 4] >> (2 * (pair & 15))) & 3;
      const double turns = (double)r.positions[axis * r.total + t] * ((double)r.inv_freq[pair] * 0.15915494309189535);
      float s, c;
      sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
      turn[i] = make_float2(c, PACK ? -s : s);
    }
  }
  __syncthreads();

#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (kind[u] == 0) continue;
    if (kind[u] == 1) {
      store8(dst[u], x[u]);
    } else if (kind[u] == 2) {
      const float2* cs = turn + tok[u] * half;
      float y[8];
      if (r.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 w = cs[chan[u] / 2 + i];
          const float x0 = (float)x[u][2 * i], x1 = (float)x[u][2 * i + 1];
          y[2 * i] = x0 * w.x - x1 * w.y;
          y[2 * i + 1] = x1 * w.x + x0 * w.y;
        }
      } else {
        const bool lower = chan[u] < half;
        const int f0 = lower ? chan[u] : chan[u] - half;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 w = cs[f0 + e];
          y[e] = (float)x[u][e] * w.x + (float)xp[u][e] * (lower ? -w.y : w.y);
        }
      }
      store8(dst[u], pack8<T>(y));
    } else {                                             // gate logits, then the padding of a packed row
      const long t = t0 + tok[u];
      T* prow = reinterpret_cast<T*>(r.packed) + t * r.ld;
      T* g = reinterpret_cast<T*>(r.gates) + t * ng;
      for (int e = chan[u]; e < chan[u] + 8; ++e) {
        if (e < ng) {
          if (PACK) prow[r.g_off + e] = g[e];
          else g[e] = prow[r.g_off + e];
        } else if (PACK && a.pad_off + (e - ng) < r.ld) {
          prow[a.pad_off + (e - ng)] = (T)0.0f;
        }
      }
    }
  }
}

template <typename T, bool PACK, int U>
static int rope_axes_u(const RopeAxesArgs& a, hipStream_t st) {
  const long items = a.base.total * a.pieces;
  const long blocks = (items + 256 * U - 1) / (256 * U);
  if (blocks > 0x7fffffffL) return -2;
  const size_t tokens = (256 * U - 1 + a.pieces - 1) / a.pieces + 1;
  const size_t smem = tokens * (a.base.rope_dim / 2) * sizeof(float2);
  hipLaunchKernelGGL((rope_axes_kernel<T, PACK, U>), dim3((unsigned)blocks), dim3(256), smem, st, a);
  return 0;
}

template <typename T>
static int rope_axes_t(const RopeAxesArgs& a, hipStream_t st) {
  // few rows: one item per thread, over as many workgroups as there are
  const bool large = a.base.total * (long)a.pieces >= 256L * 8 * 256;
  if (a.base.pack) return large ? rope_axes_u<T, true, kRopeItems>(a, st) : rope_axes_u<T, true, 1>(a, st);
  return large ? rope_axes_u<T, false, kRopeItems>(a, st) : rope_axes_u<T, false, 1>(a, st);
}

int launch_rope_axes(RopeAxesArgs a, hipStream_t st) {
  const QkvRopeArgs& r = a.base;
  const long ng = r.gates != nullptr ? 3L * r.hq : 0;
  const long pad = r.pack ? r.ld - a.pad_off : 0;
  const long pieces = ((long)r.hq * r.dk + (long)r.hkv * (r.dk + r.dv)) / 8 + (ng + pad + 7) / 8;
  if (pieces > 60000 || r.total > 0x7fffffffL) return -2;
  a.pieces = (unsigned)pieces;
  a.magic = (unsigned)((0x100000000ULL + pieces - 1) / pieces);
  a.small = r.total * pieces + 256 * kRopeItems < 0xffffffffL;
  if (r.dtype == 2) return rope_axes_t<f16_t>(a, st);
  return r.dtype == 0 ? rope_axes_t<bf16_t>(a, st) : rope_axes_t<float>(a, st);
}

}  // namespace nsa
