// The split / rotary step of qkv_rope.hip with positions on up to four axes (time, height and width of a picture's or
// film's tokens): channel pair i of a rotary head turns by pos[axis(i)][t] * inv_freq[i].
//   q_out[t][h] = R(t) q[t][h],  R = rotations by the angles, on channels [rope_off, rope_off + rope_dim); k likewise
//   pack: the reverse gather with the inverse rotation, which is the transpose, i.e. the gradient
// The angle of a far position is thousands of turns, so it is formed in 64 bits, in turns, and only what is left after
// the whole turns is rounded to 32 (a product in fp32 is 2e-3 rad off at position 32768).
//
// Bound by HBM: every element is read once and written once.  A piece is 8 channels of a row.  A thread keeps one piece
// column and walks over U rows, so where a piece lies, whether it rotates and by which pairs is worked out once, and its
// U loads travel together; a workgroup takes up to 256 neighbouring columns (short rows: several rows side by side).  The
// sines of the workgroup's rows are computed once, into LDS, while the loads travel.
#include "common.h"
#include "kernels.h"

namespace nsa {

// U: 32 bytes per thread in flight.  32768 rows of 64 / 4 heads, 192 / 128 bf16: U = 1 470 us, 2 327 (5.5 TB/s), 3 348,
// 4 337; 5003 rows of 12 / 4 heads of 128, all rotary, fp32: U = 1 20.8 us, 2 24.1.  Neighbouring workgroups take
// neighbouring columns of the same rows: 327 us against 386 with neighbouring rows.
template <typename T> constexpr int kRopeRows = sizeof(T) == 2 ? 2 : 1;

// P: type of the positions.  A choice between the two inside the kernel cost 5 % (32768 rows: 328 -> 344 us).
template <typename T, typename P, bool PACK, int U>
__global__ void __launch_bounds__(256)
rope_axes_kernel(const RopeAxesArgs a) {
  extern __shared__ float2 turn[];                       // [row of the workgroup][pair]: cosine, sine
  const QkvRopeArgs& r = a.base;
  const int pq = r.hq * r.dk / 8, pk = r.hkv * r.dk / 8, pv = r.hkv * r.dv / 8;
  const int ng = r.gates != nullptr ? 3 * r.hq : 0;
  const int half = r.rope_dim / 2;
  const unsigned slices = (unsigned)(a.pieces + a.cols - 1) / (unsigned)a.cols;
  const unsigned block = blockIdx.x / slices, col0 = (blockIdx.x - block * slices) * a.cols;
  const int side = threadIdx.x / a.cols;                 // row beside row 0 of a pass
  const int p = (int)col0 + (int)(threadIdx.x - side * a.cols);
  const long t0 = (long)block * (U * a.side) + side;
  const bool live = side < a.side && p < a.pieces;

  // 0 nothing, 1 copy, 2 rotate, 3 gate logits and padding
  int kind = 0, chan = 0;
  const T* src = nullptr;
  T* dst = nullptr;
  long sstep = 0, dstep = 0;                             // elements from one row to the next
  const int pg = a.vector_gates ? ng / 8 : 0;            // gate columns that are pieces like the others
  if (live && p < pq + pk + pv + pg) {
    T* split;
    int c, dim, poff;
    long row;
    bool rot = true;
    if (p < pq) { split = reinterpret_cast<T*>(r.q); row = (long)r.hq * r.dk; c = 8 * p; dim = r.dk; poff = r.q_off; }
    else if (p < pq + pk) { split = reinterpret_cast<T*>(r.k); row = (long)r.hkv * r.dk; c = 8 * (p - pq); dim = r.dk; poff = r.k_off; }
    else if (p < pq + pk + pv) { split = reinterpret_cast<T*>(r.v); row = (long)r.hkv * r.dv; c = 8 * (p - pq - pk); dim = r.dv; poff = r.v_off; rot = false; }
    else { split = reinterpret_cast<T*>(r.gates); row = ng; c = 8 * (p - pq - pk - pv); dim = ng; poff = r.g_off; rot = false; }
    T* packed = reinterpret_cast<T*>(r.packed) + poff + c;
    split += c;
    src = PACK ? split : packed;
    dst = PACK ? packed : split;
    sstep = PACK ? row : r.ld;
    dstep = PACK ? r.ld : row;
    chan = c % dim - r.rope_off;                         // first rotary channel of this piece (multiple of 8)
    kind = rot && chan >= 0 && chan < r.rope_dim ? 2 : 1;
  } else if (live) {
    kind = 3;
    chan = 8 * (p - pq - pk - pv);
  }
  const bool lower = chan < half;
  const long partner = lower ? half : -half;             // the other channel of a pair, when they are half a range apart

  vec8_t<T> x[U], xp[U];
  if (kind == 1 || kind == 2) {
    const T* s = src + t0 * sstep;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t0 + u * a.side < r.total) {
        x[u] = load8(s);
        if (kind == 2 && !r.interleaved) xp[u] = load8(s + partner);
      }
      s += a.side * sstep;
    }
  }

  if ((int)col0 < pq + pk) {                   // columns behind q and k have nothing to rotate
    const long w0 = (long)block * (U * a.side);
    for (int i = threadIdx.x; i < U * a.side * half; i += blockDim.x) {
      const int k = i / half, pair = i - k * half;
      const long t = w0 + k;
      if (t < r.total) {
        const int axis = (a.pair_axis[pair >> 4] >> (2 * (pair & 15))) & 3;
        const double turns = (double)reinterpret_cast<const P*>(a.positions)[axis * r.total + t] * ((double)r.inv_freq[pair] * 0.15915494309189535);
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        turn[i] = make_float2(c, PACK ? -s : s);
      }
    }
    __syncthreads();
  }

  if (kind == 1 || kind == 2) {
    T* d = dst + t0 * dstep;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t0 + u * a.side >= r.total) break;
      if (kind == 1) {
        store8(d, x[u]);
      } else {
        const float2* cs = turn + (u * a.side + side) * half;
        float y[8];
        if (r.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 w = cs[chan / 2 + i];
            const float x0 = (float)x[u][2 * i], x1 = (float)x[u][2 * i + 1];
            y[2 * i] = x0 * w.x - x1 * w.y;
            y[2 * i + 1] = x1 * w.x + x0 * w.y;
          }
        } else {
          cs += lower ? chan : chan - half;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 w = cs[e];
            y[e] = (float)x[u][e] * w.x + (float)xp[u][e] * (lower ? -w.y : w.y);
          }
        }
        store8(d, pack8<T>(y));
      }
      d += a.side * dstep;
    }
  } else if (kind == 3) {
    for (int u = 0; u < U; ++u) {
      const long t = t0 + u * a.side;
      if (t >= r.total) break;
      T* prow = reinterpret_cast<T*>(r.packed) + t * r.ld;
      T* g = reinterpret_cast<T*>(r.gates) + t * ng;
      const T* from = PACK ? g : prow + r.g_off;
      T* to = PACK ? prow + r.g_off : g;
      T y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (chan + e < ng) y[e] = from[chan + e];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (chan + e < ng) to[chan + e] = y[e];
        else if (PACK && a.pad_off + (chan + e - ng) < r.ld) prow[a.pad_off + (chan + e - ng)] = (T)0.0f;
      }
    }
  }
}

template <typename T, typename P, bool PACK, int U>
static int rope_axes_u(const RopeAxesArgs& a, hipStream_t st) {
  const long blocks = (a.base.total + U * a.side - 1) / (U * a.side);
  const long slices = (a.pieces + a.cols - 1) / a.cols;
  if (blocks * slices > 0x7fffffffL) return -2;
  const unsigned threads = (unsigned)(a.cols * a.side + 63) / 64 * 64;
  const size_t smem = (size_t)U * a.side * (a.base.rope_dim / 2) * sizeof(float2);
  hipLaunchKernelGGL((rope_axes_kernel<T, P, PACK, U>), dim3((unsigned)(blocks * slices)), dim3(threads), smem, st, a);
  return 0;
}

template <typename T, typename P>
static int rope_axes_t(const RopeAxesArgs& a, hipStream_t st) {
  // few rows: one per thread, over twice the workgroups (1000 rows of 4 / 1 heads of 64: 4.8 against 6.2 us)
  constexpr int U = kRopeRows<T>;
  const bool large = a.base.total * (long)a.pieces >= 1L << 18;
  if (a.base.pack) return large ? rope_axes_u<T, P, true, U>(a, st) : rope_axes_u<T, P, true, 1>(a, st);
  return large ? rope_axes_u<T, P, false, U>(a, st) : rope_axes_u<T, P, false, 1>(a, st);
}

template <typename P>
static int rope_axes_p(const RopeAxesArgs& a, hipStream_t st) {
  if (a.base.dtype == 2) return rope_axes_t<f16_t, P>(a, st);
  return a.base.dtype == 0 ? rope_axes_t<bf16_t, P>(a, st) : rope_axes_t<float, P>(a, st);
}

int launch_rope_axes(RopeAxesArgs a, hipStream_t st) {
  const QkvRopeArgs& r = a.base;
  const long ng = r.gates != nullptr ? 3L * r.hq : 0;
  const long pad = r.pack ? r.ld - a.pad_off : 0;
  const long pieces = ((long)r.hq * r.dk + (long)r.hkv * (r.dk + r.dv)) / 8 + (ng + pad + 7) / 8;
  if (pieces > 0x7fffffffL / 8 || r.total > 0x7fffffffL) return -2;
  a.pieces = (int)pieces;
  a.vector_gates = ng > 0 && ng % 8 == 0 && r.g_off % 8 == 0 && (reinterpret_cast<uintptr_t>(r.gates) & 15) == 0;
  const int slices = (int)((pieces + 255) / 256);
  a.cols = (int)((pieces + slices - 1) / slices);
  a.side = 256 / a.cols;
  // short rows whose heads have many pairs keep to fewer rows: at most 32 KB of sines
  while (a.side > 1 && 2 * a.side * (r.rope_dim / 2) * sizeof(float2) > 32768) --a.side;
  return a.wide ? rope_axes_p<int64_t>(a, st) : rope_axes_p<int32_t>(a, st);
}

}  // namespace nsa
