// Gated linear recurrence along a sequence, forward and backward (the mixer of the gated-linear-recurrence encoder
// layer, crnn_hip/glr.py; crnn_hip.gated_scan).
//
//   h_t = a_t h_{t-1} + r_t v_t,   a = sigmoid(f), r = 1 - a = sigmoid(-f),   y_t = h_t
//   G_t = dy_t + a_{t+1} G_{t+1};  df = G (h_{t-1} - v) a r,  dv = G r,  dh0 = a_first G_first
//
// A step is an affine map of the state, and affine maps compose: steps s .. e act as h -> A h + H with A = prod a. So a
// stretch of the sequence can be summed up before the state that enters it is known. A wave owns 64 * VEC channels and
// L consecutive steps in registers; the W waves of a workgroup take consecutive pieces of a tile of W * L steps,
// exchange their (A, H) through LDS, and each then runs its L steps from the state that really enters them: the sequence
// is walked W * L steps at a time and every element is read once. Where batch * channels alone does not fill the chip,
// the sequence is also cut into S segments: a first kernel sums up each segment (one more read of f and v), and a
// segment's workgroup composes the summaries of the segments before it.
// The backward walks the tiles from the end with the same pieces: the reverse recurrence C_t = a_t (dy_t + C_{t+1}) has
// the same A. h_{t-1} is not stored but recomputed in fp32 from the state at the tile's start (ckpt), so y's rounding
// to bf16 never enters the gradients and nothing as large as y is read.
// Both passes are bound by memory: forward f, v in, y out; backward f, v, dy in, df, dv out.
#include "common.hpp"
#include "crnn_internal.hpp"

namespace {

constexpr int L = 4;      // steps a wave holds
constexpr int kWmax = 8;  // waves of the widest tile
// channels of a lane: 4 bytes, 256 a wave and step (wider lanes leave fewer waves: 37 x 301 x 333 fp32, forward / backward 20.6 /
// 24.7 us at one channel, 21.8 / 26.2 at two; 2 x 16384 x 1024 bf16 57 / 89 at two, 76 / 109 at four)
template <typename T> constexpr int vec_of() { return sizeof(T) == 2 ? 2 : 1; }

// VEC consecutive channels at an element-aligned address
template <typename T, int VEC> struct Raw;
template <int VEC> struct Raw<bf16, VEC> { typedef unsigned short t __attribute__((ext_vector_type(VEC))); };
template <int VEC> struct Raw<float, VEC> { typedef float t __attribute__((ext_vector_type(VEC))); };
template <typename T, int VEC> struct RawU {   // the same, element-aligned
  typedef typename Raw<T, VEC>::t t __attribute__((aligned(sizeof(T))));
};

template <typename T, int VEC> __device__ __forceinline__ float elem(const typename Raw<T, VEC>::t& r, int i) {
  if constexpr (sizeof(T) == 2) return __uint_as_float((unsigned)r[i] << 16);
  else return r[i];
}
template <typename T, int VEC> __device__ __forceinline__ void set_elem(typename Raw<T, VEC>::t& r, int i, float v) {
  if constexpr (sizeof(T) == 2) r[i] = __builtin_bit_cast(unsigned short, (bf16)v);
  else r[i] = v;
}
// nv: this lane's channels that exist (0 .. VEC); FULL: all of them in every lane of the wave, which spares each access its
// branch, as whole pieces within the length do (2 x 16384 x 1024 bf16, forward / backward with all of them: 70 / 99 us,
// without 57 / 89; 256 x 32 x 1024 both ways: 13.2 / 19.9, 10.7 / 17.4)
template <typename T, int VEC, bool FULL> __device__ __forceinline__ typename Raw<T, VEC>::t ldv(const T* p, int nv) {
  typename Raw<T, VEC>::t r = {};
  if (FULL || nv == VEC) {
    r = *reinterpret_cast<const typename RawU<T, VEC>::t*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < VEC - 1; ++i)
      if (i < nv) set_elem<T, VEC>(r, i, tof(p[i]));
  }
  return r;
}
template <typename T, int VEC, bool FULL> __device__ __forceinline__ void stv(T* p, int nv, const float* v) {
  if (FULL || nv == VEC) {
    typename Raw<T, VEC>::t r = {};
#pragma unroll
    for (int i = 0; i < VEC; ++i) set_elem<T, VEC>(r, i, v[i]);
    *reinterpret_cast<typename RawU<T, VEC>::t*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < VEC - 1; ++i)
      if (i < nv) p[i] = fromf<T>(v[i]);
  }
}

// a = sigmoid(f), r = sigmoid(-f) without cancellation: e = exp(-|f|), the larger is 1 / (1 + e), the smaller e times it.
// bf16: hardware exp and reciprocal (about 1e-7 relative, far under the inputs' 2^-9); fp32: expf (1 ulp) and the IEEE division.
template <typename T> __device__ __forceinline__ void gate(float f, float& a, float& r) {
  float p, q;
  if constexpr (sizeof(T) == 2) {
    const float e = __expf(-fabsf(f));
    p = __builtin_amdgcn_rcpf(1.f + e);
    q = e * p;
  } else {
    const float e = expf(-fabsf(f));
    p = 1.f / (1.f + e);
    q = e * p;
  }
  const bool neg = f < 0.f;
  a = neg ? q : p;
  r = neg ? p : q;
}

struct ScanArgs {
  const void *f, *v, *dy;
  void *y, *df, *dv;
  long fsb, fst, vsb, vst, dsb, dst, ysb, yst, gsb, gst, wsb, wst;
  const float *h0, *dhT;
  float *hT, *dh0, *ckpt;
  float* sum;            // segment summaries [S][B][D][2]
  const int* lengths;
  int B, T, D, Dh, dir;  // Dh: channels of one direction
  int groups, S, tps;    // channel groups of one direction, segments, tiles per segment
};

// who a workgroup is: channels, direction, sample, segment
struct Who {
  int ch, nv, b, seg, len;
  bool rev;
};
template <int VEC> __device__ __forceinline__ Who who(const ScanArgs& a) {
  const int nd = a.dir == 2 ? 2 : 1, lane = threadIdx.x & 63;
  unsigned i = blockIdx.x;
  Who w;
  const int g = i % a.groups;
  i /= a.groups;
  const int d = i % nd;
  i /= nd;
  w.b = i % a.B;
  w.seg = i / a.B;
  w.rev = a.dir == 1 || d == 1;
  const int c = (g * 64 + lane) * VEC;
  w.nv = min(max(a.Dh - c, 0), VEC);
  w.ch = d * a.Dh + c;
  w.len = a.lengths ? min(max(a.lengths[w.b], 0), a.T) : a.T;
  return w;
}
// position in time of walking step u
__device__ __forceinline__ int at(const Who& w, int u) { return w.rev && u < w.len ? w.len - 1 - u : u; }

// The state (or, going back, the gradient) that enters a segment: `first` through the n summaries s0, s0 + ds, .. before it.
// The waves of the workgroup compose a share each, eight loads in flight, and join in LDS (ex): with one wave doing all of
// them this was 4 memory latencies of every workgroup of 2 x 16384 x 1024 in 32 segments.
template <int VEC, int W>
__device__ __forceinline__ void entering(const ScanArgs& a, const Who& w, const float* first, int s0, int ds, int n,
                                         float (*ex)[VEC][64], float* h) {
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int i = 0; i < VEC; ++i) h[i] = first && i < w.nv ? first[(size_t)w.b * a.D + w.ch + i] : 0.f;
  if (n == 0) return;
  const int per = (n + W - 1) / W, beg = min(n, wid * per), end = min(n, beg + per);
  const long step = (long)ds * a.B * a.D * 2;
  const float* p = a.sum + (((size_t)s0 * a.B + w.b) * a.D + w.ch) * 2 + beg * step;
  float A[VEC], H[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    A[i] = 1.f;
    H[i] = 0.f;
  }
  for (int k = beg; k < end; k += 8) {
    float m[8][2 * VEC];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 2 * VEC; ++i) m[j][i] = k + j < end && i < 2 * w.nv ? p[j * step + i] : (i & 1 ? 0.f : 1.f);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        A[i] *= m[j][2 * i];
        H[i] = m[j][2 * i] * H[i] + m[j][2 * i + 1];
      }
    p += 8 * step;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    ex[2 * wid][i][lane] = A[i];
    ex[2 * wid + 1][i][lane] = H[i];
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < W; ++q)
#pragma unroll
    for (int i = 0; i < VEC; ++i) h[i] = ex[2 * q][i][lane] * h[i] + ex[2 * q + 1][i][lane];
  __syncthreads();   // ex is the tiles' next
}

template <typename T, int VEC> using RawT = typename Raw<T, VEC>::t;

// the L steps from walking step u0 of one tensor (nothing is read at or behind the length)
template <typename T, int VEC, bool FULL>
__device__ __forceinline__ void load_piece(const Who& w, const T* p, long sb, long st, int u0, RawT<T, VEC>* r) {
  const T* base = p + w.b * sb + w.ch;
  if (u0 + L <= w.len) {
    const long step = w.rev ? -st : st;
    base += at(w, u0) * st;
#pragma unroll
    for (int i = 0; i < L; ++i) r[i] = ldv<T, VEC, FULL>(base + i * step, w.nv);
  } else {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      RawT<T, VEC> z = {};
      r[i] = z;
      if (u0 + i < w.len) r[i] = ldv<T, VEC, FULL>(base + at(w, u0 + i) * st, w.nv);
    }
  }
}
// the same steps' results; zero at and behind the length, nothing at or behind T
template <typename T, int VEC, bool FULL>
__device__ __forceinline__ void store_piece(const Who& w, int T_, T* p, long sb, long st, int u0, const float (*v)[VEC]) {
  T* base = p + w.b * sb + w.ch;
  if (u0 + L <= w.len) {
    const long step = w.rev ? -st : st;
    base += at(w, u0) * st;
#pragma unroll
    for (int i = 0; i < L; ++i) stv<T, VEC, FULL>(base + i * step, w.nv, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if (u0 + i >= T_) break;
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = u0 + i < w.len ? v[i][e] : 0.f;
      stv<T, VEC, FULL>(base + at(w, u0 + i) * st, w.nv, o);
    }
  }
}
// every lane of the wave has all its channels
template <int VEC> __device__ __forceinline__ bool full_wave(const ScanArgs& a) {
  return (int)(blockIdx.x % a.groups + 1) * 64 * VEC <= a.Dh;
}

template <typename T, int VEC, int W, bool FULL> __device__ __forceinline__ void scan_fwd(const ScanArgs& a, float (*ex)[W][2][VEC][64]) {
  constexpr int TL = W * L;
  const Who w = who<VEC>(a);
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (a.T + TL - 1) / TL, t0 = w.seg * a.tps, t1 = min(tiles, t0 + a.tps);
  const T *f = (const T*)a.f, *v = (const T*)a.v;
  float h[VEC];
  entering<VEC, W>(a, w, a.h0, 0, 1, w.seg, &ex[0][0][0], h);
  RawT<T, VEC> fr[L], vr[L];
  load_piece<T, VEC, FULL>(w, f, a.fsb, a.fst, t0 * TL + wid * L, fr);
  load_piece<T, VEC, FULL>(w, v, a.vsb, a.vst, t0 * TL + wid * L, vr);
  for (int t = t0; t < t1; ++t) {
    const int u0 = t * TL + wid * L;
    float al[L][VEC], ul[L][VEC], A[VEC], H[VEC];
#pragma unroll
    for (int s = 0; s < L; ++s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float r;
        gate<T>(elem<T, VEC>(fr[s], i), al[s][i], r);
        ul[s][i] = r * elem<T, VEC>(vr[s], i);
      }
    if (u0 + L > w.len) {
#pragma unroll
      for (int s = 0; s < L; ++s)
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (u0 + s >= w.len) {
            al[s][i] = 1.f;
            ul[s][i] = 0.f;
          }
    }
    if (t + 1 < t1) {   // the next tile's piece while this one is finished
      load_piece<T, VEC, FULL>(w, f, a.fsb, a.fst, u0 + TL, fr);
      load_piece<T, VEC, FULL>(w, v, a.vsb, a.vst, u0 + TL, vr);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      A[i] = al[0][i];
      H[i] = ul[0][i];
    }
#pragma unroll
    for (int s = 1; s < L; ++s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        A[i] *= al[s][i];
        H[i] = al[s][i] * H[i] + ul[s][i];
      }
    if (a.ckpt && wid == 0) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (FULL || i < w.nv) a.ckpt[((size_t)w.b * tiles + t) * a.D + w.ch + i] = h[i];
    }
    float hin[VEC];
    if constexpr (W > 1) {
      const int p = t & 1;   // two LDS sets in turn: one barrier per tile
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        ex[p][wid][0][i][lane] = A[i];
        ex[p][wid][1][i][lane] = H[i];
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < W; ++q) {
        if (q == wid)
#pragma unroll
          for (int i = 0; i < VEC; ++i) hin[i] = h[i];
#pragma unroll
        for (int i = 0; i < VEC; ++i) h[i] = ex[p][q][0][i][lane] * h[i] + ex[p][q][1][i][lane];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        hin[i] = h[i];
        h[i] = A[i] * h[i] + H[i];
      }
    }
#pragma unroll
    for (int s = 0; s < L; ++s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) ul[s][i] = hin[i] = al[s][i] * hin[i] + ul[s][i];
    store_piece<T, VEC, FULL>(w, a.T, (T*)a.y, a.ysb, a.yst, u0, ul);
  }
  if (a.hT && w.seg == a.S - 1 && wid == 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < w.nv) a.hT[(size_t)w.b * a.D + w.ch + i] = h[i];
  }
}
template <typename T, int VEC, int W> __global__ __launch_bounds__(64 * W) void scan_fwd_kernel(ScanArgs a) {
  __shared__ float ex[2][W][2][VEC][64];
  if (full_wave<VEC>(a)) scan_fwd<T, VEC, W, true>(a, ex);
  else scan_fwd<T, VEC, W, false>(a, ex);
}

// (A, H) of a segment, or (A, C) of the reverse recurrence (BACK): each wave sums up its share of the segment, then the
// shares are joined in order
template <typename T, int VEC, int W, bool BACK, bool FULL> __device__ __forceinline__ void scan_sum(const ScanArgs& a, float (*ex)[2][VEC][64]) {
  const Who w = who<VEC>(a);
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = a.tps * L, beg = w.seg * a.tps * W * L + wid * per;   // this wave's steps [beg, beg + per)
  const T *f = (const T*)a.f, *q = BACK ? (const T*)a.dy : (const T*)a.v;
  const long qsb = BACK ? a.dsb : a.vsb, qst = BACK ? a.dst : a.vst;
  float A[VEC], H[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    A[i] = 1.f;
    H[i] = 0.f;
  }
  RawT<T, VEC> fr[L], qr[L];
  const int first = BACK ? beg + per - L : beg;
  load_piece<T, VEC, FULL>(w, f, a.fsb, a.fst, first, fr);
  load_piece<T, VEC, FULL>(w, q, qsb, qst, first, qr);
  for (int k = 0; k < a.tps; ++k) {
    const int u0 = BACK ? first - k * L : first + k * L;
    float al[L][VEC], ul[L][VEC];
#pragma unroll
    for (int s = 0; s < L; ++s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float r;
        gate<T>(elem<T, VEC>(fr[s], i), al[s][i], r);
        ul[s][i] = BACK ? elem<T, VEC>(qr[s], i) : r * elem<T, VEC>(qr[s], i);
      }
    if (u0 + L > w.len) {
#pragma unroll
      for (int s = 0; s < L; ++s)
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (u0 + s >= w.len) {
            al[s][i] = 1.f;
            ul[s][i] = 0.f;
          }
    }
    if (k + 1 < a.tps) {
      load_piece<T, VEC, FULL>(w, f, a.fsb, a.fst, BACK ? u0 - L : u0 + L, fr);
      load_piece<T, VEC, FULL>(w, q, qsb, qst, BACK ? u0 - L : u0 + L, qr);
    }
#pragma unroll
    for (int s = 0; s < L; ++s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int j = BACK ? L - 1 - s : s;
        A[i] *= al[j][i];
        H[i] = BACK ? al[j][i] * (ul[j][i] + H[i]) : al[j][i] * H[i] + ul[j][i];
      }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    ex[wid][0][i][lane] = A[i];
    ex[wid][1][i][lane] = H[i];
  }
  __syncthreads();
  if (wid == 0) {
    float sa[VEC], sh[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      sa[i] = 1.f;
      sh[i] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const int j = BACK ? W - 1 - k : k;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        sa[i] *= ex[j][0][i][lane];
        sh[i] = ex[j][0][i][lane] * sh[i] + ex[j][1][i][lane];
      }
    }
    float* p = a.sum + (((size_t)w.seg * a.B + w.b) * a.D + w.ch) * 2;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < w.nv) {
        p[2 * i] = sa[i];
        p[2 * i + 1] = sh[i];
      }
  }
}

template <typename T, int VEC, int W, bool BACK> __global__ __launch_bounds__(64 * W) void scan_sum_kernel(ScanArgs a) {
  __shared__ float ex[W][2][VEC][64];
  if (who<VEC>(a).seg == (BACK ? 0 : a.S - 1)) return;   // nobody comes after it
  if (full_wave<VEC>(a)) scan_sum<T, VEC, W, BACK, true>(a, ex);
  else scan_sum<T, VEC, W, BACK, false>(a, ex);
}

template <typename T, int VEC, int W, bool FULL> __device__ __forceinline__ void scan_bwd(const ScanArgs& a, float (*ex)[W][3][VEC][64]) {
  constexpr int TL = W * L;
  const Who w = who<VEC>(a);
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (a.T + TL - 1) / TL, t0 = w.seg * a.tps, t1 = min(tiles, t0 + a.tps);
  const T *f = (const T*)a.f, *v = (const T*)a.v, *dy = (const T*)a.dy;
  float c[VEC];
  entering<VEC, W>(a, w, a.dhT, a.S - 1, -1, a.S - 1 - w.seg, &ex[0][0][0], c);
  RawT<T, VEC> fr[L], vr[L], dr[L];
  const int ub = (t1 - 1) * TL + wid * L;
  load_piece<T, VEC, FULL>(w, f, a.fsb, a.fst, ub, fr);
  load_piece<T, VEC, FULL>(w, v, a.vsb, a.vst, ub, vr);
  load_piece<T, VEC, FULL>(w, dy, a.dsb, a.dst, ub, dr);
  for (int t = t1 - 1; t >= t0; --t) {
    const int u0 = t * TL + wid * L;
    float al[L][VEC], rl[L][VEC], vl[L][VEC], dl[L][VEC], A[VEC], H[VEC], C[VEC], hin[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      hin[i] = FULL || i < w.nv ? a.ckpt[((size_t)w.b * tiles + t) * a.D + w.ch + i] : 0.f;
      A[i] = 1.f;
      H[i] = C[i] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < L; ++s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        gate<T>(elem<T, VEC>(fr[s], i), al[s][i], rl[s][i]);
        vl[s][i] = elem<T, VEC>(vr[s], i);
        dl[s][i] = elem<T, VEC>(dr[s], i);
      }
    if (u0 + L > w.len) {
#pragma unroll
      for (int s = 0; s < L; ++s)
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (u0 + s >= w.len) {
            al[s][i] = 1.f;
            rl[s][i] = vl[s][i] = dl[s][i] = 0.f;
          }
    }
#pragma unroll
    for (int s = 0; s < L; ++s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        A[i] *= al[s][i];
        H[i] = al[s][i] * H[i] + rl[s][i] * vl[s][i];
      }
#pragma unroll
    for (int s = L - 1; s >= 0; --s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) C[i] = al[s][i] * (dl[s][i] + C[i]);
    if (t > t0) {
      load_piece<T, VEC, FULL>(w, f, a.fsb, a.fst, u0 - TL, fr);
      load_piece<T, VEC, FULL>(w, v, a.vsb, a.vst, u0 - TL, vr);
      load_piece<T, VEC, FULL>(w, dy, a.dsb, a.dst, u0 - TL, dr);
    }
    float cin[VEC];
    if constexpr (W > 1) {
      const int p = t & 1;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        ex[p][wid][0][i][lane] = A[i];
        ex[p][wid][1][i][lane] = H[i];
        ex[p][wid][2][i][lane] = C[i];
      }
      __syncthreads();
      for (int q = 0; q < wid; ++q)   // the state that enters this wave's piece
#pragma unroll
        for (int i = 0; i < VEC; ++i) hin[i] = ex[p][q][0][i][lane] * hin[i] + ex[p][q][1][i][lane];
#pragma unroll
      for (int q = W - 1; q >= 0; --q) {   // the gradient that enters it from behind, and the tile's
        if (q == wid)
#pragma unroll
          for (int i = 0; i < VEC; ++i) cin[i] = c[i];
#pragma unroll
        for (int i = 0; i < VEC; ++i) c[i] = ex[p][q][0][i][lane] * c[i] + ex[p][q][2][i][lane];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        cin[i] = c[i];
        c[i] = A[i] * c[i] + C[i];
      }
    }
    float hp[L][VEC];
#pragma unroll
    for (int s = 0; s < L; ++s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        hp[s][i] = hin[i];
        hin[i] = al[s][i] * hin[i] + rl[s][i] * vl[s][i];
      }
#pragma unroll
    for (int s = L - 1; s >= 0; --s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float g = dl[s][i] + cin[i], gv = g * rl[s][i];
        cin[i] = al[s][i] * g;
        dl[s][i] = gv * al[s][i] * (hp[s][i] - vl[s][i]);
        rl[s][i] = gv;
      }
    store_piece<T, VEC, FULL>(w, a.T, (T*)a.df, a.gsb, a.gst, u0, dl);
    store_piece<T, VEC, FULL>(w, a.T, (T*)a.dv, a.wsb, a.wst, u0, rl);
  }
  if (a.dh0 && w.seg == 0 && wid == 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < w.nv) a.dh0[(size_t)w.b * a.D + w.ch + i] = c[i];
  }
}
template <typename T, int VEC, int W> __global__ __launch_bounds__(64 * W) void scan_bwd_kernel(ScanArgs a) {
  __shared__ float ex[2][W][3][VEC][64];
  if (full_wave<VEC>(a)) scan_bwd<T, VEC, W, true>(a, ex);
  else scan_bwd<T, VEC, W, false>(a, ex);
}

// T = 0: no steps, the state passes through
__global__ __launch_bounds__(256) void scan_pass_kernel(const float* in, float* out, long n) {
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) out[i] = in ? in[i] : 0.f;
}

// The plan: 64 * VEC channels per wave, W waves (W * L steps) per tile, S segments of tps tiles.
struct Plan {
  int W, S, tps, groups, tiles;
};
Plan scan_plan(int dtype, int B, int T, int D, int dir) {
  const int Dh = dir == 2 ? D / 2 : D, nd = dir == 2 ? 2 : 1;
  Plan p;
  const int ch = 64 * (dtype == CRNN_BF16 ? vec_of<bf16>() : vec_of<float>());
  p.groups = (Dh + ch - 1) / ch;
  const long rows = (long)p.groups * nd * B;   // workgroups without segments
  const long cu = crnn_cu_count();
  const int wmax = rows < 4 * cu ? kWmax : kWmax / 2;
  p.W = 1;
  while (p.W < wmax && T > p.W * L) p.W *= 2;
  p.tiles = (T + p.W * L - 1) / (p.W * L);   // T <= kMaxT: no overflow
  p.S = 1;
  // Segments where rows leave half of the CUs idle, or some of them for long (forward / backward, us, with segments and without:
  // 96 rows of 300 steps 12.8 / 16.0, 13.4 / 20.3; 200 of 300 19.0 / 24.1, 14.7 / 22.5; 160 of 512 22 / 30, 20 / 33; 192 of 2000
  // 85 / 146, 85 / 163). Two workgroups per CU (2 x 16384 x 1024 bf16: 57 / 89; 58 / 95 at three, 61 / 97 at four).
  if (p.W == kWmax && p.tiles > 2 && (2 * rows < cu || (rows < cu && p.tiles > 24))) {
    long s = (2 * cu + rows - 1) / rows;
    if (s > p.tiles / 2) s = p.tiles / 2;
    if (s > 128) s = 128;
    p.S = (int)(s < 1 ? 1 : s);
  }
  p.tps = (p.tiles + p.S - 1) / p.S;
  if (p.tiles > 0) p.S = (p.tiles + p.tps - 1) / p.tps;
  return p;
}

template <typename T, int W, bool BACK> int scan_go(const ScanArgs& a, hipStream_t st) {
  constexpr int kVec = vec_of<T>();
  const int nd = a.dir == 2 ? 2 : 1;
  const long blocks = (long)a.groups * nd * a.B * a.S;
  if (blocks > 0xffffffffL / (64 * W)) return crnn_set_error(hipErrorInvalidValue, "gated_scan: a grid of 2^32 threads or more");
  const dim3 grid((unsigned)blocks), block(64 * W);
  if (a.S > 1) {
    if constexpr (W == kWmax) {   // only the widest tiles are cut into segments
      hipLaunchKernelGGL((scan_sum_kernel<T, kVec, W, BACK>), grid, block, 0, st, a);
      const int rc = (int)hipGetLastError();
      if (rc) return rc;
    }
  }
  if constexpr (BACK) hipLaunchKernelGGL((scan_bwd_kernel<T, kVec, W>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((scan_fwd_kernel<T, kVec, W>), grid, block, 0, st, a);
  return (int)hipGetLastError();
}
template <typename T, bool BACK> int scan_run(ScanArgs& a, hipStream_t st) {
  const Plan p = scan_plan(sizeof(T) == 2 ? CRNN_BF16 : CRNN_F32, a.B, a.T, a.D, a.dir);
  a.Dh = a.dir == 2 ? a.D / 2 : a.D;
  a.groups = p.groups;
  a.S = p.S;
  a.tps = p.tps;
  if (p.W == 1) return scan_go<T, 1, BACK>(a, st);
  if (p.W == 2) return scan_go<T, 2, BACK>(a, st);
  if (p.W == 4) return scan_go<T, 4, BACK>(a, st);
  return scan_go<T, kWmax, BACK>(a, st);
}
// Step counters are 32 bits. The passes run past T by less than a tile, the summaries by less than the last segment, tps tiles: with
// two segments or more that is at most half of T and a tile, so 2^30 + 2^29 + 64 steps.
constexpr int kMaxT = 1 << 30;
bool bad_shape(int dtype, int B, int T, int D, int dir) {
  return (dtype != CRNN_F32 && dtype != CRNN_BF16) || B < 0 || T < 0 || T > kMaxT || D < 0 || D > kMaxT || dir < 0 || dir > 2 || (dir == 2 && D % 2);
}

}  // namespace

extern "C" {

size_t crnn_gated_scan_ckpt_bytes(int dtype, int B, int T, int D, int dir) {
  if (bad_shape(dtype, B, T, D, dir) || !B || !T || !D) return 0;
  return (size_t)B * scan_plan(dtype, B, T, D, dir).tiles * D * sizeof(float);
}

size_t crnn_gated_scan_workspace(int dtype, int B, int T, int D, int dir) {
  if (bad_shape(dtype, B, T, D, dir) || !B || !T || !D) return 0;
  const Plan p = scan_plan(dtype, B, T, D, dir);
  return p.S > 1 ? (size_t)p.S * B * D * 2 * sizeof(float) : 0;
}

int crnn_gated_scan_fwd(int dtype, const void* f, long fsb, long fst, const void* v, long vsb, long vst, const float* h0,
                        const int* lengths, void* y, long ysb, long yst, float* hT, float* ckpt, float* ws, size_t ws_bytes,
                        int B, int T, int D, int dir, void* stream) {
  if (bad_shape(dtype, B, T, D, dir))
    return crnn_set_error(hipErrorInvalidValue, "gated_scan_fwd: dtype fp32 or bf16, B/T/D >= 0, T, D <= 2^30, dir 0..2 (2: even D)");
  hipStream_t st = (hipStream_t)stream;
  if (!B || !D) return 0;
  if (!T) {
    if (hT && hT != h0) {
      hipLaunchKernelGGL(scan_pass_kernel, dim3(grid_for((long)B * D)), dim3(256), 0, st, h0, hT, (long)B * D);
      return (int)hipGetLastError();
    }
    return 0;
  }
  if (!f || !v || !y) return crnn_set_error(hipErrorInvalidValue, "gated_scan_fwd: null f / v / y");
  const size_t need = crnn_gated_scan_workspace(dtype, B, T, D, dir);
  if (need && (!ws || ws_bytes < need)) return crnn_set_error(hipErrorInvalidValue, "gated_scan_fwd: workspace too small");
  if (need && hT && hT == h0)   // one segment's workgroup would overwrite what another still reads
    return crnn_set_error(hipErrorInvalidValue, "gated_scan_fwd: hT == h0 needs an unsegmented sequence (workspace 0)");
  ScanArgs a = {};
  a.f = f; a.fsb = fsb; a.fst = fst;
  a.v = v; a.vsb = vsb; a.vst = vst;
  a.y = y; a.ysb = ysb; a.yst = yst;
  a.h0 = h0; a.hT = hT; a.ckpt = ckpt; a.sum = ws; a.lengths = lengths;
  a.B = B; a.T = T; a.D = D; a.dir = dir;
  return dtype == CRNN_BF16 ? scan_run<bf16, false>(a, st) : scan_run<float, false>(a, st);
}

int crnn_gated_scan_bwd(int dtype, const void* dy, long dsb, long dst, const void* f, long fsb, long fst, const void* v,
                        long vsb, long vst, const int* lengths, const float* dhT, const float* ckpt, void* df, long gsb,
                        long gst, void* dv, long wsb, long wst, float* dh0, float* ws, size_t ws_bytes, int B, int T, int D,
                        int dir, void* stream) {
  if (bad_shape(dtype, B, T, D, dir))
    return crnn_set_error(hipErrorInvalidValue, "gated_scan_bwd: dtype fp32 or bf16, B/T/D >= 0, T, D <= 2^30, dir 0..2 (2: even D)");
  hipStream_t st = (hipStream_t)stream;
  if (!B || !D) return 0;
  if (!T) {
    if (dh0 && dh0 != dhT) {
      hipLaunchKernelGGL(scan_pass_kernel, dim3(grid_for((long)B * D)), dim3(256), 0, st, dhT, dh0, (long)B * D);
      return (int)hipGetLastError();
    }
    return 0;
  }
  if (!dy || !f || !v || !df || !dv || !ckpt) return crnn_set_error(hipErrorInvalidValue, "gated_scan_bwd: null dy / f / v / df / dv / ckpt");
  const size_t need = crnn_gated_scan_workspace(dtype, B, T, D, dir);
  if (need && (!ws || ws_bytes < need)) return crnn_set_error(hipErrorInvalidValue, "gated_scan_bwd: workspace too small");
  if (need && dh0 && dh0 == dhT)   // the first segment's workgroup would overwrite what the others still read
    return crnn_set_error(hipErrorInvalidValue, "gated_scan_bwd: dh0 == dhT needs an unsegmented sequence (workspace 0)");
  ScanArgs a = {};
  a.dy = dy; a.dsb = dsb; a.dst = dst;
  a.f = f; a.fsb = fsb; a.fst = fst;
  a.v = v; a.vsb = vsb; a.vst = vst;
  a.df = df; a.gsb = gsb; a.gst = gst;
  a.dv = dv; a.wsb = wsb; a.wst = wst;
  a.dhT = dhT; a.dh0 = dh0; a.ckpt = const_cast<float*>(ckpt); a.sum = ws; a.lengths = lengths;
  a.B = B; a.T = T; a.D = D; a.dir = dir;
  return dtype == CRNN_BF16 ? scan_run<bf16, true>(a, st) : scan_run<float, true>(a, st);
}

}  // extern "C"
