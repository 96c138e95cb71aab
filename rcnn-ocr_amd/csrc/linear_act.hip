// nn.Linear with its epilogue, forward and backward (the projections and the feed-forward of the gated-linear-recurrence
// encoder layer, crnn_hip/glr.py; crnn_hip.linear).
//
//   y = act(z) + res,  z = x w^T + bias;    dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = sum_m dz
//
// The products run on the shared MFMA cores (gemm.hpp, gemm256.hpp); what is here is the epilogue (bias, activation,
// residual, the pre-activation for the backward: nothing is read or written twice), the pass that turns dy into dz and
// sums its columns, and the split-K weight gradient in fixed order.
#include "gemm.hpp"
#include "gemm256.hpp"
#include "crnn_internal.hpp"

using namespace gemm;

namespace {

// ---------------------------------------------------------------- four elements at an element-aligned address
template <typename T> __device__ __forceinline__ f32x4 ld4u(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const f32x4_u*>(p);
  } else {
    const bf16x4 b = *reinterpret_cast<const bf16x4_u*>(p);
    return f32x4{(float)b[0], (float)b[1], (float)b[2], (float)b[3]};
  }
}
template <typename T> __device__ __forceinline__ void st4u(T* p, f32x4 v) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4_u*>(p) = v;
  else *reinterpret_cast<bf16x4_u*>(p) = bf16x4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
}

// ---------------------------------------------------------------- activations
// Phi(-|z|) = erfc(|z| / sqrt 2) / 2 and e = exp(-z^2 / 2). For bf16 results erfc(x) = t P(t) e^{-x^2}, t = 1 / (1 + 0.435 x), P the
// degree-5 polynomial of least relative error over 0 <= x <= 9.4 (3.7e-6, fitted by reweighted least squares; half a bf16 step
// is 3.9e-3; the constants below carry the half and the sqrt 2): 14 instructions where erfcf takes several times that. They are
// not hidden under the matrix instructions (one workgroup per CU): 32768 x 768 -> 1536 takes 84 us with relu, 107 with this.
__device__ __forceinline__ float gauss_tail(float z, float& e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.30759145f, 1.f));   // 0.435 / sqrt 2
  e = __builtin_amdgcn_exp2f(z * z * -0.72134752f);                          // log2(e) / 2
  float p = -0.075867921f;
  p = fmaf(p, t, 0.19190247f);
  p = fmaf(p, t, 0.0050641913f);
  p = fmaf(p, t, 0.13742310f);
  p = fmaf(p, t, 0.11849837f);
  p = fmaf(p, t, 0.12297796f);
  return p * t * e;
}
template <typename T, int ACT> __device__ __forceinline__ float act(float z) {
  if constexpr (ACT == CRNN_ACT_RELU) return z > 0.f ? z : (z == z ? 0.f : z);
  if constexpr (ACT == CRNN_ACT_GELU) {
    if constexpr (sizeof(T) == 2) {
      float e;
      const float q = gauss_tail(z, e);
      return fmaf(-fminf(fabsf(z), 20.f), q, fmaxf(z, 0.f));   // z Phi(z); the min keeps infinities off q = 0
    } else {
      return 0.5f * z * erfcf(-0.70710678118654752f * z);
    }
  }
  if constexpr (ACT == CRNN_ACT_SILU) {
    if constexpr (sizeof(T) == 2) return z * sigmoid_fast(z);
    else return z / (1.f + expf(-z));
  }
  return z;
}
// act'(z)
template <typename T> __device__ __forceinline__ float dact(int kind, float z) {
  constexpr float kC = 0.3989422804014327f;   // 1 / sqrt(2 pi)
  if (kind == CRNN_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (kind == CRNN_ACT_GELU) {
    if constexpr (sizeof(T) == 2) {
      float e;
      const float q = gauss_tail(z, e);
      return fmaf(z * kC, e, 0.5f + copysignf(0.5f - q, z));
    } else {
      return 0.5f * erfcf(-0.70710678118654752f * z) + z * expf(-0.5f * z * z) * kC;
    }
  }
  if (kind == CRNN_ACT_SILU) {
    if constexpr (sizeof(T) == 2) {
      const float s = sigmoid_fast(z);
      return s * (1.f + z * (1.f - s));
    } else {
      const float s = 1.f / (1.f + expf(-z)), r = 1.f / (1.f + expf(z));
      return s * (1.f + z * r);
    }
  }
  return 1.f;
}

// ---------------------------------------------------------------- forward epilogue
template <typename T, int ACT, bool OWN = false> struct ActEpi {
  static constexpr bool kStats = false;
  // the deep kernels: the wave's accumulators through its LDS, so that a lane stores 8 consecutive columns (16 bytes), and
  // the residual's loads all in flight before the first store (between stores that may alias them each waits for its own:
  // 32768 x 1536 -> 768 with residual 139 us, 86 together)
  static constexpr bool kOwnTile = OWN;
  T *y, *z;
  const T* res;
  const void* bias;
  long ldy, ldz, ldr;
  int M, N, bias_f32;
  __device__ __forceinline__ float b(int n) const { return bias_f32 ? ((const float*)bias)[n] : tof(((const T*)bias)[n]); }
  __device__ __forceinline__ void store(int m, int n, f32x4 v, int) const {
    if (m >= M || n >= N) return;
    if (n + 4 <= N) {
      if (bias)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += b(n + r);
      if (z) st4u<T>(z + m * ldz + n, v);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = act<T, ACT>(v[r]);
      if (res) v += ld4u<T>(res + m * ldr + n);
      st4u<T>(y + m * ldy + n, v);
      return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < N) {
        float u = v[r];
        if (bias) u += b(n + r);
        if (z) z[m * ldz + n + r] = fromf<T>(u);
        u = act<T, ACT>(u);
        if (res) u += tof(res[m * ldr + n + r]);
        y[m * ldy + n + r] = fromf<T>(u);
      }
  }
  template <int MI, int NI, int WM, int WN>
  __device__ __forceinline__ void own_tile(const f32x4 (&acc)[MI][NI], float* stg, int lane, int rbase, int cbase) const {
    static_assert(WM == 128 && (WN == 64 || WN == 32), "256-row tiles");
    constexpr int CH = WN / 4;            // 16-byte chunks of a row
    constexpr int LPR = WN / 8;           // lanes per row in the read-back
    constexpr int RPI = 64 / LPR;         // rows per read-back instruction
    constexpr int NIT = 64 / RPI;
    const int mr = lane & 15, g = lane >> 4;
    const int c = (lane % LPR) * 8, n = cbase + c, rl = lane / LPR;
    const bool full = n + 8 <= N;         // this lane's 8 columns as vectors
    float bs[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bs[e] = bias && n + e < N ? b(n + e) : 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 rv[NIT];
      if (res && full) {
#pragma unroll
        for (int it = 0; it < NIT; ++it) {
          const int m = rbase + h * 64 + it * RPI + rl;
          rv[it] = *reinterpret_cast<const bf16x8_u*>(res + (m < M ? m : M - 1) * ldr + n);
        }
      }
#pragma unroll
      for (int ii = 0; ii < MI / 2; ++ii)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const int r = ii * 16 + mr, q = (4 * j + g) ^ (r & (CH - 1));
          *reinterpret_cast<f32x4*>(stg + r * WN + 4 * q) = acc[h * (MI / 2) + ii][j];
        }
#pragma unroll
      for (int it = 0; it < NIT; ++it) {
        const int r = it * RPI + rl, m = rbase + h * 64 + r;
        const int q0 = (c / 4) ^ (r & (CH - 1)), q1 = (c / 4 + 1) ^ (r & (CH - 1));
        const f32x4 lo = *reinterpret_cast<const f32x4*>(stg + r * WN + 4 * q0);
        const f32x4 hi = *reinterpret_cast<const f32x4*>(stg + r * WN + 4 * q1);
        float u[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u[e] = lo[e] + bs[e];
          u[4 + e] = hi[e] + bs[4 + e];
        }
        if (m < M && full) {
          if (z) *reinterpret_cast<bf16x8_u*>(z + m * ldz + n) = pack8<bf16>(u);
#pragma unroll
          for (int e = 0; e < 8; ++e) u[e] = act<bf16, ACT>(u[e]);
          if (res) {
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] += (float)rv[it][e];
          }
          *reinterpret_cast<bf16x8_u*>(y + m * ldy + n) = pack8<bf16>(u);
        } else if (m < M) {
          for (int e = 0; e < 8 && n + e < N; ++e) {
            if (z) z[m * ldz + n + e] = (bf16)u[e];
            float o = act<bf16, ACT>(u[e]);
            if (res) o += (float)res[m * ldr + n + e];
            y[m * ldy + n + e] = (bf16)o;
          }
        }
      }
    }
  }
  __device__ __forceinline__ void stats(int, int, f32x4, f32x4) const {}
};

// ---------------------------------------------------------------- operands
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int round8i(int n) { return (n + 7) & ~7; }
// the LDS-DMA kernels and gemm.hpp's loaders read 16-byte vectors of 8 elements (fp32: two of 4): the base, the row pitch and the
// row length have to be whole vectors. Other operands are copied into such rows for the deep kernels, and read as they lie by
// the register-staged ones (1027 x 509 x 1021 fp32, forward / backward: 28.6 / 63.3 us with copies, 25.5 / 59.9 without).
bool direct(const void* p, long ld, int cols, int es) {
  return aligned16(p) && ld * es % 16 == 0 && cols % 8 == 0 && ld < 0x7fffffffL;
}
// rows of one launch: the loaders address an operand with 32-bit byte offsets, and a grid of 32 x 32 tiles over `cols` columns has
// to stay under 2^32 threads
long max_rows(long ld, int es, int cols = 1) {
  long r = 0x7fffffffL / (ld * es);
  const long g = (1L << 23) / ((cols + 31L) / 32) * 32;
  if (r > g) r = g < 256 ? 256 : g;
  return r >= 256 ? r / 256 * 256 : r;
}

// dst[rows][cols8] (zero behind cols) = src[rows][ld], up to two matrices in one launch (blockIdx.y)
struct PadJob {
  const void* src;
  void* dst;
  long ld, rows;
  int cols;
};
template <typename T> __global__ __launch_bounds__(256) void pad_copy_kernel(PadJob j0, PadJob j1) {
  const PadJob j = blockIdx.y ? j1 : j0;
  const int c8 = (j.cols + 7) / 8;
  const long n8 = j.rows * c8;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n8; i += gridDim.x * 256L) {
    const long r = i / c8;
    const int c = (int)(i - r * c8) * 8;
    st8<T>((T*)j.dst + (r * c8 + c / 8) * 8, ld8_row<T>((const T*)j.src + r * j.ld, c, j.cols));
  }
}
// copies the given jobs (src NULL: none)
template <typename T> int pad_copy(PadJob a, PadJob b, hipStream_t st) {
  if (!a.src) {
    a = b;
    b.src = nullptr;
  }
  if (!a.src) return 0;
  const long na = a.rows * (round8i(a.cols) / 8), nb = b.src ? b.rows * (round8i(b.cols) / 8) : 0;
  hipLaunchKernelGGL(pad_copy_kernel<T>, dim3(grid_for(na > nb ? na : nb, 256, 4096), b.src ? 2 : 1), dim3(256), 0, st, a, b);
  return (int)hipGetLastError();
}

// loaders of the register-staged kernels for operands as they lie (gemm.hpp's interface): element (row, k) at p[row * ld + k] ..
template <typename T> struct RowsAny {
  static constexpr bool kRowVec = false;
  const T* p;
  long ld;
  int rows, K;
  struct Ctx { const T* row; };
  typedef int Prep;
  __device__ __forceinline__ Ctx row_ctx(int r) const { return Ctx{r < rows ? p + r * ld : nullptr}; }
  __device__ __forceinline__ Prep prep(int k0) const { return k0; }
  __device__ __forceinline__ typename VT<T>::v8 load(const Ctx& c, Prep k0, int kofs) const {
    return c.row ? ld8_row<T>(c.row, k0 + kofs, K) : zero8<T>();
  }
};
// .. and at p[k * ld + row], 8 rows per vector
template <typename T> struct ColsAny {
  static constexpr bool kRowVec = true;
  const T* p;
  long ld;
  int rows, K;
  struct Ctx { int r8; };
  typedef int Prep;
  __device__ __forceinline__ Ctx row_ctx(int r8) const { return Ctx{r8}; }
  __device__ __forceinline__ Prep prep(int k0) const { return k0; }
  __device__ __forceinline__ typename VT<T>::v8 load(const Ctx& c, Prep k0, int kofs) const {
    const int k = k0 + kofs;
    return k < K ? ld8_row<T>(p + k * ld, c.r8, rows) : zero8<T>();
  }
};

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// ---------------------------------------------------------------- tile plans
// Products with rows as outputs (forward, dx). bf16: the deep 256-row kernels where their tiles fill three quarters of the
// CUs; a round of 256 x 256 tiles costs 1.4 rounds of 256 x 128 ones, so the fewer weighted rounds win (32768 x 768 x 1536:
// 86 us at 2 rounds of the former, 94 at 3 of the latter; 8192 x 1024 x 512: 24 at half a round, 20 at a whole one).
// Else 64 x 64 register-staged tiles where there is one per CU (4096 x 512 x 512: 12.8 us; 256 x 128 tiles 19.8, 128 x 128
// 19.8, 32 x 32 13.6), else 32 x 32 (500 x 520 x 512: 8.0 against 9.1). fp32 (exact-fp32 MFMA, 1/16 of the bf16 rate): 64 x 64
// at two per CU or more (8192 x 1024 x 512: 84.8 us, 128 x 128 83.0, 32 x 32 101; forward and input gradient of 4096 x 512 x 512
// 25.9 and 22.9, 32 x 32 28.2 and 28.6), else 32 x 32 with 64-deep stages (1032 x 1024 x 512: 19.7 against 24.4 of 64 x 64;
// 304 x 520 x 1000: 13.1 against 28.7).
// 0: register-staged, else the columns of the deep kernel's tile
int deep_tile(int es, long M, int N, int K) {
  const long cu = crnn_cu_count(), t256 = (M + 255) / 256 * ((N + 255) / 256), t128 = (M + 255) / 256 * ((N + 127) / 128);
  if (es != 2 || K < 256 || N < 128 || t128 * 4 < cu * 3) return 0;
  return (t256 + cu - 1) / cu * 7 <= (t128 + cu - 1) / cu * 5 ? 256 : 128;
}
template <typename T, int ACT, class LA, class LB>
int staged_run(const LA& la, const LB& lb, const ActEpi<T, ACT>& ep, int M, int N, int K, hipStream_t st) {
  const long cu = crnn_cu_count(), t64 = (long)((M + 63) / 64) * ((N + 63) / 64);
  if (t64 >= (sizeof(T) == 2 ? cu : 2 * cu)) return launch<T, 64, 64>(la, lb, ep, M, N, K, 1, st);
  return launch<T, 32, 32, 64>(la, lb, ep, M, N, K, 1, st);
}
template <typename T, int ACT, class LA, class LB>
int tiles_run(const LA& la, const LB& lb, const ActEpi<T, ACT>& ep, int M, int N, int K, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    const int tile = deep_tile(2, M, N, K);
    const ActEpi<T, ACT, true> eo{ep.y, ep.z, ep.res, ep.bias, ep.ldy, ep.ldz, ep.ldr, ep.M, ep.N, ep.bias_f32};
    if (tile == 256) return launch256<256, 256>(la, lb, eo, M, N, K, st);
    if (tile == 128) return launch256<256, 128>(la, lb, eo, M, N, K, st);
  }
  return staged_run<T, ACT>(la, lb, ep, M, N, K, st);
}

// ---------------------------------------------------------------- few rows
// M <= 16 * MT rows (single frames of running lines): the product is a read of w, so a workgroup takes 16 of its rows (output
// columns) and its 8 waves split K: fragments straight from memory to registers (a lane holds 8 consecutive k of a row, the
// layout of the matrix instruction's operands), no staging, and one join in LDS. Any alignment: nothing is copied first.
// bf16 2048 x 2048 (8 MB of w), us: 4.9 / 6.2 / 8.1 at 1 / 16 / 32 rows, 10.6 in 32 x 32 tiles; 64 rows 11.6 against 10.8, so those
// stay with the tiles (fp32: 7.9 / 10.8 / 15.5 against 19.5; 512 x 1024 bf16, launch-bound: 4.6 / 4.6 / 5.3 against 5.0).
constexpr int SKINNY_ROWS = 32, SKW = 8;
template <typename T, int ACT, int MT>
__global__ __launch_bounds__(64 * SKW) void skinny_kernel(const T* __restrict__ x, long ldx, const T* __restrict__ w, long ldw,
                                                          ActEpi<T, ACT> ep, int M, int N, int K) {
  __shared__ f32x4 red[SKW][MT][64];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g8 = 8 * (lane >> 4);
  const int n0 = blockIdx.x * 16;
  const T* wr = w + min(n0 + c, N - 1) * ldw;   // rows past the end repeat the last: their outputs are not stored
  const T* xr[MT];
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    xr[i] = x + min(i * 16 + c, M - 1) * ldx;
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  constexpr int U = 4;   // steps of 32 in flight
  for (int k0 = wid * 32; k0 < K; k0 += SKW * 32 * U) {
    typename VT<T>::v8 b[U], a[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * SKW * 32 + g8;
      b[u] = ld8_row<T>(wr, k, K);
#pragma unroll
      for (int i = 0; i < MT; ++i) a[u][i] = ld8_row<T>(xr[i], k, K);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i) mma<T>(acc[i], b[u], a[u][i]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) red[wid][i][lane] = acc[i];
  __syncthreads();
  if (wid < MT) {
    f32x4 v = red[0][wid][lane];
#pragma unroll
    for (int q = 1; q < SKW; ++q) v += red[q][wid][lane];
    ep.store(wid * 16 + c, n0 + 4 * (lane >> 4), v, 0);
  }
}
template <typename T, int ACT>
int skinny_run(const T* x, long ldx, const T* w, long ldw, const ActEpi<T, ACT>& ep, int M, int N, int K, hipStream_t st) {
  const dim3 grid((N + 15) / 16), block(64 * SKW);
  if (M <= 16) hipLaunchKernelGGL((skinny_kernel<T, ACT, 1>), grid, block, 0, st, x, ldx, w, ldw, ep, M, N, K);
  else hipLaunchKernelGGL((skinny_kernel<T, ACT, 2>), grid, block, 0, st, x, ldx, w, ldw, ep, M, N, K);
  return (int)hipGetLastError();
}

template <typename T, int ACT>
int fwd_act(const T* x, long ldx, const T* w, long ldw, const void* bias, int bias_f32, const T* res, long ldr, T* y, long ldy, T* z,
            long ldz, long M, int N, int K, hipStream_t st) {
  if (M <= SKINNY_ROWS) {
    const ActEpi<T, ACT> ep{y, z, res, bias, ldy, ldz, ldr, (int)M, N, bias_f32};
    return skinny_run<T, ACT>(x, ldx, w, ldw, ep, (int)M, N, K, st);
  }
  const bool any = !direct(x, ldx, K, sizeof(T)) || !direct(w, ldw, K, sizeof(T));   // then the plan is register-staged (fwd_copies)
  const long step = max_rows(ldx, sizeof(T), N);
  for (long m0 = 0; m0 < M; m0 += step) {
    const int m = (int)(M - m0 < step ? M - m0 : step);
    const ActEpi<T, ACT> ep{y + m0 * ldy, z ? z + m0 * ldz : nullptr, res ? res + m0 * ldr : nullptr, bias, ldy, ldz, ldr, m, N, bias_f32};
    const int rc = any ? staged_run<T, ACT>(RowsAny<T>{x + m0 * ldx, ldx, m, K}, RowsAny<T>{w, ldw, N, K}, ep, m, N, K, st)
                       : tiles_run<T, ACT>(RowMajorK<T>{x + m0 * ldx, (int)ldx, m, K}, RowMajorK<T>{w, (int)ldw, N, K}, ep, m, N, K, st);
    if (rc) return rc;
  }
  return 0;
}

// what the forward copies into aligned rows first: only the deep kernels ask for it
struct FwdCopies { bool x, w; };
FwdCopies fwd_copies(int es, const void* x, long ldx, const void* w, long ldw, long M, int N, int K) {
  if (M <= SKINNY_ROWS || !deep_tile(es, M, N, round8i(K))) return {false, false};
  return {!direct(x, ldx, K, es), !direct(w, ldw, K, es)};
}

template <typename T>
int fwd_t(const void* x, long ldx, const void* w, long ldw, const void* bias, int bias_f32, int kind, const void* res, long ldr,
          void* y, long ldy, void* z, long ldz, char* ws, long M, int N, int K, hipStream_t st) {
  const T *xp = (const T*)x, *wp = (const T*)w;
  PadJob jx = {}, jw = {};
  const FwdCopies cp = fwd_copies(sizeof(T), x, ldx, w, ldw, M, N, K);
  const int K8 = round8i(K);
  if (cp.x) {
    jx = {x, ws, ldx, M, K};
    xp = (const T*)ws;
    ldx = K8;
    ws += up256((size_t)M * K8 * sizeof(T));
  }
  if (cp.w) {
    jw = {w, ws, ldw, N, K};
    wp = (const T*)ws;
    ldw = K8;
  }
  const int rc = pad_copy<T>(jx, jw, st);
  if (rc) return rc;
#define FWD(A) fwd_act<T, A>(xp, ldx, wp, ldw, bias, bias_f32, (const T*)res, ldr, (T*)y, ldy, (T*)z, ldz, M, N, cp.x || cp.w ? K8 : K, st)
  if (kind == CRNN_ACT_RELU) return FWD(CRNN_ACT_RELU);
  if (kind == CRNN_ACT_GELU) return FWD(CRNN_ACT_GELU);
  if (kind == CRNN_ACT_SILU) return FWD(CRNN_ACT_SILU);
  return FWD(CRNN_ACT_NONE);
#undef FWD
}

// ---------------------------------------------------------------- backward
// dz = dy act'(z) into dz [M][N8] (zero behind N; NULL: only the sums), and the partial column sums part[g][N] of row slice
// g (NULL: none). A thread owns 8 columns; the 8 row lanes of a workgroup join in LDS. fp32 throughout, the column sums add the unrounded
// values. dz is rounded once to the operands' type, since the bf16 matrix instructions take nothing else, and z was when it was stored
// (which halves what this pass reads). Against 64 bits, 8192 x 512 -> 1024 gelu bf16, relative norms: dx and dw 2.4e-3, of which
// the results' own rounding is 1.66e-3, dz's 1.66e-3 and z's 0.55e-3 (db 1.77e-3). Without them: dz in two bf16 parts, twice the matrix
// work of dx and dw.
template <typename T>
__global__ __launch_bounds__(256) void dz_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ z, long ldz, int kind,
                                                 T* __restrict__ dz, int N8, float* __restrict__ part, long M, int N) {
  __shared__ float red[8][32 * 8 + 8];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int n = (blockIdx.x * 32 + cl) * 8;
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = 0.f;
  constexpr int R = 2;   // rows in flight
  if (n < N8)
    for (long mb = (long)blockIdx.y * 8 + rl; mb < M; mb += 8L * R * gridDim.y) {
      typename VT<T>::v8 gr[R], zr[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const long m = mb + 8L * r * gridDim.y;
        gr[r] = zero8<T>();
        if (m < M) {
          gr[r] = ld8_row<T>(dy + m * lddy, n, N);
          if (z) zr[r] = ld8_row<T>(z + m * ldz, n, N);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const long m = mb + 8L * r * gridDim.y;
        if (m >= M) break;
        float g[8], q[8];
        unpack8<T>(gr[r], g);
        if (z) {
          unpack8<T>(zr[r], q);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] *= dact<T>(kind, q[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += g[e];
        if (dz) st8<T>(dz + m * N8 + n, pack8<T>(g));
      }
    }
  if (!part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[rl][cl * 8 + e] = s[e];
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c < N) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) t += red[r][threadIdx.x];
    part[(size_t)blockIdx.y * N + c] = t;
  }
}

template <typename O> __device__ __forceinline__ void put(O* o, float v, int accumulate) {
  if constexpr (sizeof(O) == 4) *o = accumulate ? *o + v : v;
  else *o = fromf<O>(v);
}

// split-K partials of dw into fp32 slabs [S][Nr][Kc] (whole vectors), then one fixed-order sum into dw [N][K]
struct SlabEpi {
  static constexpr bool kStats = false;
  float* ws;
  int M, N;
  __device__ __forceinline__ void store(int m, int n, f32x4 v, int kz) const {
    if (m < M && n < N) *reinterpret_cast<f32x4*>(ws + ((size_t)kz * M + m) * N + n) = v;
  }
  __device__ __forceinline__ void stats(int, int, f32x4, f32x4) const {}
};
// the last pass of the backward, one launch: workgroups [0, wblocks) add the S slabs into dw [N][K], the others G partial rows
// of the column sums into db (32 columns each, 8 row lanes); every sum in a fixed order
template <typename OW, typename OB>
__global__ __launch_bounds__(256) void reduce_kernel(const float* __restrict__ slab, int S, int Nr, int Kc, OW* __restrict__ dw,
                                                     int wblocks, const float* __restrict__ part, int G, OB* __restrict__ db, int N,
                                                     int K, int accumulate) {
  if ((int)blockIdx.x >= wblocks) {
    __shared__ float red[8][32];
    const int col = threadIdx.x & 31, rl = threadIdx.x >> 5, n = ((int)blockIdx.x - wblocks) * 32 + col;
    float s = 0.f;
    if (n < N) {
      int g = rl;
      for (; g + 15 * 8 < G; g += 16 * 8) {
        float v[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) v[u] = part[(size_t)(g + 8 * u) * N + n];
#pragma unroll
        for (int u = 0; u < 16; ++u) s += v[u];
      }
      for (; g < G; g += 8) s += part[(size_t)g * N + n];
    }
    red[rl][col] = s;
    __syncthreads();
    if (rl == 0 && n < N) {
#pragma unroll
      for (int r = 1; r < 8; ++r) s += red[r][col];
      put<OB>(db + n, s, accumulate);
    }
    return;
  }
  const long total = (long)Nr * Kc;
  for (long i4 = blockIdx.x * 256L + threadIdx.x; 4 * i4 < total; i4 += wblocks * 256L) {
    const long i = 4 * i4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    int z = 0;
    for (; z + 8 <= S; z += 8) {
      f32x4 v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = *reinterpret_cast<const f32x4*>(slab + (size_t)(z + q) * total + i);
#pragma unroll
      for (int q = 0; q < 8; ++q) s += v[q];
    }
    for (; z < S; ++z) s += *reinterpret_cast<const f32x4*>(slab + (size_t)z * total + i);
    const int n = (int)(i / Kc), k = (int)(i - (long)n * Kc);   // Kc % 8 == 0: the four share a row
    if (n >= N) continue;
    OW* o = dw + (size_t)n * K + k;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + e < K) put<OW>(o + e, s[e], accumulate);
  }
}

// row slices of the column sums: four workgroups per CU (a row a lane where there are few), few partial rows to add. With two rows
// in flight a lane; gelu' and the sums of 32768 x 1536 bf16, us: 45.5, two per CU and four rows 60, eight per CU 42.4; of
// 8192 x 1024: 12.3, 14.1, 13.4
int dz_slices(long M, int N) {
  const long cb = (round8i(N) + 255) / 256;
  long g = (4L * crnn_cu_count() + cb - 1) / cb;
  const long most = (M + 7) / 8;
  if (g > most) g = most;
  if (g > 256) g = 256;
  return (int)(g < 1 ? 1 : g);
}
// The weight gradient over `rows` rows: tile and K splits. Its outputs are few and its sum is long, so K is split until the
// chip is full, as long as a split keeps enough of the sum to be worth its slab (written and read once as fp32). bf16: the deep
// 256 x 256 kernel at one workgroup per CU if a split keeps 1024 rows (768 x 1536 over 32768: 75 us in 14 splits; 128 x 128
// 100 in 7), else 128 x 128 at two per CU if it keeps 512 (1024 x 512 over 8192: 21 in 16; 64 x 64 23, 256 x 256 23 in 32), else
// 64 x 64 (512 x 512 over 4096: 10.9 in 8; 128 x 128 11.6). fp32: 64 x 64 at four per CU (1024 x 512 over 1032: 19.9; 128 x 128
// 30.7) of 256 rows or more, of 128 where that leaves fewer than two (512 x 520 over 500: 17.1 and 10.8; 700 x 300 over 2000:
// 27.3 and 23.8; 1024 x 512 over 1024, which has two: 21.7 and 24.3).
struct DwPlan { int tile, splits; };
DwPlan dw_plan(int es, int Nr, int Kc, long rows) {
  const long cu = crnn_cu_count();
  auto tiles = [&](int b) { return (long)((Nr + b - 1) / b) * ((Kc + b - 1) / b); };
  auto split = [&](long wg, long least) {   // splits to reach wg workgroups, each of `least` rows or more
    const long s = wg < 1 ? 1 : wg, most = rows / least < 1 ? 1 : rows / least;
    return eff_splits((int)rows, (int)(s < most ? s : most));
  };
  if (es == 2) {
    const long s256 = cu / tiles(256), s128 = 2 * cu / tiles(128);
    if (s256 >= 1 ? rows / s256 >= 1024 : true) return {256, split(s256, 1024)};
    if (s128 >= 1 && rows / s128 >= 512) return {128, split(s128, 512)};
    return {64, split(2 * cu / tiles(64), 256)};
  }
  const int s = split(4 * cu / tiles(64), 256);
  return {64, s * tiles(64) < 2 * cu ? split(4 * cu / tiles(64), 128) : s};
}

// the layout of crnn_linear_bwd's workspace
struct BwdPlan {
  bool copy_x, copy_w, own_dz;
  int N8, K8, slices, slabs;
  size_t o_dz, o_x, o_w, o_part, o_slab, total;
};
BwdPlan bwd_plan(int dtype, const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw, int kind, int need_dx,
                 int need_dw, int need_db, long M, int N, int K) {
  const int es = dtype == CRNN_BF16 ? 2 : 4;
  BwdPlan p = {};
  p.N8 = round8i(N);
  p.K8 = round8i(K);
  // operands that are not whole aligned vectors are copied for the deep kernels only; without an activation dy is dz
  const bool deep_dx = need_dx && deep_tile(es, M, K, p.N8), deep_dw = need_dw && dw_plan(es, p.N8, p.K8, M).tile == 256;
  p.own_dz = (need_dx || need_dw) && (kind != CRNN_ACT_NONE || (!direct(dy, lddy, N, es) && (deep_dx || deep_dw)));
  p.copy_x = !direct(x, ldx, K, es) && deep_dw;
  p.copy_w = !direct(w, ldw, K, es) && deep_dx;
  p.slices = need_db ? dz_slices(M, N) : 0;
  const long ldz_ = p.own_dz ? p.N8 : lddy, ldx_ = p.copy_x ? p.K8 : ldx;
  if (need_dw && M > 0) {
    const long step = max_rows(ldz_ > ldx_ ? ldz_ : ldx_, es);
    for (long m0 = 0; m0 < M; m0 += step) p.slabs += dw_plan(es, p.N8, p.K8, M - m0 < step ? M - m0 : step).splits;
  }
  size_t o = 0;
  p.o_dz = o;
  if (p.own_dz) o += up256((size_t)M * p.N8 * es);
  p.o_x = o;
  if (p.copy_x) o += up256((size_t)M * p.K8 * es);
  p.o_w = o;
  if (p.copy_w) o += up256((size_t)N * p.K8 * es);
  p.o_part = o;
  o += up256((size_t)p.slices * N * sizeof(float));
  p.o_slab = o;
  o += (size_t)p.slabs * p.N8 * p.K8 * sizeof(float);
  p.total = o;
  return p;
}

template <typename T>
int bwd_t(const BwdPlan& p, const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw, const void* z, long ldz,
          int kind, void* dx, long lddx, void* dw, int dw_f32, void* db, int db_f32, int accumulate, char* ws, long M, int N, int K,
          hipStream_t st) {
  int rc = 0;
  const T *dzp = (const T*)dy, *xp = (const T*)x, *wp = (const T*)w;
  long ldd = lddy;
  float* part = (float*)(ws + p.o_part);
  if ((p.own_dz || db) && M > 0) {
    T* out = p.own_dz ? (T*)(ws + p.o_dz) : nullptr;
    const int gy = db ? p.slices : dz_slices(M, N);
    hipLaunchKernelGGL(dz_kernel<T>, dim3((p.N8 + 255) / 256, gy), dim3(256), 0, st, (const T*)dy, lddy, (const T*)z, ldz, kind, out,
                       p.N8, db ? part : nullptr, M, N);
    if ((rc = (int)hipGetLastError())) return rc;
    if (out) {
      dzp = out;
      ldd = p.N8;
    }
  }
  const bool dz_direct = p.own_dz || direct(dy, lddy, N, sizeof(T));
  if (M > 0) {
    PadJob jx = {}, jw = {};
    if (p.copy_x) {
      jx = {x, ws + p.o_x, ldx, M, K};
      xp = (const T*)(ws + p.o_x);
      ldx = p.K8;
    }
    if (p.copy_w) {
      jw = {w, ws + p.o_w, ldw, N, K};
      wp = (const T*)(ws + p.o_w);
      ldw = p.K8;
    }
    if ((rc = pad_copy<T>(jx, jw, st))) return rc;
  }
  if (dx && M > 0) {
    const long step = max_rows(ldd, sizeof(T), K);
    for (long m0 = 0; m0 < M; m0 += step) {
      const int m = (int)(M - m0 < step ? M - m0 : step);
      const ActEpi<T, CRNN_ACT_NONE> ep{(T*)dx + m0 * lddx, nullptr, nullptr, nullptr, lddx, 0, 0, m, K, 0};
      // (columns behind K of a copied w, and behind N of an own dz, are zero)
      if (dz_direct && direct(wp, ldw, p.copy_w ? p.K8 : K, sizeof(T)))
        rc = tiles_run<T, CRNN_ACT_NONE>(RowMajorK<T>{dzp + m0 * ldd, (int)ldd, m, p.N8}, ColMajorK<T>{wp, (int)ldw, p.K8, N}, ep, m, K,
                                         p.N8, st);
      else
        rc = staged_run<T, CRNN_ACT_NONE>(RowsAny<T>{dzp + m0 * ldd, ldd, m, N}, ColsAny<T>{wp, ldw, K, N}, ep, m, K, p.N8, st);
      if (rc) return rc;
    }
  }
  const float* slab = (const float*)(ws + p.o_slab);
  int S = 0;
  if (dw && M > 0) {
    const long step = max_rows(ldd > ldx ? ldd : ldx, sizeof(T));
    for (long m0 = 0; m0 < M; m0 += step) {
      const int m = (int)(M - m0 < step ? M - m0 : step);
      const DwPlan d = dw_plan(sizeof(T), p.N8, p.K8, m);
      const SlabEpi ep{(float*)(ws + p.o_slab) + (size_t)S * p.N8 * p.K8, p.N8, p.K8};
      auto staged = [&](auto la, auto lb) {
        return sizeof(T) == 2 && d.tile != 64 ? launch<T, 128, 128>(la, lb, ep, p.N8, p.K8, m, d.splits, st)
                                              : launch<T, 64, 64>(la, lb, ep, p.N8, p.K8, m, d.splits, st);
      };
      if (dz_direct && direct(xp, ldx, p.copy_x ? p.K8 : K, sizeof(T))) {
        const ColMajorK<T> la{dzp + m0 * ldd, (int)ldd, p.N8, m}, lb{xp + m0 * ldx, (int)ldx, p.K8, m};
        if constexpr (sizeof(T) == 2) rc = d.tile == 256 ? launch256<256, 256>(la, lb, ep, p.N8, p.K8, m, st, d.splits) : staged(la, lb);
        else rc = staged(la, lb);
      } else {   // (rows of dz behind N and columns of x behind K are zero)
        rc = staged(ColsAny<T>{dzp + m0 * ldd, ldd, N, m}, ColsAny<T>{xp + m0 * ldx, ldx, K, m});
      }
      if (rc) return rc;
      S += d.splits;
    }
  }
  if (dw || db) {
    const int wb = dw ? grid_for((long)p.N8 * p.K8 / 4, 256, 2048) : 0, bb = db ? (N + 31) / 32 : 0, G = M > 0 ? p.slices : 0;
    auto go = [&](auto ow, auto ob) {
      typedef decltype(ow) OW;
      typedef decltype(ob) OB;
      hipLaunchKernelGGL((reduce_kernel<OW, OB>), dim3(wb + bb), dim3(256), 0, st, slab, S, p.N8, p.K8, (OW*)dw, wb, part, G, (OB*)db,
                         N, K, accumulate);
    };
    if (dw_f32 || sizeof(T) == 4) {
      if (db_f32 || sizeof(T) == 4) go(float(), float());
      else go(float(), bf16());
    } else {
      if (db_f32) go(bf16(), float());
      else go(bf16(), bf16());
    }
    rc = (int)hipGetLastError();
  }
  return rc;
}

bool bad_linear(int dtype, int kind, long M, int N, int K) {
  return (dtype != CRNN_F32 && dtype != CRNN_BF16) || kind < CRNN_ACT_NONE || kind > CRNN_ACT_SILU || M < 0 || N < 1 || K < 1 ||
         N > 0x7ffffff0 || K > 0x7ffffff0;
}
// an operand row has to stay under the loaders' 2 GiB, and so does w
bool too_big(int es, long ldx, long ldw, int N, int K) {
  const long k8 = round8i(K);
  return (ldx > k8 ? ldx : k8) * es > 0x7fffffffL || (ldw > k8 ? ldw : k8) > 0x7fffffffL / es / (long)N;
}

}  // namespace

extern "C" {

size_t crnn_linear_fwd_workspace(int dtype, const void* x, long ldx, const void* w, long ldw, long M, int N, int K) {
  if (bad_linear(dtype, 0, M, N, K)) return 0;
  const int es = dtype == CRNN_BF16 ? 2 : 4;
  const FwdCopies cp = fwd_copies(es, x, ldx, w, ldw, M, N, K);
  return (cp.x ? up256((size_t)M * round8i(K) * es) : 0) + (cp.w ? up256((size_t)N * round8i(K) * es) : 0);
}

int crnn_linear_fwd(int dtype, const void* x, long ldx, const void* w, long ldw, const void* bias, int bias_f32, int act, const void* res,
                    long ldr, void* y, long ldy, void* z, long ldz, void* ws, size_t ws_bytes, long M, int N, int K, void* stream) {
  if (bad_linear(dtype, act, M, N, K)) return crnn_set_error(hipErrorInvalidValue, "linear_fwd: dtype fp32 or bf16, act CRNN_ACT_*, M >= 0, N, K >= 1");
  if (ldx < K || ldw < K || ldy < N || (z && ldz < N) || (res && ldr < N)) return crnn_set_error(hipErrorInvalidValue, "linear_fwd: a row stride is shorter than its row");
  if (M == 0) return 0;
  if (!x || !w || !y) return crnn_set_error(hipErrorInvalidValue, "linear_fwd: null x / w / y");
  if (too_big(dtype == CRNN_BF16 ? 2 : 4, ldx, ldw, N, K)) return crnn_set_error(hipErrorInvalidValue, "linear_fwd: w (or a row of x) of 2 GiB or more");
  const size_t need = crnn_linear_fwd_workspace(dtype, x, ldx, w, ldw, M, N, K);
  if (need && (!ws || !aligned16(ws) || ws_bytes < need)) return crnn_set_error(hipErrorInvalidValue, "linear_fwd: workspace too small or unaligned");
  hipStream_t st = (hipStream_t)stream;
  return dtype == CRNN_BF16 ? fwd_t<bf16>(x, ldx, w, ldw, bias, bias_f32, act, res, ldr, y, ldy, z, ldz, (char*)ws, M, N, K, st)
                            : fwd_t<float>(x, ldx, w, ldw, bias, bias_f32, act, res, ldr, y, ldy, z, ldz, (char*)ws, M, N, K, st);
}

size_t crnn_linear_bwd_workspace(int dtype, const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw, int act,
                                 int need_dx, int need_dw, int need_db, long M, int N, int K) {
  if (bad_linear(dtype, act, M, N, K)) return 0;
  return bwd_plan(dtype, dy, lddy, x, ldx, w, ldw, act, need_dx, need_dw, need_db, M, N, K).total;
}

int crnn_linear_bwd(int dtype, const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw, const void* z, long ldz,
                    int act, void* dx, long lddx, void* dw, int dw_f32, void* db, int db_f32, int accumulate, void* ws, size_t ws_bytes,
                    long M, int N, int K, void* stream) {
  if (bad_linear(dtype, act, M, N, K)) return crnn_set_error(hipErrorInvalidValue, "linear_bwd: dtype fp32 or bf16, act CRNN_ACT_*, M >= 0, N, K >= 1");
  if (lddy < N || (dw && ldx < K) || (dx && (ldw < K || lddx < K)) || (act != CRNN_ACT_NONE && ldz < N))
    return crnn_set_error(hipErrorInvalidValue, "linear_bwd: a row stride is shorter than its row");
  if (M > 0 && (!dy || (dw && !x) || (dx && !w) || (act != CRNN_ACT_NONE && !z))) return crnn_set_error(hipErrorInvalidValue, "linear_bwd: null dy / x / w / z");
  if (accumulate && ((dw && !dw_f32 && dtype != CRNN_F32) || (db && !db_f32 && dtype != CRNN_F32)))
    return crnn_set_error(hipErrorInvalidValue, "linear_bwd: accumulate needs fp32 dw and db");
  if (too_big(dtype == CRNN_BF16 ? 2 : 4, dw ? ldx : K, dx ? ldw : K, N, K) || too_big(dtype == CRNN_BF16 ? 2 : 4, lddy, K, N, K))
    return crnn_set_error(hipErrorInvalidValue, "linear_bwd: w (or a row of x, dy) of 2 GiB or more");
  const BwdPlan p = bwd_plan(dtype, dy, lddy, x, ldx, w, ldw, act, dx != nullptr, dw != nullptr, db != nullptr, M, N, K);
  if (p.total && (!ws || !aligned16(ws) || ws_bytes < p.total)) return crnn_set_error(hipErrorInvalidValue, "linear_bwd: workspace too small or unaligned");
  hipStream_t st = (hipStream_t)stream;
  if (act == CRNN_ACT_NONE) z = nullptr;
  return dtype == CRNN_BF16 ? bwd_t<bf16>(p, dy, lddy, x, ldx, w, ldw, z, ldz, act, dx, lddx, dw, dw_f32, db, db_f32, accumulate, (char*)ws, M, N, K, st)
                            : bwd_t<float>(p, dy, lddy, x, ldx, w, ldw, z, ldz, act, dx, lddx, dw, dw_f32, db, db_f32, accumulate, (char*)ws, M, N, K, st);
}

}  // extern "C"
