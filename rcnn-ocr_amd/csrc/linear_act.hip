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

// ---------------------------------------------------------------- activations
// Phi(-|z|) = erfc(|z| / sqrt 2) / 2. For bf16 results erfc(x) = t P(t) e^{-x^2}, t = 1 / (1 + 0.435 x), P the degree-5
// polynomial of least relative error over 0 <= x <= 9.4 (3.7e-6, fitted by reweighted least squares; half a bf16 step is
// 3.9e-3): 15 instructions where erfcf takes several times that, and the epilogue runs them for every output.
__device__ __forceinline__ float gauss_tail(float z, float& e) {
  const float x = 0.70710678f * fabsf(z);
  const float t = __builtin_amdgcn_rcpf(1.f + 0.435f * x);
  e = __expf(-x * x);
  float p = -0.15173584f;
  p = p * t + 0.38380495f;
  p = p * t + 0.010128383f;
  p = p * t + 0.27484620f;
  p = p * t + 0.23699674f;
  p = p * t + 0.24595593f;
  return 0.5f * p * t * e;
}
template <typename T, int ACT> __device__ __forceinline__ float act(float z) {
  if constexpr (ACT == CRNN_ACT_RELU) return z > 0.f ? z : (z == z ? 0.f : z);
  if constexpr (ACT == CRNN_ACT_GELU) {
    if constexpr (sizeof(T) == 2) {
      float e;
      const float q = gauss_tail(z, e);
      return z * (z < 0.f ? q : 1.f - q);
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
      return (z < 0.f ? q : 1.f - q) + z * e * kC;
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
template <typename T, int ACT, bool ROW8 = false> struct ActEpi {
  static constexpr bool kStats = false;
  static constexpr bool kRow8 = ROW8;   // 8 columns per lane through the wave's LDS (gemm256.hpp row8_epilogue)
  T *y, *z;
  const T* res;
  const void* bias;
  long ldy, ldz, ldr;
  int M, N, bias_f32;
  int vec;   // y, z, res rows aligned for 4-column vectors (8-column ones with ROW8)
  __device__ __forceinline__ float b(int n) const { return bias_f32 ? ((const float*)bias)[n] : tof(((const T*)bias)[n]); }
  __device__ __forceinline__ f32x4 b4(int n) const { return bias_f32 ? ld4f<float>((const float*)bias + n) : ld4f<T>((const T*)bias + n); }
  __device__ __forceinline__ void store(int m, int n, f32x4 v, int) const {
    if (m >= M || n >= N) return;
    if (vec && n + 4 <= N) {
      if (bias) v += b4(n);
      if (z) st4<T>(z + m * ldz + n, v);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = act<T, ACT>(v[r]);
      if (res) v += ld4f<T>(res + m * ldr + n);
      st4<T>(y + m * ldy + n, v);
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
  __device__ __forceinline__ void store8(int m, int n, f32x4 lo, f32x4 hi, int kz) const {
    if constexpr (sizeof(T) == 2) {
      if (vec && n + 8 <= N) {
        if (m >= M) return;
        float u[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          u[r] = lo[r];
          u[4 + r] = hi[r];
        }
        if (bias) {
          const f32x4 b0 = b4(n), b1 = b4(n + 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            u[r] += b0[r];
            u[4 + r] += b1[r];
          }
        }
        if (z) st8<T>(z + m * ldz + n, pack8<T>(u));
#pragma unroll
        for (int r = 0; r < 8; ++r) u[r] = act<T, ACT>(u[r]);
        if (res) {
          float q[8];
          unpack8<T>(ld8<T>(res + m * ldr + n), q);
#pragma unroll
          for (int r = 0; r < 8; ++r) u[r] += q[r];
        }
        st8<T>(y + m * ldy + n, pack8<T>(u));
        return;
      }
    }
    store(m, n, lo, kz);
    store(m, n + 4, hi, kz);
  }
  __device__ __forceinline__ void stats(int, int, f32x4, f32x4) const {}
};

// ---------------------------------------------------------------- operands
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int round8i(int n) { return (n + 7) & ~7; }
// the MFMA loaders read 16-byte vectors of 8 elements (fp32: two of 4): the base, the row pitch and the row length have to
// be whole vectors
bool direct(const void* p, long ld, int cols, int es) {
  return aligned16(p) && ld * es % 16 == 0 && cols % 8 == 0 && ld < 0x7fffffffL;
}
// rows of one launch: the loaders address an operand with 32-bit byte offsets
long max_rows(long ld, int es) {
  const long r = 0x7fffffffL / (ld * es);
  return r >= 256 ? r / 256 * 256 : r;
}

// dst[rows][cols8] (zero behind cols) = src[rows][ld]
template <typename T>
__global__ __launch_bounds__(256) void pad_copy_kernel(const T* __restrict__ src, long ld, T* __restrict__ dst, long rows, int cols,
                                                       int cols8) {
  const long n8 = rows * (cols8 / 8);
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n8; i += gridDim.x * 256L) {
    const long r = i / (cols8 / 8);
    const int c = (int)(i - r * (cols8 / 8)) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? tof(src[r * ld + c + e]) : 0.f;
    st8<T>(dst + r * cols8 + c, pack8<T>(v));
  }
}
template <typename T> int pad_copy(const void* src, long ld, void* dst, long rows, int cols, hipStream_t st) {
  const long n8 = rows * (round8i(cols) / 8);
  if (n8 == 0) return 0;
  hipLaunchKernelGGL(pad_copy_kernel<T>, dim3(grid_for(n8)), dim3(256), 0, st, (const T*)src, ld, (T*)dst, rows, cols, round8i(cols));
  return (int)hipGetLastError();
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// ---------------------------------------------------------------- tile plans
// bf16: the deep 256-row kernels where their tiles alone fill three quarters of the CUs, else the register-staged ones;
// fp32 (exact-fp32 MFMA): register-staged
template <typename T, class LA, class LB, class E, class E8>
int tiles_run(const LA& la, const LB& lb, const E& ep, const E8& ep8, bool row8, int M, int N, int K, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    const long cu = crnn_cu_count();
    const long t256 = (long)((M + 255) / 256) * ((N + 255) / 256), t128 = (long)((M + 255) / 256) * ((N + 127) / 128);
    if (K >= 256) {
      if (N >= 256 && t256 * 4 >= cu * 3)
        return row8 ? launch256<256, 256>(la, lb, ep8, M, N, K, st) : launch256<256, 256>(la, lb, ep, M, N, K, st);
      if (N >= 128 && t128 * 4 >= cu * 3)
        return row8 ? launch256<256, 128>(la, lb, ep8, M, N, K, st) : launch256<256, 128>(la, lb, ep, M, N, K, st);
    }
  }
  const long work = (long)M * N;
  if (M >= 128 && N >= 128 && work >= 128L * 128 * 128) return launch<T, 128, 128>(la, lb, ep, M, N, K, 1, st);
  if (work >= 64L * 64 * 128) return launch<T, 64, 64>(la, lb, ep, M, N, K, 1, st);
  return launch<T, 32, 32>(la, lb, ep, M, N, K, 1, st);
}

template <typename T, int ACT>
int fwd_act(const T* x, long ldx, const T* w, long ldw, const void* bias, int bias_f32, const T* res, long ldr, T* y, long ldy, T* z,
            long ldz, long M, int N, int K8, hipStream_t st) {
  const long step = max_rows(ldx, sizeof(T));
  const long m16 = 16 / sizeof(T);   // elements of a 16-byte vector
  const bool al = aligned16(y) && ldy % m16 == 0 && (!z || (aligned16(z) && ldz % m16 == 0)) &&
                  (!res || (aligned16(res) && ldr % m16 == 0)) && (!bias || aligned16(bias));
  for (long m0 = 0; m0 < M; m0 += step) {
    const int m = (int)(M - m0 < step ? M - m0 : step);
    const RowMajorK<T> la{x + m0 * ldx, (int)ldx, m, K8};
    const RowMajorK<T> lb{w, (int)ldw, N, K8};
    const ActEpi<T, ACT> ep{y + m0 * ldy, z ? z + m0 * ldz : nullptr, res ? res + m0 * ldr : nullptr, bias, ldy, ldz, ldr, m, N,
                            bias_f32, al};
    const ActEpi<T, ACT, true> ep8{ep.y, ep.z, ep.res, bias, ldy, ldz, ldr, m, N, bias_f32, al};
    const int rc = tiles_run<T>(la, lb, ep, ep8, al, m, N, K8, st);
    if (rc) return rc;
  }
  return 0;
}

template <typename T>
int fwd_t(const void* x, long ldx, const void* w, long ldw, const void* bias, int bias_f32, int kind, const void* res, long ldr,
          void* y, long ldy, void* z, long ldz, char* ws, long M, int N, int K, hipStream_t st) {
  const int K8 = round8i(K);
  const T *xp = (const T*)x, *wp = (const T*)w;
  if (!direct(x, ldx, K, sizeof(T))) {
    const int rc = pad_copy<T>(x, ldx, ws, M, K, st);
    if (rc) return rc;
    xp = (const T*)ws;
    ldx = K8;
    ws += up256((size_t)M * K8 * sizeof(T));
  }
  if (!direct(w, ldw, K, sizeof(T))) {
    const int rc = pad_copy<T>(w, ldw, ws, N, K, st);
    if (rc) return rc;
    wp = (const T*)ws;
    ldw = K8;
  }
#define FWD(A) fwd_act<T, A>(xp, ldx, wp, ldw, bias, bias_f32, (const T*)res, ldr, (T*)y, ldy, (T*)z, ldz, M, N, K8, st)
  if (kind == CRNN_ACT_RELU) return FWD(CRNN_ACT_RELU);
  if (kind == CRNN_ACT_GELU) return FWD(CRNN_ACT_GELU);
  if (kind == CRNN_ACT_SILU) return FWD(CRNN_ACT_SILU);
  return FWD(CRNN_ACT_NONE);
#undef FWD
}

// ---------------------------------------------------------------- backward
// dz = dy act'(z) into dz [M][N8] (zero behind N; NULL: only the sums), and the partial column sums part[g][N] of row slice
// g (NULL: none). A thread owns 8 columns; the 8 row lanes of a workgroup join in LDS. fp32 throughout, dz rounded once to
// the operands' type for the products; the column sums add the unrounded values.
template <typename T>
__global__ __launch_bounds__(256) void dz_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ z, long ldz, int kind,
                                                 T* __restrict__ dz, int N8, float* __restrict__ part, long M, int N) {
  __shared__ float red[8][32 * 8 + 8];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int n = (blockIdx.x * 32 + cl) * 8;
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = 0.f;
  if (n < N8)
    for (long m = (long)blockIdx.y * 8 + rl; m < M; m += 8L * gridDim.y) {
      float g[8], q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[e] = n + e < N ? tof(dy[m * lddy + n + e]) : 0.f;
        q[e] = z && n + e < N ? tof(z[m * ldz + n + e]) : 0.f;
      }
      if (z)
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] *= dact<T>(kind, q[e]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += g[e];
      if (dz) st8<T>(dz + m * N8 + n, pack8<T>(g));
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

// out[n] (+)= sum_g part[g][n]: 64 columns per workgroup, 16 row lanes, fixed order
template <typename O>
__global__ __launch_bounds__(1024) void db_reduce_kernel(const float* __restrict__ part, int G, int N, O* __restrict__ out, int accumulate) {
  __shared__ float red[16][64];
  const int col = threadIdx.x & 63, rl = threadIdx.x >> 6, n = blockIdx.x * 64 + col;
  float s = 0.f;
  if (n < N) {
    int g = rl;
    for (; g + 7 * 16 < G; g += 8 * 16) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = part[(size_t)(g + 16 * u) * N + n];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
    for (; g < G; g += 16) s += part[(size_t)g * N + n];
  }
  red[rl][col] = s;
  __syncthreads();
  if (rl == 0 && n < N) {
#pragma unroll
    for (int r = 1; r < 16; ++r) s += red[r][col];
    put<O>(out + n, s, accumulate);
  }
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
template <typename O>
__global__ __launch_bounds__(256) void dw_reduce_kernel(const float* __restrict__ ws, int S, int Nr, int Kc, O* __restrict__ dw, int N,
                                                        int K, int accumulate) {
  const long total = (long)Nr * Kc;
  for (long i4 = blockIdx.x * 256L + threadIdx.x; 4 * i4 < total; i4 += gridDim.x * 256L) {
    const long i = 4 * i4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    int z = 0;
    for (; z + 8 <= S; z += 8) {
      f32x4 v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = *reinterpret_cast<const f32x4*>(ws + (size_t)(z + q) * total + i);
#pragma unroll
      for (int q = 0; q < 8; ++q) s += v[q];
    }
    for (; z < S; ++z) s += *reinterpret_cast<const f32x4*>(ws + (size_t)z * total + i);
    const int n = (int)(i / Kc), k = (int)(i - (long)n * Kc);   // Kc % 8 == 0: the four share a row
    if (n >= N) continue;
    O* o = dw + (size_t)n * K + k;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + e < K) put<O>(o + e, s[e], accumulate);
  }
}

// row slices of the column sums: enough workgroups for the chip, few partial rows
int dz_slices(long M, int N) {
  const long cb = (round8i(N) + 255) / 256;
  long g = (2L * crnn_cu_count() + cb - 1) / cb;
  const long most = (M + 31) / 32;
  if (g > most) g = most;
  if (g > 256) g = 256;
  return (int)(g < 1 ? 1 : g);
}
// K splits of one launch of the weight gradient over `rows` rows
int dw_splits(int Nr, int Kc, long rows) {
  const long tiles = (long)((Nr + 127) / 128) * ((Kc + 127) / 128);
  long s = (crnn_cu_count() + tiles - 1) / tiles;
  const long smax = (rows + 16 * 64 - 1) / (16 * 64);
  if (s > smax) s = smax;
  if (s < 1) s = 1;
  return eff_splits((int)rows, (int)s);
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
  p.own_dz = (need_dx || need_dw) && (kind != CRNN_ACT_NONE || !direct(dy, lddy, N, es));
  p.copy_x = need_dw && !direct(x, ldx, K, es);
  p.copy_w = need_dx && !direct(w, ldw, K, es);
  p.slices = need_db ? dz_slices(M, N) : 0;
  const long ldz_ = p.own_dz ? p.N8 : lddy, ldx_ = p.copy_x ? p.K8 : ldx;
  if (need_dw && M > 0) {
    const long step = max_rows(ldz_ > ldx_ ? ldz_ : ldx_, es);
    for (long m0 = 0; m0 < M; m0 += step) p.slabs += dw_splits(p.N8, p.K8, M - m0 < step ? M - m0 : step);
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
  if (db) {
    const int G = M > 0 ? p.slices : 0;
    const dim3 grid((N + 63) / 64);
    if (db_f32) hipLaunchKernelGGL(db_reduce_kernel<float>, grid, dim3(1024), 0, st, part, G, N, (float*)db, accumulate);
    else hipLaunchKernelGGL(db_reduce_kernel<T>, grid, dim3(1024), 0, st, part, G, N, (T*)db, accumulate);
    if ((rc = (int)hipGetLastError())) return rc;
  }
  if (p.copy_x && M > 0) {
    if ((rc = pad_copy<T>(x, ldx, ws + p.o_x, M, K, st))) return rc;
    xp = (const T*)(ws + p.o_x);
    ldx = p.K8;
  }
  if (dx && M > 0) {
    if (p.copy_w) {
      if ((rc = pad_copy<T>(w, ldw, ws + p.o_w, N, K, st))) return rc;
      wp = (const T*)(ws + p.o_w);
      ldw = p.K8;
    }
    const long step = max_rows(ldd, sizeof(T));
    const bool al = aligned16(dx) && lddx * (long)sizeof(T) % 16 == 0;
    for (long m0 = 0; m0 < M; m0 += step) {
      const int m = (int)(M - m0 < step ? M - m0 : step);
      const RowMajorK<T> la{dzp + m0 * ldd, (int)ldd, m, p.N8};
      const ColMajorK<T> lb{wp, (int)ldw, p.K8, N};
      const ActEpi<T, CRNN_ACT_NONE> ep{(T*)dx + m0 * lddx, nullptr, nullptr, nullptr, lddx, 0, 0, m, K, 0, al};
      const ActEpi<T, CRNN_ACT_NONE, true> ep8{ep.y, nullptr, nullptr, nullptr, lddx, 0, 0, m, K, 0, al};
      if ((rc = tiles_run<T>(la, lb, ep, ep8, al, m, K, p.N8, st))) return rc;
    }
  }
  if (dw) {
    float* slab = (float*)(ws + p.o_slab);
    int s0 = 0;
    if (M > 0) {
      const long step = max_rows(ldd > ldx ? ldd : ldx, sizeof(T));
      for (long m0 = 0; m0 < M; m0 += step) {
        const int m = (int)(M - m0 < step ? M - m0 : step);
        const int S = dw_splits(p.N8, p.K8, m);
        const ColMajorK<T> la{dzp + m0 * ldd, (int)ldd, p.N8, m};
        const ColMajorK<T> lb{xp + m0 * ldx, (int)ldx, p.K8, m};
        const SlabEpi ep{slab + (size_t)s0 * p.N8 * p.K8, p.N8, p.K8};
        if ((rc = launch<T, 128, 128>(la, lb, ep, p.N8, p.K8, m, S, st))) return rc;
        s0 += S;
      }
    }
    const int blocks = grid_for((long)p.N8 * p.K8 / 4, 256, 2048);
    if (dw_f32) hipLaunchKernelGGL(dw_reduce_kernel<float>, dim3(blocks), dim3(256), 0, st, slab, s0, p.N8, p.K8, (float*)dw, N, K, accumulate);
    else hipLaunchKernelGGL(dw_reduce_kernel<T>, dim3(blocks), dim3(256), 0, st, slab, s0, p.N8, p.K8, (T*)dw, N, K, accumulate);
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
  size_t n = 0;
  if (!direct(x, ldx, K, es)) n += up256((size_t)M * round8i(K) * es);
  if (!direct(w, ldw, K, es)) n += up256((size_t)N * round8i(K) * es);
  return n;
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
