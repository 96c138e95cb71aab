// Layer norm over the last axis, forward and backward (the pre-norms of the gated-linear-recurrence encoder layer,
// crnn_hip/glr.py; crnn_hip.layer_norm).
//
//   y = xhat w + b,  xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - mean(g) - xhat mean(g xhat)),  g = dy w;   dw = sum_m dy xhat,  db = sum_m dy
//
// Both passes are bound by memory: the forward reads x and writes y, the backward reads x, dy and writes dx. A row lives
// in registers (8 consecutive elements per lane and chunk), so each is read once: WPR waves own a row of up to
// WPR * 64 * 8 * KC columns, and narrow rows share a wave, LPR lanes each. Rows wider than the widest such tile loop over
// memory (the *_wide kernels).
// The weight gradients sum over rows: a wave keeps its columns' sums in registers over all the rows it walks, the
// workgroup joins its waves in LDS and writes one partial row, and ln_colsum adds the partial rows in a fixed order.
#include <type_traits>
#include "common.hpp"
#include "crnn_internal.hpp"

namespace {

template <typename T> __device__ __forceinline__ void ldrow8(const T* row, int c, int n, float* f) {
  unpack8<T>(ld8_row<T>(row, c, n), f);
}
template <typename T> __device__ __forceinline__ void strow8(T* row, int c, int n, const float* f) {
  if (c + 8 <= n) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<bf16x8_u*>(row + c) = pack8<bf16>(f);
    } else {
      *reinterpret_cast<f32x4_u*>(row + c) = f32x4{f[0], f[1], f[2], f[3]};
      *reinterpret_cast<f32x4_u*>(row + c + 4) = f32x4{f[4], f[5], f[6], f[7]};
    }
  } else if (c < n) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (c + i < n) row[c + i] = fromf<T>(f[i]);
  }
}

// sum of a and of b over aligned groups of LPR lanes (every lane gets both)
template <int LPR = 64> __device__ __forceinline__ void wave_sum2(float& a, float& b) {
  a = rowgroup_sum<LPR < 16 ? LPR : 16>(a);
  b = rowgroup_sum<LPR < 16 ? LPR : 16>(b);
  if constexpr (LPR >= 32) {
    a += __shfl_xor(a, 16, 64);
    b += __shfl_xor(b, 16, 64);
  }
  if constexpr (LPR >= 64) {
    a += __shfl_xor(a, 32, 64);
    b += __shfl_xor(b, 32, 64);
  }
}
// ... over the WPR waves of a row; red: 2 * WPR floats of LDS, two sets used in turn (`set`), so that one barrier per sum is
// enough
template <int WPR, int LPR> __device__ __forceinline__ void row_sum2(float& a, float& b, float (*red)[2 * WPR], int set, int wid) {
  static_assert(WPR == 1 || LPR == 64, "whole waves");
  wave_sum2<LPR>(a, b);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) {
      red[set][2 * wid] = a;
      red[set][2 * wid + 1] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) {
      a += red[set][2 * w];
      b += red[set][2 * w + 1];
    }
  }
}

// mean and rstd of the row in x (KC chunks of 8 per lane): the plain mean first, then the deviations from it, whose own
// sum corrects the mean's rounding (a row far off centre keeps its variance)
template <int WPR, int KC, int LPR>
__device__ __forceinline__ void row_stats(const float (*x)[8], const int* c, int N, float eps, float (*red)[2 * WPR],
                                          int wid, float& mean, float& rstd) {
  const float inv = 1.f / (float)N;
  float s = 0.f, z = 0.f;
#pragma unroll
  for (int k = 0; k < KC; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[k][i];   // 0 past the end
  row_sum2<WPR, LPR>(s, z, red, 0, wid);
  const float m0 = s * inv;
  float d = 0.f, q = 0.f;
#pragma unroll
  for (int k = 0; k < KC; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = c[k] + i < N ? x[k][i] - m0 : 0.f;
      d += e;
      q += e * e;
    }
  row_sum2<WPR, LPR>(d, q, red, 1, wid);
  d *= inv;
  mean = m0 + d;
  rstd = 1.f / sqrtf(fmaxf(q * inv - d * d, 0.f) + eps);
}

// rows per workgroup pass: 4 waves of 64 / LPR rows (WPR = 1), or one row on all WPR waves
template <int WPR> constexpr int ln_threads() { return WPR == 1 ? 256 : WPR * 64; }
template <int WPR, int LPR> constexpr int ln_rpb() { return WPR == 1 ? 4 * (64 / LPR) : 1; }

template <typename T, int WPR, int KC, int LPR>
__global__ __launch_bounds__(ln_threads<WPR>()) void ln_fwd_kernel(const T* __restrict__ x, long ldx, const float* __restrict__ w,
                                                                   const float* __restrict__ b, T* __restrict__ y, long ldy,
                                                                   float* __restrict__ mean, float* __restrict__ rstd, long M,
                                                                   int N, float eps) {
  __shared__ float red[2][2 * WPR];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wr = WPR == 1 ? 0 : wid;
  const int lr = lane % LPR, sub = lane / LPR;   // lane of its row, row of the wave
  int c[KC];
  float wv[KC][8], bv[KC][8];
#pragma unroll
  for (int k = 0; k < KC; ++k) {
    c[k] = ((k * WPR + wr) * LPR + lr) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wv[k][i] = 1.f;
      bv[k][i] = 0.f;
    }
    if (w) ldrow8<float>(w, c[k], N, wv[k]);
    if (b) ldrow8<float>(b, c[k], N, bv[k]);
  }
  constexpr long RPB = ln_rpb<WPR, LPR>();
  for (long mb = (long)blockIdx.x * RPB + (WPR == 1 ? wid * (64 / LPR) : 0); mb < M; mb += (long)gridDim.x * RPB) {
    const long m = mb + sub;
    const int n = LPR == 64 || m < M ? N : 0;   // columns of this lane's row: none past the last one
    float v[KC][8];
#pragma unroll
    for (int k = 0; k < KC; ++k) ldrow8<T>(x + m * ldx, c[k], n, v[k]);
    float mu, rs;
    row_stats<WPR, KC, LPR>(v, c, N, eps, red, wr, mu, rs);
    if (mean && lr == 0 && wr == 0 && (LPR == 64 || n)) {
      mean[m] = mu;
      rstd[m] = rs;
    }
#pragma unroll
    for (int k = 0; k < KC; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = (v[k][i] - mu) * rs * wv[k][i] + bv[k][i];
      strow8<T>(y + m * ldy, c[k], n, v[k]);
    }
  }
}

template <typename T, int WPR, int KC, int LPR>
__global__ __launch_bounds__(ln_threads<WPR>(), WPR == 1 ? 3 : 1) void ln_bwd_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ x,
                                                                   long ldx, const float* __restrict__ w,
                                                                   const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                   const T* dres, long ldr, T* dx, long lddx,
                                                                   float* __restrict__ part, long M, int N) {
  constexpr int NV = ln_threads<WPR>() / LPR;   // row lanes of the workgroup
  constexpr int COLS = WPR * KC * LPR * 8;
  __shared__ float red[2][2 * WPR];
  __shared__ __attribute__((aligned(16))) float join[WPR == 1 ? NV * COLS : 4];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wr = WPR == 1 ? 0 : wid;
  const float inv = 1.f / (float)N;
  const int lr = lane % LPR, sub = lane / LPR;
  int c[KC];
  float wv[KC][8], sw[KC][8], sb[KC][8];
#pragma unroll
  for (int k = 0; k < KC; ++k) {
    c[k] = ((k * WPR + wr) * LPR + lr) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wv[k][i] = 1.f;
      sw[k][i] = sb[k][i] = 0.f;
    }
    if (w) ldrow8<float>(w, c[k], N, wv[k]);
  }
  int set = 0;
  constexpr long RPB = ln_rpb<WPR, LPR>();
  const long step = (long)gridDim.x * RPB;
  long mb = (long)blockIdx.x * RPB + (WPR == 1 ? wid * (64 / LPR) : 0);
  typename VT<T>::v8 xr[KC], gr[KC];   // the next row, on its way while this one is worked on
  auto fetch = [&](long m) {
    const int n = LPR == 64 || m < M ? N : 0;
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      xr[k] = ld8_row<T>(x + m * ldx, c[k], n);
      gr[k] = ld8_row<T>(dy + m * lddy, c[k], n);
    }
  };
  if (mb < M) fetch(mb + sub);
  for (; mb < M; mb += step) {
    const long m = mb + sub;
    const int n = LPR == 64 || m < M ? N : 0;   // columns of this lane's row: none past the last one
    const bool live = LPR == 64 || n;
    const float mu = live ? mean[m] : 0.f, rs = live ? rstd[m] : 0.f;
    float xh[KC][8], g[KC][8];
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      unpack8<T>(xr[k], xh[k]);
      unpack8<T>(gr[k], g[k]);
    }
    if (mb + step < M) fetch(m + step);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < KC; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        xh[k][i] = (xh[k][i] - mu) * rs;   // past the end g is 0, so xhat's value there enters no sum
        sb[k][i] += g[k][i];
        sw[k][i] += g[k][i] * xh[k][i];
        g[k][i] *= wv[k][i];
        s1 += g[k][i];
        s2 += g[k][i] * xh[k][i];
      }
    row_sum2<WPR, LPR>(s1, s2, red, set, wr);
    set ^= 1;
    s1 *= inv;
    s2 *= inv;
    if (dx) {
#pragma unroll
      for (int k = 0; k < KC; ++k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[k][i] = rs * (g[k][i] - s1 - xh[k][i] * s2);
        if (dres) {
          float r[8];
          ldrow8<T>(dres + m * ldr, c[k], n, r);
#pragma unroll
          for (int i = 0; i < 8; ++i) g[k][i] += r[i];
        }
        strow8<T>(dx + m * lddx, c[k], n, g[k]);
      }
    }
  }
  if (!part) return;
  float* pw = part + (size_t)blockIdx.x * 2 * N;   // [grid][2][N]: dw, then db
  if constexpr (WPR > 1) {
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      strow8<float>(pw, c[k], N, sw[k]);
      strow8<float>(pw + N, c[k], N, sb[k]);
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {   // dw, then db through the same LDS
      if (h) __syncthreads();
#pragma unroll
      for (int k = 0; k < KC; ++k)
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float* s = h ? sb[k] : sw[k];
          *reinterpret_cast<f32x4*>(join + (wid * (64 / LPR) + sub) * COLS + c[k] + i) =
              f32x4{s[i], s[i + 1], s[i + 2], s[i + 3]};
        }
      __syncthreads();
      for (int n = threadIdx.x; n < N; n += ln_threads<WPR>()) {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) s += join[v * COLS + n];
        pw[(size_t)h * N + n] = s;
      }
    }
  }
}

constexpr int kGridX = 1 << 20;   // most workgroups along the columns: 2^30 threads of the widest (a grid ends below 2^32)

// out_w[n], out_b[n] (+)= the sum of G partial rows [G][2][N]: 64 columns of the 2N per workgroup, 16 row lanes, fixed order
__global__ __launch_bounds__(1024) void ln_colsum_kernel(const float* __restrict__ part, int G, int N, float* __restrict__ dw,
                                                         float* __restrict__ db, int accumulate) {
  __shared__ float red[16][64];
  const int col = threadIdx.x & 63, rl = threadIdx.x >> 6;
  const long W = 2L * N;
  for (long j0 = (long)blockIdx.x * 64; j0 < W; j0 += (long)gridDim.x * 64) {
    const long j = j0 + col;
    float s = 0.f;
    if (j < W) {
      const float* p = part + j;
      int g = rl;
      for (; g + 7 * 16 < G; g += 8 * 16) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = p[(size_t)(g + 16 * u) * W];
#pragma unroll
        for (int u = 0; u < 8; ++u) s += v[u];
      }
      for (; g < G; g += 16) s += p[(size_t)g * W];
    }
    red[rl][col] = s;
    __syncthreads();
    if (rl == 0 && j < W) {
#pragma unroll
      for (int r = 1; r < 16; ++r) s += red[r][col];
      float* o = j < N ? dw : db;
      if (o) {
        const long n = j < N ? j : j - N;
        o[n] = accumulate ? o[n] + s : s;
      }
    }
    __syncthreads();   // red is the next columns'
  }
}

// ---- rows wider than the widest register tile: one workgroup per row, the row read again from L2
constexpr int LW = 1024;
__device__ __forceinline__ void block_sum2(float& a, float& b, float (*red)[32], int set) {
  wave_sum2(a, b);
  const int wid = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    red[set][2 * wid] = a;
    red[set][2 * wid + 1] = b;
  }
  __syncthreads();
  a = b = 0.f;
#pragma unroll
  for (int w = 0; w < LW / 64; ++w) {
    a += red[set][2 * w];
    b += red[set][2 * w + 1];
  }
}

// f(n, p, q) adds column n's terms of two sums; 64 columns of a lane at a time, so that the longest rows (2^30) add 2^14 sums of 64
// terms instead of 2^20 terms one by one
template <class F> __device__ __forceinline__ void wide_sum2(int N, float& a, float& b, F f) {
  a = b = 0.f;
  for (int n0 = threadIdx.x; n0 < N; n0 += 64 * LW) {
    float p = 0.f, q = 0.f;
    const int end = min(N, n0 + 64 * LW);
    for (int n = n0; n < end; n += LW) f(n, p, q);
    a += p;
    b += q;
  }
}

template <typename T>
__global__ __launch_bounds__(LW) void ln_fwd_wide_kernel(const T* __restrict__ x, long ldx, const float* __restrict__ w,
                                                         const float* __restrict__ b, T* __restrict__ y, long ldy,
                                                         float* __restrict__ mean, float* __restrict__ rstd, long M, int N,
                                                         float eps) {
  __shared__ float red[2][32];
  const float inv = 1.f / (float)N;
  for (long m = blockIdx.x; m < M; m += gridDim.x) {
    const T* row = x + m * ldx;
    float s, z;
    wide_sum2(N, s, z, [&](int n, float& p, float&) { p += tof(row[n]); });
    block_sum2(s, z, red, 0);
    const float m0 = s * inv;
    float d, q;
    wide_sum2(N, d, q, [&](int n, float& p, float& r) {
      const float e = tof(row[n]) - m0;
      p += e;
      r += e * e;
    });
    block_sum2(d, q, red, 1);
    d *= inv;
    const float mu = m0 + d, rs = 1.f / sqrtf(fmaxf(q * inv - d * d, 0.f) + eps);
    if (mean && threadIdx.x == 0) {
      mean[m] = mu;
      rstd[m] = rs;
    }
    for (int n = threadIdx.x; n < N; n += LW)
      y[m * ldy + n] = fromf<T>((tof(row[n]) - mu) * rs * (w ? w[n] : 1.f) + (b ? b[n] : 0.f));
  }
}

template <typename T>
__global__ __launch_bounds__(LW) void ln_bwd_wide_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                                                         const float* __restrict__ w, const float* __restrict__ mean,
                                                         const float* __restrict__ rstd, const T* dres, long ldr, T* dx,
                                                         long lddx, long M, int N) {
  __shared__ float red[2][32];
  const float inv = 1.f / (float)N;
  int set = 0;
  for (long m = blockIdx.x; m < M; m += gridDim.x) {
    const float mu = mean[m], rs = rstd[m];
    float s1, s2;
    wide_sum2(N, s1, s2, [&](int n, float& p, float& q) {
      const float g = tof(dy[m * lddy + n]) * (w ? w[n] : 1.f);
      p += g;
      q += g * (tof(x[m * ldx + n]) - mu) * rs;
    });
    block_sum2(s1, s2, red, set);
    set ^= 1;
    s1 *= inv;
    s2 *= inv;
    for (int n = threadIdx.x; n < N; n += LW) {
      const float g = tof(dy[m * lddy + n]) * (w ? w[n] : 1.f);
      float v = rs * (g - s1 - (tof(x[m * ldx + n]) - mu) * rs * s2);
      if (dres) v += tof(dres[m * ldr + n]);
      dx[m * lddx + n] = fromf<T>(v);
    }
  }
}

// partial rows of the weight gradients for the wide rows: workgroup (64 columns, row slice)
template <typename T>
__global__ __launch_bounds__(256) void ln_wgrad_wide_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                                                            const float* __restrict__ mean, const float* __restrict__ rstd,
                                                            float* __restrict__ part, long M, int N, int G) {
  __shared__ float red[2][4][64];
  const int col = threadIdx.x & 63, rl = threadIdx.x >> 6, g = blockIdx.y;
  for (long n0 = (long)blockIdx.x * 64; n0 < N; n0 += (long)gridDim.x * 64) {
    const long n = n0 + col;
    float sw = 0.f, sb = 0.f;
    if (n < N)
      for (long m = (long)g * 4 + rl; m < M; m += 4L * G) {
        const float d = tof(dy[m * lddy + n]);
        sb += d;
        sw += d * (tof(x[m * ldx + n]) - mean[m]) * rstd[m];
      }
    red[0][rl][col] = sw;
    red[1][rl][col] = sb;
    __syncthreads();
    if (rl == 0 && n < N) {
#pragma unroll
      for (int r = 1; r < 4; ++r) {
        sw += red[0][r][col];
        sb += red[1][r][col];
      }
      part[(size_t)g * 2 * N + n] = sw;
      part[(size_t)g * 2 * N + N + n] = sb;
    }
    __syncthreads();   // red is the next columns'
  }
}

// the register tile of a width: (waves per row, chunks of 8 per lane, lanes of a wave per row); {0, 0, 0}: the wide kernels.
// Rows of up to 256 columns share a wave, since a wave's latency is what a short row costs; forward / backward in us with a wave
// per row and with the lanes below: 65536 x 64 bf16 18.4 / 25.9 and 5.5 / 10.3, x 128 19.4 / 30.9 and 8.0 / 15.6, x 256
// 19.4 / 31.8 and 12.5 / 22.8, x 19 fp32 20.2 / 39.0 and 6.4 / 12.5
struct LnPlan { int wpr, kc, lpr; };
LnPlan ln_plan(int N) {
  if (N <= 64) return {1, 1, 8};
  if (N <= 128) return {1, 1, 16};
  if (N <= 256) return {1, 1, 32};
  if (N <= 512) return {1, 1, 64};
  if (N <= 1024) return {1, 2, 64};
  if (N <= 2048) return {4, 1, 64};
  if (N <= 4096) return {4, 2, 64};
  if (N <= 8192) return {16, 1, 64};
  if (N <= 16384) return {16, 2, 64};
  return {0, 0, 0};
}
// f(integral_constant wpr, kc, lpr) for a plan with a register tile
template <class F> int ln_dispatch(const LnPlan& p, F&& f) {
#define LN_CASE(W, K, L)                    \
  if (p.wpr == W && p.kc == K && p.lpr == L) \
  return f(std::integral_constant<int, W>{}, std::integral_constant<int, K>{}, std::integral_constant<int, L>{})
  LN_CASE(1, 1, 8);
  LN_CASE(1, 1, 16);
  LN_CASE(1, 1, 32);
  LN_CASE(1, 1, 64);
  LN_CASE(1, 2, 64);
  LN_CASE(4, 1, 64);
  LN_CASE(4, 2, 64);
  LN_CASE(16, 1, 64);
  LN_CASE(16, 2, 64);
#undef LN_CASE
  return (int)hipErrorInvalidValue;
}

constexpr int kMaxN = 1 << 30;   // column counters are 32 bits

// workgroups of the backward: enough rows in flight, few partial rows to add up, and two rows a wave or more so that the
// next one's loads run under this one's sums (65536 x 768 bf16, backward: 85 us at 2 workgroups per CU, 66 at 3, 88 at 4;
// 32768 x 1536, 4 waves a row and fewer registers: 91, 67, 62; 1999 x 1021 fp32: 14.8 at one row a wave, 13.4 at two, 15.9 at
// four)
int ln_bwd_grid(long M, int N) {
  const LnPlan p = ln_plan(N);
  const long rows = p.wpr == 1 ? 8 * (64 / p.lpr) : 2, want = (M + rows - 1) / rows;
  const long cap = (p.wpr == 4 && p.kc == 1 ? 4L : 3L) * crnn_cu_count();
  return (int)(want < 1 ? 1 : want < cap ? want : cap);
}
int ln_wide_slices(long M) {
  const long s = (M + 63) / 64;
  return (int)(s < 1 ? 1 : s < 64 ? s : 64);
}

template <typename T>
int ln_fwd_t(const void* x, long ldx, const float* w, const float* b, void* y, long ldy, float* mean, float* rstd, long M, int N,
             float eps, hipStream_t st) {
  const LnPlan p = ln_plan(N);
  if (p.wpr)
    return ln_dispatch(p, [&](auto W, auto K, auto L) {
      constexpr int wpr = decltype(W)::value, kc = decltype(K)::value, lpr = decltype(L)::value, rpb = ln_rpb<wpr, lpr>();
      const long g = (M + rpb - 1) / rpb, cap = 8L * crnn_cu_count();
      hipLaunchKernelGGL((ln_fwd_kernel<T, wpr, kc, lpr>), dim3((int)(g < cap ? g : cap)), dim3(ln_threads<wpr>()), 0, st, (const T*)x,
                         ldx, w, b, (T*)y, ldy, mean, rstd, M, N, eps);
      return (int)hipGetLastError();
    });
  const long cap = 2L * crnn_cu_count();
  hipLaunchKernelGGL(ln_fwd_wide_kernel<T>, dim3((int)(M < cap ? M : cap)), dim3(LW), 0, st, (const T*)x, ldx, w, b, (T*)y, ldy,
                     mean, rstd, M, N, eps);
  return (int)hipGetLastError();
}

template <typename T>
int ln_bwd_t(const void* dy, long lddy, const void* x, long ldx, const float* w, const float* mean, const float* rstd,
             const void* dres, long ldr, void* dx, long lddx, float* dw, float* db, int accumulate, float* ws, long M, int N,
             hipStream_t st) {
  const LnPlan p = ln_plan(N);
  float* part = dw || db ? ws : nullptr;
  int rc = 0, G = 0;
  if (M > 0 && p.wpr) {
    G = ln_bwd_grid(M, N);
    rc = ln_dispatch(p, [&](auto W, auto K, auto L) {
      constexpr int wpr = decltype(W)::value, kc = decltype(K)::value, lpr = decltype(L)::value;
      hipLaunchKernelGGL((ln_bwd_kernel<T, wpr, kc, lpr>), dim3(G), dim3(ln_threads<wpr>()), 0, st, (const T*)dy, lddy, (const T*)x,
                         ldx, w, mean, rstd, (const T*)dres, ldr, (T*)dx, lddx, part, M, N);
      return (int)hipGetLastError();
    });
  } else if (M > 0) {
    if (part) {   // before dx: dx may be dres, and neither dy nor x may be dx, so the order is free; kept first
      G = ln_wide_slices(M);
      hipLaunchKernelGGL(ln_wgrad_wide_kernel<T>, dim3(grid_for(N, 64, kGridX), G), dim3(256), 0, st, (const T*)dy, lddy, (const T*)x,
                         ldx, mean, rstd, part, M, N, G);
      rc = (int)hipGetLastError();
    }
    if (!rc && dx) {
      const long cap = 2L * crnn_cu_count();
      hipLaunchKernelGGL(ln_bwd_wide_kernel<T>, dim3((int)(M < cap ? M : cap)), dim3(LW), 0, st, (const T*)dy, lddy, (const T*)x,
                         ldx, w, mean, rstd, (const T*)dres, ldr, (T*)dx, lddx, M, N);
      rc = (int)hipGetLastError();
    }
  }
  if (rc || !part) return rc;
  hipLaunchKernelGGL(ln_colsum_kernel, dim3(grid_for(2L * N, 64, kGridX)), dim3(1024), 0, st, part, G, N, dw, db, accumulate);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

int crnn_layernorm_fwd(int dtype, const void* x, long ldx, const float* w, const float* b, void* y, long ldy, float* mean,
                       float* rstd, long M, int N, float eps, void* stream) {
  if (dtype != CRNN_F32 && dtype != CRNN_BF16) return crnn_set_error(hipErrorInvalidValue, "layernorm_fwd: dtype fp32 or bf16");
  if (M < 0 || N < 1 || N > kMaxN || ldx < N || ldy < N)
    return crnn_set_error(hipErrorInvalidValue, "layernorm_fwd: M >= 0, 1 <= N <= 2^30, ld >= N");
  if ((mean == nullptr) != (rstd == nullptr)) return crnn_set_error(hipErrorInvalidValue, "layernorm_fwd: mean and rstd go together");
  if (M == 0) return 0;
  if (!x || !y) return crnn_set_error(hipErrorInvalidValue, "layernorm_fwd: null x / y");
  hipStream_t st = (hipStream_t)stream;
  return dtype == CRNN_BF16 ? ln_fwd_t<bf16>(x, ldx, w, b, y, ldy, mean, rstd, M, N, eps, st)
                            : ln_fwd_t<float>(x, ldx, w, b, y, ldy, mean, rstd, M, N, eps, st);
}

size_t crnn_layernorm_bwd_workspace(int dtype, long M, int N) {
  (void)dtype;
  if (M < 0 || N < 1 || N > kMaxN) return 0;
  const size_t g = ln_plan(N).wpr ? (size_t)ln_bwd_grid(M, N) : (size_t)ln_wide_slices(M);
  return g * 2 * (size_t)N * sizeof(float);
}

int crnn_layernorm_bwd(int dtype, const void* dy, long lddy, const void* x, long ldx, const float* w, const float* mean,
                       const float* rstd, const void* dres, long ldr, void* dx, long lddx, float* dw, float* db,
                       int accumulate, float* ws, size_t ws_bytes, long M, int N, void* stream) {
  if (dtype != CRNN_F32 && dtype != CRNN_BF16) return crnn_set_error(hipErrorInvalidValue, "layernorm_bwd: dtype fp32 or bf16");
  if (M < 0 || N < 1 || N > kMaxN || lddy < N || ldx < N || (dx && lddx < N) || (dres && ldr < N))
    return crnn_set_error(hipErrorInvalidValue, "layernorm_bwd: M >= 0, 1 <= N <= 2^30, ld >= N");
  if (dx && dx == dres && lddx != ldr)   // a row of dx would be written over another row's dres before that is read
    return crnn_set_error(hipErrorInvalidValue, "layernorm_bwd: dx over dres needs the same row stride");
  if (M > 0 && (!dy || !x || !mean || !rstd)) return crnn_set_error(hipErrorInvalidValue, "layernorm_bwd: null dy / x / mean / rstd");
  if ((dw || db) && (!ws || ws_bytes < crnn_layernorm_bwd_workspace(dtype, M, N)))
    return crnn_set_error(hipErrorInvalidValue, "layernorm_bwd: workspace too small");
  if (M == 0 && !dw && !db) return 0;
  hipStream_t st = (hipStream_t)stream;
  return dtype == CRNN_BF16
             ? ln_bwd_t<bf16>(dy, lddy, x, ldx, w, mean, rstd, dres, ldr, dx, lddx, dw, db, accumulate, ws, M, N, st)
             : ln_bwd_t<float>(dy, lddy, x, ldx, w, mean, rstd, dres, ldr, dx, lddx, dw, db, accumulate, ws, M, N, st);
}

}  // extern "C"
