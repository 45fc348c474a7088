// Layer norm over the channels of a token, forward and backward (include/yk.h, yk_layer_norm).
//
//   y  = (x - mu) r w + b,  r = 1 / sqrt(mean((x - mu)^2) + eps)
//   dx = r (g - mean(g) - h mean(g h)),  g = dy w,  h = (x - mu) r
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// All of it is bound by HBM: 2 bytes-per-element streams forward, 3 backward.  A row is read once
// into registers by NT lanes (NV 16-byte chunks each) and the variance is the mean of (x - mu)^2
// over those registers, not a difference of moments, so a row's offset costs no digits.  Backward, a
// workgroup walks rows and keeps the column sums of dw / db in registers; they meet in LDS, go
// to scratch as one float32 row per workgroup, and a second kernel adds those rows in a fixed order
// (no atomics: equal calls give equal bits).
//
// 163840 x 640 bf16: forward 78 us, 5.4 TB/s, backward 122 us, 5.1 TB/s (what a large copy reaches here),
// and 4.6 for the rows of partial sums.  10001 x 1027 fp16, rows aligned to 2 bytes: 16 and 31 us.
// 320 x 320 float32: 3.4 us, a launch and one row's latency.
#include "token_common.h"

namespace yk {
namespace tok {

struct NormArgs {
  const char* x;
  const void* w;
  const void* b;
  char* y;
  float* mean;
  float* rstd;
  int64_t m, x_stride, y_stride;
  int c, param_f32, dtype;
  float eps;
};

struct NormGradArgs {
  const char* dy;
  const char* x;
  const void* w;
  const float* mean;
  const float* rstd;
  char* dx;
  float* part;  // [gridDim.x][2][c] column sums of dy h and dy, or NULL
  int64_t m, dy_stride, x_stride, dx_stride;
  int c, param_f32, dtype;
};

// v of the lane n places round the row of 16 lanes
template <int kN>
__device__ __forceinline__ float rotate16(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + kN, 0xf, 0xf, true));
}
// Sum over the NT lanes of a row, in every one of them: rotations within 16 lanes (vector speed),
// then across them, for more than a wave through one LDS word per wave.
template <int NT>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v += rotate16<8>(v);
  v += rotate16<4>(v);
  v += rotate16<2>(v);
  v += rotate16<1>(v);
  if constexpr (NT >= 64) {
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
  }
  if constexpr (NT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) v += red[i];
  }
  return v;
}

template <class Tr>
__device__ __forceinline__ float elem(const u32x4& u, int e) {
  if constexpr (Tr::kBytes == 4) {
    return __uint_as_float(u[e]);
  } else {
    const unsigned short h = (unsigned short)(u[e >> 1] >> ((e & 1) * 16));
    return to_f32<Tr>(__builtin_bit_cast(typename Tr::T, h));
  }
}

template <class Tr>
__device__ __forceinline__ void store16(typename Tr::T* p, const float* v, int n) {
  constexpr int kEpc = 16 / Tr::kBytes;
  typename Tr::T t[kEpc];
#pragma unroll
  for (int e = 0; e < kEpc; ++e) t[e] = from_f32<Tr>(v[e]);
  if (n >= kEpc) {
    u32x4 u;
    __builtin_memcpy(&u, t, 16);
    *(u32x4_any*)p = u;
  } else {
#pragma unroll
    for (int e = 0; e < kEpc; ++e)
      if (e < n) p[e] = t[e];
  }
}

// kEpc parameters from column c0 (those at or past c: `fill`)
template <class Tr>
__device__ __forceinline__ void params(const void* p, int c0, int c, int is_f32, int dtype, float fill, float* out) {
  constexpr int kEpc = 16 / Tr::kBytes;
  if (!p) {
#pragma unroll
    for (int e = 0; e < kEpc; ++e) out[e] = fill;
  } else if (Tr::kBytes == 2 && !is_f32) {
    const u32x4 u = load16<Tr>((const typename Tr::T*)p + c0, c - c0);
#pragma unroll
    for (int e = 0; e < kEpc; ++e) out[e] = elem<Tr>(u, e);
  } else {
#pragma unroll
    for (int e0 = 0; e0 < kEpc; e0 += 4) {
      const u32x4 u = load16<F32>((const float*)p + c0 + e0, c - c0 - e0);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e0 + e] = __uint_as_float(u[e]);
    }
  }
}

template <class Tr, int NT, int NV>
__global__ __launch_bounds__(256) void norm_kernel(NormArgs a) {
  using T = typename Tr::T;
  constexpr int kEpc = 16 / Tr::kBytes;
  __shared__ float red[4];
  const int lane = threadIdx.x % NT;
  const int64_t row = (int64_t)blockIdx.x * (256 / NT) + threadIdx.x / NT;
  const int64_t r = row < a.m ? row : a.m - 1;  // (whole waves stay in the reductions)
  const T* x = (const T*)a.x + r * a.x_stride;
  u32x4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = (i * NT + lane) * kEpc;
    raw[i] = load16<Tr>(x + c0, a.c - c0);
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < kEpc; ++e) s += elem<Tr>(raw[i], e);
  const float mean = row_sum<NT>(s, red) / (float)a.c;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int n = a.c - (i * NT + lane) * kEpc;
#pragma unroll
    for (int e = 0; e < kEpc; ++e) {
      const float d = e < n ? elem<Tr>(raw[i], e) - mean : 0.f;
      q += d * d;
    }
  }
  const float rstd = 1.f / sqrtf(row_sum<NT>(q, red) / (float)a.c + a.eps);
  if (row >= a.m) return;
  if (lane == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  T* y = (T*)a.y + row * a.y_stride;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = (i * NT + lane) * kEpc;
    if (c0 >= a.c) break;
    float w[kEpc], b[kEpc], v[kEpc];
    params<Tr>(a.w, c0, a.c, a.param_f32, a.dtype, 1.f, w);
    params<Tr>(a.b, c0, a.c, a.param_f32, a.dtype, 0.f, b);
#pragma unroll
    for (int e = 0; e < kEpc; ++e) v[e] = (elem<Tr>(raw[i], e) - mean) * rstd * w[e] + b[e];
    store16<Tr>(y + c0, v, a.c - c0);
  }
}

// Rows too wide for registers: a workgroup per row, three passes (the second and third from L2).
template <class Tr>
__global__ __launch_bounds__(256) void norm_wide_kernel(NormArgs a) {
  using T = typename Tr::T;
  constexpr int kEpc = 16 / Tr::kBytes;
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.x_stride;
  T* y = (T*)a.y + row * a.y_stride;
  float s = 0.f, q = 0.f;
  for (int c0 = threadIdx.x * kEpc; c0 < a.c; c0 += 256 * kEpc) {
    const u32x4 u = load16<Tr>(x + c0, a.c - c0);
#pragma unroll
    for (int e = 0; e < kEpc; ++e) s += elem<Tr>(u, e);
  }
  const float mean = row_sum<256>(s, red) / (float)a.c;
  for (int c0 = threadIdx.x * kEpc; c0 < a.c; c0 += 256 * kEpc) {
    const u32x4 u = load16<Tr>(x + c0, a.c - c0);
#pragma unroll
    for (int e = 0; e < kEpc; ++e) {
      const float d = c0 + e < a.c ? elem<Tr>(u, e) - mean : 0.f;
      q += d * d;
    }
  }
  const float rstd = 1.f / sqrtf(row_sum<256>(q, red) / (float)a.c + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  for (int c0 = threadIdx.x * kEpc; c0 < a.c; c0 += 256 * kEpc) {
    const u32x4 u = load16<Tr>(x + c0, a.c - c0);
    float w[kEpc], b[kEpc], v[kEpc];
    params<Tr>(a.w, c0, a.c, a.param_f32, a.dtype, 1.f, w);
    params<Tr>(a.b, c0, a.c, a.param_f32, a.dtype, 0.f, b);
#pragma unroll
    for (int e = 0; e < kEpc; ++e) v[e] = (elem<Tr>(u, e) - mean) * rstd * w[e] + b[e];
    store16<Tr>(y + c0, v, a.c - c0);
  }
}

template <class Tr, int NT, int NV>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void norm_grad_kernel(NormGradArgs a) {
  using T = typename Tr::T;
  constexpr int kEpc = 16 / Tr::kBytes, kRows = NT < 256 ? 256 / NT : 1;
  extern __shared__ float lds[];  // [kRows][c] while the column sums meet; row_sum's words
  const int lane = threadIdx.x % NT, sub = threadIdx.x / NT;
  u32x4 w[NV];  // dtype, or unused with float32 parameters next to 16-bit rows
  float aw[NV * kEpc], ab[NV * kEpc];
#pragma unroll
  for (int i = 0; i < NV * kEpc; ++i) aw[i] = ab[i] = 0.f;
  const bool own_w = a.w && (Tr::kBytes == 4 || !a.param_f32);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = (i * NT + lane) * kEpc;
    if (own_w) w[i] = load16<Tr>((const T*)a.w + c0, a.c - c0);
  }
  const float inv = 1.f / (float)a.c;
  const int64_t step = (int64_t)gridDim.x * kRows;
  u32x4 xn[NV], gn[NV];  // the next row, on its way while one is worked on
  float mean_n = 0.f, rstd_n = 0.f;
  auto fetch = [&](int64_t row) {
    const bool live = row < a.m;
    const int64_t r = live ? row : a.m - 1;
    const T* x = (const T*)a.x + r * a.x_stride;
    const T* dy = (const T*)a.dy + r * a.dy_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = (i * NT + lane) * kEpc;
      xn[i] = load16<Tr>(x + c0, a.c - c0);
      gn[i] = load16<Tr>(dy + c0, live ? a.c - c0 : 0);
    }
    mean_n = a.mean[r];
    rstd_n = a.rstd[r];
  };
  fetch((int64_t)blockIdx.x * kRows + sub);
  for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < a.m; row0 += step) {
    const int64_t row = row0 + sub;
    const bool live = row < a.m;
    const float rstd = rstd_n, mean = mean_n;
    float h[NV * kEpc], g[NV * kEpc];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float wf[kEpc];
      if (!own_w) params<Tr>(a.w, (i * NT + lane) * kEpc, a.c, a.param_f32, a.dtype, 1.f, wf);
#pragma unroll
      for (int e = 0; e < kEpc; ++e) {
        const int k = i * kEpc + e;
        const float d = elem<Tr>(gn[i], e);
        h[k] = (elem<Tr>(xn[i], e) - mean) * rstd;  // (as forward: x rstd - mean rstd would round the offset's product)
        g[k] = d * (own_w ? elem<Tr>(w[i], e) : wf[e]);
        s1 += g[k];
        s2 = fmaf(g[k], h[k], s2);
        aw[k] = fmaf(d, h[k], aw[k]);
        ab[k] += d;
      }
    }
    if (row0 + step < a.m) fetch(row + step);
    if (a.dx) {
      s1 = row_sum<NT>(s1, lds) * inv;
      s2 = row_sum<NT>(s2, lds) * inv;
      if (live) {
        T* dx = (T*)a.dx + row * a.dx_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c0 = (i * NT + lane) * kEpc;
          if (c0 >= a.c) break;
          float v[kEpc];
#pragma unroll
          for (int e = 0; e < kEpc; ++e) v[e] = rstd * fmaf(-h[i * kEpc + e], s2, g[i * kEpc + e] - s1);
          store16<Tr>(dx + c0, v, a.c - c0);
        }
      }
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = a.part + ((int64_t)blockIdx.x * 2 + which) * a.c;
    const float* acc = which ? ab : aw;
    if constexpr (kRows == 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * NT + lane) * kEpc;
#pragma unroll
        for (int e = 0; e < kEpc; e += 4) store16<F32>(out + c + e, acc + i * kEpc + e, a.c - c - e);
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV * kEpc; ++i) {
        const int c = (i / kEpc * NT + lane) * kEpc + i % kEpc;
        if (c < a.c) lds[sub * a.c + c] = acc[i];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.c; c += 256) {
        float v = 0.f;
#pragma unroll
        for (int s = 0; s < kRows; ++s) v += lds[s * a.c + c];
        out[c] = v;
      }
    }
  }
}

// Rows too wide for registers: dx by a workgroup per row in two passes ...
template <class Tr>
__global__ __launch_bounds__(256) void norm_grad_wide_kernel(NormGradArgs a) {
  using T = typename Tr::T;
  constexpr int kEpc = 16 / Tr::kBytes;
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.x_stride;
  const T* dy = (const T*)a.dy + row * a.dy_stride;
  T* dx = (T*)a.dx + row * a.dx_stride;
  const float mean = a.mean[row], rstd = a.rstd[row], inv = 1.f / (float)a.c;
  float s1 = 0.f, s2 = 0.f;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    for (int c0 = threadIdx.x * kEpc; c0 < a.c; c0 += 256 * kEpc) {
      const u32x4 xr = load16<Tr>(x + c0, a.c - c0), gr = load16<Tr>(dy + c0, a.c - c0);
      float w[kEpc], v[kEpc];
      params<Tr>(a.w, c0, a.c, a.param_f32, a.dtype, 1.f, w);
#pragma unroll
      for (int e = 0; e < kEpc; ++e) {
        const float h = (elem<Tr>(xr, e) - mean) * rstd, g = elem<Tr>(gr, e) * w[e];
        if (pass == 0) {
          s1 += g;
          s2 += g * h;
        }
        v[e] = rstd * (g - s1 - h * s2);
      }
      if (pass) store16<Tr>(dx + c0, v, a.c - c0);
    }
    if (pass == 0) {
      s1 = row_sum<256>(s1, red) * inv;
      s2 = row_sum<256>(s2, red) * inv;
    }
  }
}

// ... and the column sums by workgroups of 64 chunks x 4 rows, blockIdx.y a block of rows.
template <class Tr>
__global__ __launch_bounds__(256) void norm_cols_kernel(NormGradArgs a) {
  using T = typename Tr::T;
  constexpr int kEpc = 16 / Tr::kBytes;
  __shared__ float lds[4][64 * kEpc];
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6;
  const int c0 = (blockIdx.x * 64 + lane) * kEpc;
  float aw[kEpc], ab[kEpc];
#pragma unroll
  for (int e = 0; e < kEpc; ++e) aw[e] = ab[e] = 0.f;
  for (int64_t row = (int64_t)blockIdx.y * 4 + sub; row < a.m; row += (int64_t)gridDim.y * 4) {
    const u32x4 xr = load16<Tr>((const T*)a.x + row * a.x_stride + c0, a.c - c0);
    const u32x4 gr = load16<Tr>((const T*)a.dy + row * a.dy_stride + c0, a.c - c0);
    const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
    for (int e = 0; e < kEpc; ++e) {
      const float d = elem<Tr>(gr, e);
      aw[e] += d * ((elem<Tr>(xr, e) - mean) * rstd);
      ab[e] += d;
    }
  }
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEpc; ++e) lds[sub][lane * kEpc + e] = which ? ab[e] : aw[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * kEpc; i += 256) {
      const int c = blockIdx.x * 64 * kEpc + i;
      if (c < a.c) a.part[((int64_t)blockIdx.y * 2 + which) * a.c + c] = (lds[0][i] + lds[1][i]) + (lds[2][i] + lds[3][i]);
    }
  }
}

// dw / db from the workgroups' rows: 32 columns x 32 ranges of rows, 8 loads in flight each, all
// added in a fixed order.
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const float* part, int n_part, int c, void* dw, void* db,
                                                           int param_f32, int dtype) {
  __shared__ float lds[32][33];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, which = blockIdx.y;
  void* out = which ? db : dw;
  if (!out) return;
  float s = 0.f;
  if (col < c) {
    const float* p = part + (int64_t)which * c + col;
    for (int r0 = g; r0 < n_part; r0 += 256) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = r0 + 32 * i < n_part ? p[(int64_t)(r0 + 32 * i) * 2 * c] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
  }
  lds[g][lane] = s;
  __syncthreads();
  if (g == 0 && col < c) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += lds[i][lane];
    store_param(out, col, v, param_f32, dtype);
  }
}

constexpr int kMaxChunks = 4 * 256;       // a row in the registers of a workgroup
constexpr int kGradGroups = 768;          // workgroups (and rows of partial sums) of the backward pass

constexpr int kNarrowRows = 8192;

// run(part, its workgroups) for the parts of a call's rows that a launch holds each, `per` rows per workgroup
template <class F>
void for_rows(const NormArgs& a, int64_t per, int bytes, F&& run) {
  const int64_t most = most_groups(256) * per;
  for (int64_t r0 = 0; r0 < a.m; r0 += most) {
    NormArgs p = a;
    p.x += r0 * a.x_stride * bytes, p.y += r0 * a.y_stride * bytes;
    if (p.mean) p.mean += r0;
    if (p.rstd) p.rstd += r0;
    p.m = a.m - r0 < most ? a.m - r0 : most;
    run(p, dim3((unsigned)cdiv(p.m, per)));
  }
}
template <class Tr, int NT>
void launch_norm(const NormArgs& all, int nv, hipStream_t st) {
  for_rows(all, 256 / NT, Tr::kBytes, [&](const NormArgs& a, dim3 grid) {
    if constexpr (NT == 16) {
      switch (nv) {
        case 5: launch((norm_kernel<Tr, NT, 5>), grid, dim3(256), 0, st, a); return;
        case 6: launch((norm_kernel<Tr, NT, 6>), grid, dim3(256), 0, st, a); return;
        case 7: launch((norm_kernel<Tr, NT, 7>), grid, dim3(256), 0, st, a); return;
        case 8: launch((norm_kernel<Tr, NT, 8>), grid, dim3(256), 0, st, a); return;
        default: break;
      }
    }
    switch (nv) {
      case 1: launch((norm_kernel<Tr, NT, 1>), grid, dim3(256), 0, st, a); break;
      case 2: launch((norm_kernel<Tr, NT, 2>), grid, dim3(256), 0, st, a); break;
      case 3: launch((norm_kernel<Tr, NT, 3>), grid, dim3(256), 0, st, a); break;
      default: launch((norm_kernel<Tr, NT, 4>), grid, dim3(256), 0, st, a); break;
    }
  });
}
template <class Tr>
void run_norm(const NormArgs& a, hipStream_t st) {
  const int chunks = (int)cdiv(a.c, 16 / Tr::kBytes);
  // 16 lanes a row while that fills the chip (wider rows then use every lane); else a wave, a workgroup
  if (chunks <= 16 || (chunks <= 8 * 16 && a.m >= kNarrowRows)) launch_norm<Tr, 16>(a, (int)cdiv(chunks, 16), st);
  else if (chunks <= 4 * 64) launch_norm<Tr, 64>(a, (int)cdiv(chunks, 64), st);
  else if (chunks <= kMaxChunks) launch_norm<Tr, 256>(a, (int)cdiv(chunks, 256), st);
  else for_rows(a, 1, Tr::kBytes, [&](const NormArgs& p, dim3 grid) { launch(norm_wide_kernel<Tr>, grid, dim3(256), 0, st, p); });
}

template <class Tr, int NT>
void launch_norm_grad(const NormGradArgs& a, int nv, int groups, hipStream_t st) {
  const size_t lds = NT >= 256 ? NT / 64 * 4 : (size_t)(256 / NT) * a.c * 4;
  const dim3 block(NT < 256 ? 256 : NT);
  if (nv == 1) launch((norm_grad_kernel<Tr, NT, 1>), dim3(groups), block, lds, st, a);
  else launch((norm_grad_kernel<Tr, NT, 2>), dim3(groups), block, lds, st, a);
}
// Lanes per row of the backward pass: at most two chunks each, whose sums, row and next row are some
// 150 registers (four took 270, one wave per SIMD: 10000 x 8192 bf16 187 us).  Two of 16 lanes only with
// rows enough to fill the chip (163840 x 192 bf16, x given as dy too: 32 us, in 64 lanes 61).
inline int grad_lanes(int64_t m, int chunks) {
  if (chunks <= 16 || (chunks <= 32 && m >= kNarrowRows)) return 16;
  return chunks <= 128 ? 64 : chunks <= 512 ? 256 : 512;
}
// Workgroups: enough for the chip, several rows each so that their sums are not most of the traffic
inline int grad_groups(int64_t m, int c, int bytes) {
  const int nt = grad_lanes(m, (int)cdiv(c, 16 / bytes));
  const int64_t turns = cdiv(m, nt < 256 ? 256 / nt : 1);
  const int64_t g = turns / 4 < 128 ? 128 : turns / 4;
  return (int)(turns < g ? turns : g > kGradGroups ? kGradGroups : g);
}
template <class Tr>
void run_norm_grad(const NormGradArgs& a, hipStream_t st) {
  const int chunks = (int)cdiv(a.c, 16 / Tr::kBytes);
  const int groups = grad_groups(a.m, a.c, Tr::kBytes);
  if (chunks > kMaxChunks) {
    for (int64_t r0 = 0; a.dx && r0 < a.m; r0 += most_groups(256)) {
      NormGradArgs p = a;
      p.x += r0 * a.x_stride * Tr::kBytes, p.dy += r0 * a.dy_stride * Tr::kBytes, p.dx += r0 * a.dx_stride * Tr::kBytes;
      p.mean += r0, p.rstd += r0;
      launch(norm_grad_wide_kernel<Tr>, dim3((unsigned)(a.m - r0 < most_groups(256) ? a.m - r0 : most_groups(256))), dim3(256), 0,
                         st, p);
    }
    if (a.part)
      launch(norm_cols_kernel<Tr>, dim3((unsigned)cdiv(chunks, 64), groups), dim3(256), 0, st, a);
    return;
  }
  switch (grad_lanes(a.m, chunks)) {
    case 16: launch_norm_grad<Tr, 16>(a, (int)cdiv(chunks, 16), groups, st); break;
    case 64: launch_norm_grad<Tr, 64>(a, (int)cdiv(chunks, 64), groups, st); break;
    case 256: launch_norm_grad<Tr, 256>(a, (int)cdiv(chunks, 256), groups, st); break;
    default: launch_norm_grad<Tr, 512>(a, (int)cdiv(chunks, 512), groups, st); break;
  }
}

int check_rows(const char* fn, int dtype, int64_t m, int64_t c) {
  YK_CHECK_ARG(tok_bytes(dtype), std::string(fn) + ": dtype must be YK_ACT_BF16, YK_ACT_F32 or YK_ACT_F16");
  YK_CHECK_ARG(m >= 0 && m <= INT32_MAX && c >= 1 && c <= (1 << 30), std::string(fn) + ": sizes out of range (m in [0, 2^31), c in [1, 2^30])");
  return YK_OK;
}

}  // namespace tok
}  // namespace yk

using namespace yk::tok;

extern "C" {

int yk_layer_norm(yk_ctx* ctx, const yk_layer_norm_args* a, void* stream) {
  YK_CHECK_ARG(ctx && a, "yk_layer_norm: NULL argument");
  if (const int rc = check_rows("yk_layer_norm", a->dtype, a->m, a->c)) return rc;
  YK_CHECK_ARG(a->eps >= 0.f, "yk_layer_norm: eps must be >= 0");
  if (a->m == 0) return YK_OK;
  YK_CHECK_ARG(a->x && a->y, "yk_layer_norm: x and y must be set");
  YK_CHECK_ARG(a->x_stride >= 0 && (a->m == 1 || a->y_stride >= a->c),
               "yk_layer_norm: a negative row stride, or y's is shorter than its row");
  yk::DeviceGuard g(ctx->device);
  NormArgs k{(const char*)a->x, a->w, a->b, (char*)a->y, a->mean, a->rstd, a->m, a->x_stride, a->y_stride,
             (int)a->c, a->param_f32 || a->dtype == YK_ACT_F32, a->dtype, a->eps};
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == YK_ACT_F32) run_norm<F32>(k, st);
  else if (a->dtype == YK_ACT_BF16) run_norm<B16>(k, st);
  else run_norm<H16>(k, st);
  return launched("yk_layer_norm");
}

int yk_layer_norm_backward_workspace(const yk_layer_norm_grad_args* a, int64_t* bytes) {
  YK_CHECK_ARG(a && bytes, "yk_layer_norm_backward_workspace: NULL argument");
  if (const int rc = check_rows("yk_layer_norm_backward_workspace", a->dtype, a->m, a->c)) return rc;
  *bytes = (int64_t)grad_groups(a->m, (int)a->c, tok_bytes(a->dtype)) * 2 * a->c * 4;
  return YK_OK;
}

int yk_layer_norm_backward(yk_ctx* ctx, const yk_layer_norm_grad_args* a, void* stream) {
  YK_CHECK_ARG(ctx && a, "yk_layer_norm_backward: NULL argument");
  if (const int rc = check_rows("yk_layer_norm_backward", a->dtype, a->m, a->c)) return rc;
  const bool cols = a->dw || a->db;
  if (!cols && (!a->dx || a->m == 0)) return YK_OK;
  int64_t need = 0;
  if (const int rc = yk_layer_norm_backward_workspace(a, &need)) return rc;
  YK_CHECK_ARG(a->m == 0 || (a->dy && a->x && a->mean && a->rstd), "yk_layer_norm_backward: dy, x, mean and rstd must be set");
  YK_CHECK_ARG(a->x_stride >= 0 && a->dy_stride >= 0 && (!a->dx || a->m <= 1 || a->dx_stride >= a->c),
               "yk_layer_norm_backward: a negative row stride, or dx's is shorter than its row");
  YK_CHECK_ARG(!cols || need == 0 || (a->ws && a->ws_bytes >= need && (uintptr_t)a->ws % 16 == 0),
               "yk_layer_norm_backward: dw / db need yk_layer_norm_backward_workspace bytes of 16-byte aligned scratch");
  yk::DeviceGuard g(ctx->device);
  const hipStream_t st = (hipStream_t)stream;
  const int f32 = a->param_f32 || a->dtype == YK_ACT_F32;
  NormGradArgs k{(const char*)a->dy, (const char*)a->x, a->w, a->mean, a->rstd, (char*)a->dx,
                 cols ? (float*)a->ws : nullptr, a->m, a->dy_stride, a->x_stride, a->dx_stride, (int)a->c, f32, a->dtype};
  if (a->m > 0) {
    if (a->dtype == YK_ACT_F32) run_norm_grad<F32>(k, st);
    else if (a->dtype == YK_ACT_BF16) run_norm_grad<B16>(k, st);
    else run_norm_grad<H16>(k, st);
  }
  if (cols)
    launch(norm_reduce_kernel, dim3((unsigned)cdiv(a->c, 32), 2), dim3(1024), 0, st, (const float*)a->ws,
                       grad_groups(a->m, (int)a->c, tok_bytes(a->dtype)), (int)a->c, a->dw, a->db, f32, a->dtype);
  return launched("yk_layer_norm_backward");
}

}  // extern "C"
