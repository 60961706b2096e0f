// h = x + r,  y = h * rsqrt(mean(h^2) + eps) * w  over the last axis: the residual's addition and the root-mean-square norm
// in one pass (RMSNorm rrnco/models/nn/attn_freenet.py:13-26 behind the skip connection), its gradient, and a form
// that hands y on in 8 bits with a scale for every 128 columns.
//
//   forward    s = rsqrt(mean h^2 + eps); the norm is taken of the 32-bit sum, h and y are rounded once each when stored
//   backward   g = dy w, n = h s:   dx = dr = dh + s (g - n mean(g n)),   dw = sum over the rows of dy n
//   8 bits     a = max |y| over a group of 128 columns, scale = max(a / 448, 2^-126) (1 for a group of zeros), q = e4m3(y / scale)
//
// Bound by memory: each tensor is read and written once, a row's elements stay in registers between the two uses.
// 51 200 x 128 float32: forward 18.5 us (5.7 TB/s, part of it from the cache), backward 21.5 us, dw's second launch 4; 8 192 x 4 096 bf16 to 8 bits 38 - 48 us (4.9 TB/s, a copy's rate).
// A team of TPR lanes owns a row (TPR 16 .. 1024, chosen so that a lane holds 16 bytes up to a width of 64 such pieces and at
// most 64 bytes beyond), so that narrow rows share a wave and the sum of squares is a few lane exchanges.
// dw: each workgroup sums its rows in registers, the teams are joined through LDS in a fixed order and one partial row per
// workgroup is written; a second launch adds the partials in order (no atomics: the same result every time).
#include "rr_types.h"

namespace {

template <int TPR>
__device__ __forceinline__ float team_sum(float v, float* red) {          // red: one float per wave of the workgroup
#pragma unroll
  for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) v += __shfl_xor(v, o);
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += red[i];                              // TPR > 64: the workgroup is one team
  }
  return v;
}

// 1 / sqrt(mean h^2 + eps) from the sum of squares.  Where that left the range of 32 bits (elements beyond 1e18, or under 1e-15 with hardly an eps) it is taken
// again of the elements times a power of two
template <int TPR, int NC, int VEC>
__device__ __forceinline__ float rstd_of(float ss, const float (&v)[NC][VEC], int E, float eps, float* red) {
  const float m = ss / (float)E + eps;
  if (m >= 0x1p-100f && m < INFINITY) return 1.0f / sqrtf(m);            // (one value in all lanes of the team)
  const float f = m < 1.f ? 0x1p75f : 0x1p-75f;
  ss = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < VEC; ++i) ss = fmaf(v[c][i] * f, v[c][i] * f, ss);
  return f / sqrtf(team_sum<TPR>(ss, red) / (float)E + eps * f * f);
}

template <typename T> struct code;
template <> struct code<float> { static constexpr int v = RR_F32; };
template <> struct code<rr_f16> { static constexpr int v = RR_F16; };
template <> struct code<rr_bf16> { static constexpr int v = RR_BF16; };

// N weights from column c on, n of them in the row, of the inputs' type or float32; ones without a weight
template <typename T, int N>
__device__ __forceinline__ void load_w(const void* w, int w32, int c, int n, float (&x)[N]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 1.f;
  } else if (w32 || code<T>::v == RR_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      float v[4];
      rr_load_first<float, 4>((const float*)w + c + i, n - i, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i + e] = v[e];
    }
  } else {
    rr_load_first<T, N>((const T*)w + c, n, x);
  }
}

// ------------------------------------------------------------------------------------------------ forward
template <typename T, int TPR, int NC, bool FP8>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_rms_fwd(const T* __restrict__ x, long ldx, const T* __restrict__ res, long ldr,
                                                                  const void* __restrict__ w, int w32, T* __restrict__ y, T* __restrict__ h,
                                                                  float* __restrict__ rstd, uint8_t* __restrict__ q, float* __restrict__ qs,
                                                                  long rows, int E, float eps) {
  constexpr int VEC = rr_vec_of<T>::N, BLK = TPR > 256 ? TPR : 256, TEAMS = BLK / TPR;
  __shared__ float red[BLK / 64];
  const int team = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  const long row = (long)blockIdx.x * TEAMS + team;
  const bool live = row < rows;                                            // (a dead team still takes part in the barriers)
  float v[NC][VEC];
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * TPR + lane) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[c][i] = 0.f;
    if (live && col < E) {
      rr_load_first<T, VEC>(x + row * ldx + col, E - col, v[c]);
      if (res != nullptr) {
        float r[VEC];
        rr_load_first<T, VEC>(res + row * ldr + col, E - col, r);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[c][i] += r[i];
      }
      if (h != nullptr) rr_store_first<T, VEC>(h + row * (long)E + col, E - col, v[c]);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) ss = fmaf(v[c][i], v[c][i], ss);
  }
  ss = team_sum<TPR>(ss, red);
  const float s = rstd_of<TPR>(ss, v, E, eps, red);
  if (rstd != nullptr && live && lane == 0) rstd[row] = s;
  if constexpr (!FP8) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + lane) * VEC;
      if (live && col < E) {
        float g[VEC];
        load_w<T, VEC>(w, w32, col, E - col, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[i] = v[c][i] * s * g[i];
        rr_store_first<T, VEC>(y + row * (long)E + col, E - col, g);
      }
    }
  } else {
    const int G = (E + 127) / 128;
    float a[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + lane) * VEC;
      a[c] = 0.f;
      if (live && col < E) {
        float g[VEC];
        load_w<T, VEC>(w, w32, col, E - col, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) { v[c][i] = v[c][i] * s * g[i]; a[c] = fmaxf(a[c], fabsf(v[c][i])); }      // (zeros behind the row's end)
      }
      constexpr int GL = 128 / VEC;               // lanes of a group
#pragma unroll
      for (int o = 1; o < (TPR < GL ? TPR : GL); o <<= 1) a[c] = fmaxf(a[c], __shfl_xor(a[c], o));
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + lane) * VEC;
      if (live && col < E) {
        const float sc = a[c] == 0.f ? 1.f : fmaxf(a[c] / 448.0f, 0x1p-126f);      // (a smaller one has no finite reciprocal)
        if (col % 128 == 0) qs[row * G + col / 128] = sc;
        const float inv = 1.0f / sc;                                       // one quotient a group; y * inv is off by a step of float32 at the most
        uint32_t p[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
          float z[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            z[e] = v[c][i + e] * inv;
            z[e] = z[e] != z[e] ? z[e] : fminf(fmaxf(z[e], -448.f), 448.f);      // the product may pass 448 by a rounding
          }
          int b = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
          p[i / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], b, true);
        }
        uint8_t* dst = q + row * (long)E + col;
        if (col + VEC <= E) __builtin_memcpy(dst, p, VEC);
        else {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (col + i < E) dst[i] = (uint8_t)(p[i / 4] >> (8 * (i % 4)));
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward
template <typename T, int TPR, int NC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_rms_bwd(const T* __restrict__ x, long ldx, const T* __restrict__ res, long ldr,
                                                                  const void* __restrict__ w, int w32, const T* __restrict__ dy, long lddy,
                                                                  const T* __restrict__ dh, long lddh, const float* __restrict__ rstd,
                                                                  T* __restrict__ dx, float* __restrict__ dwp, long rows, int E) {
  constexpr int VEC = rr_vec_of<T>::N, BLK = TPR > 256 ? TPR : 256, TEAMS = BLK / TPR;
  __shared__ float red[BLK / 64];
  __shared__ float join[TEAMS > 1 ? TEAMS * TPR * VEC : 1];
  const int team = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  float gw[NC][VEC], acc[NC][VEC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * TPR + lane) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) { gw[c][i] = 0.f; acc[c][i] = 0.f; }
    if (col < E) load_w<T, VEC>(w, w32, col, E - col, gw[c]);
  }
  for (long r0 = (long)blockIdx.x * TEAMS; r0 < rows; r0 += (long)gridDim.x * TEAMS) {     // (uniform in the workgroup: the barriers inside are met)
    const long row = r0 + team;
    const bool live = row < rows;
    float n[NC][VEC], g[NC][VEC];
    const float s = live ? rstd[row] : 0.f;
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + lane) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) { n[c][i] = 0.f; g[c][i] = 0.f; }
      if (live && col < E) {
        rr_load_first<T, VEC>(x + row * ldx + col, E - col, n[c]);
        if (res != nullptr) {
          float r[VEC];
          rr_load_first<T, VEC>(res + row * ldr + col, E - col, r);
#pragma unroll
          for (int i = 0; i < VEC; ++i) n[c][i] += r[i];
        }
        rr_load_first<T, VEC>(dy + row * lddy + col, E - col, g[c]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        n[c][i] *= s;
        acc[c][i] = fmaf(g[c][i], n[c][i], acc[c][i]);
        g[c][i] *= gw[c][i];
        dot = fmaf(g[c][i], n[c][i], dot);
      }
    }
    dot = team_sum<TPR>(dot, red) / (float)E;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + lane) * VEC;
      if (live && col < E) {
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = 0.f;
        if (dh != nullptr) rr_load_first<T, VEC>(dh + row * lddh + col, E - col, o);
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = fmaf(s, g[c][i] - n[c][i] * dot, o[i]);
        rr_store_first<T, VEC>(dx + row * (long)E + col, E - col, o);
      }
    }
  }
  if (dwp == nullptr) return;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * TPR + lane) * VEC;
    if constexpr (TEAMS > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VEC; ++i) join[(team * TPR + lane) * VEC + i] = acc[c][i];
      __syncthreads();
      if (team == 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float t = 0.f;
          for (int k = 0; k < TEAMS; ++k) t += join[(k * TPR + lane) * VEC + i];
          acc[c][i] = t;
        }
      }
    }
    if (team == 0 && col < E) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (col + i < E) dwp[(long)blockIdx.x * E + col + i] = acc[c][i];
    }
  }
}

// dw[c] = sum of the P partial rows: 16 columns a workgroup, 64 lanes of rows each, joined in order through LDS
__global__ __launch_bounds__(1024) void k_rms_dw(const float* __restrict__ dwp, int P, int E, void* __restrict__ dw, int dtype) {
  __shared__ float part[64][17];
  const int lane = threadIdx.x & 15, row = threadIdx.x >> 4, c = blockIdx.x * 16 + lane;
  float t = 0.f;
  if (c < E) {
#pragma unroll 4
    for (int p = row; p < P; p += 64) t += dwp[(long)p * E + c];
  }
  part[row][lane] = t;
#pragma unroll
  for (int h = 32; h > 0; h >>= 1) {
    __syncthreads();
    if (row < h) part[row][lane] += part[row + h][lane];
  }
  if (row == 0 && c < E) {
    t = part[0][lane];
    if (dtype == RR_F32) ((float*)dw)[c] = t;
    else if (dtype == RR_F16) ((rr_f16*)dw)[c] = (rr_f16)t;
    else ((rr_bf16*)dw)[c] = (rr_bf16)t;
  }
}

// team size and pieces a lane by the number of 16-byte pieces of a row
#define RR_NORM_DISPATCH(RUN)                                                                                                              \
  do {                                                                                                                                    \
    const int pieces = (E + rr_vec_of<T>::N - 1) / rr_vec_of<T>::N;                                                                       \
    if (pieces <= 16) { RUN(16, 1); } else if (pieces <= 32) { RUN(32, 1); } else if (pieces <= 64) { RUN(64, 1); }                        \
    else if (pieces <= 128) { RUN(64, 2); } else if (pieces <= 256) { RUN(64, 4); } else if (pieces <= 512) { RUN(256, 2); }               \
    else if (pieces <= 1024) { RUN(256, 4); } else { RUN(1024, 4); }      /* up to 16 384 float32 */                                       \
  } while (0)

template <typename T>
int norm_fwd(const void* x, long ldx, const void* res, long ldr, const void* w, int w32, void* y, void* h, float* rstd, uint8_t* q, float* qs, long rows, int E,
             float eps, hipStream_t st) {
#define RR_GRID(TPR) dim3((unsigned)((rows + (TPR > 256 ? 1 : 256 / TPR) - 1) / (TPR > 256 ? 1 : 256 / TPR))), dim3(TPR > 256 ? TPR : 256)
#define RR_GO8(TPR, NC) \
  hipLaunchKernelGGL((k_rms_fwd<T, TPR, NC, true>), RR_GRID(TPR), 0, st, (const T*)x, ldx, (const T*)res, ldr, w, w32, (T*)y, (T*)h, rstd, q, qs, rows, E, eps)
#define RR_GOT(TPR, NC) \
  hipLaunchKernelGGL((k_rms_fwd<T, TPR, NC, false>), RR_GRID(TPR), 0, st, (const T*)x, ldx, (const T*)res, ldr, w, w32, (T*)y, (T*)h, rstd, q, qs, rows, E, eps)
  if (q != nullptr) RR_NORM_DISPATCH(RR_GO8);
  else RR_NORM_DISPATCH(RR_GOT);
  return rr_check(hipGetLastError());
}

template <typename T>
int norm_bwd(const void* x, long ldx, const void* res, long ldr, const void* w, int w32, const void* dy, long lddy, const void* dh, long lddh, const float* rstd,
             void* dx, void* dw, float* dwp, int parts, long rows, int E, hipStream_t st) {
#define RR_GOB(TPR, NC) \
  hipLaunchKernelGGL((k_rms_bwd<T, TPR, NC>), dim3((unsigned)parts), dim3(TPR > 256 ? TPR : 256), 0, st, (const T*)x, ldx, (const T*)res, ldr, w, w32, \
                     (const T*)dy, lddy, (const T*)dh, lddh, rstd, (T*)dx, dw != nullptr ? dwp : (float*)nullptr, rows, E)
  RR_NORM_DISPATCH(RR_GOB);
  if (dw != nullptr) hipLaunchKernelGGL(k_rms_dw, dim3((E + 15) / 16), dim3(1024), 0, st, dwp, parts, E, dw, w32 ? RR_F32 : code<T>::v);
  return rr_check(hipGetLastError());
}

}  // namespace

extern "C" int rr_add_rms_norm(int dtype, const void* x, long long ldx, const void* res, long long ldr, const void* w, int w_is_f32, void* y, void* h, float* rstd,
                               uint8_t* q, float* qscale, long long rows, int E, float eps, hipStream_t st) {
  if (rows < 0 || E < 1 || E > 16384 || x == nullptr || rows > 0x7fffffffLL || (y == nullptr) == (q == nullptr) || (q == nullptr) != (qscale == nullptr) || ldx < 0 || ldr < 0)
    return RR_EINVAL;
  if (res == nullptr) ldr = 0;
  // a launch holds fewer than 2^32 threads: 16 .. 64 a row up to 128 columns, at most 1 024 beyond
  const long long most = E <= 128 ? 1 << 25 : 1 << 21, size = dtype == RR_F32 ? 4 : 2, G = (E + 127) / 128;
  for (; rows > most; rows -= most) {
    const int rc = rr_add_rms_norm(dtype, x, ldx, res, ldr, w, w_is_f32, y, h, rstd, q, qscale, most, E, eps, st);
    if (rc != RR_OK) return rc;
    x = (const char*)x + most * ldx * size;
    if (res != nullptr) res = (const char*)res + most * ldr * size;
    if (y != nullptr) y = (char*)y + most * E * size;
    if (h != nullptr) h = (char*)h + most * E * size;
    if (rstd != nullptr) rstd += most;
    if (q != nullptr) { q += most * E; qscale += most * G; }
  }
  if (rows == 0) return RR_OK;
  switch (dtype) {
    case RR_F32: return norm_fwd<float>(x, ldx, res, ldr, w, w_is_f32, y, h, rstd, q, qscale, rows, E, eps, st);
    case RR_F16: return norm_fwd<rr_f16>(x, ldx, res, ldr, w, w_is_f32, y, h, rstd, q, qscale, rows, E, eps, st);
    case RR_BF16: return norm_fwd<rr_bf16>(x, ldx, res, ldr, w, w_is_f32, y, h, rstd, q, qscale, rows, E, eps, st);
  }
  return RR_EINVAL;
}

extern "C" int rr_add_rms_norm_parts(long long rows, int E) {      // workgroups of the backward = partial rows of dw (floats [parts][E])
  const long long per = E <= 4096 ? 4 : 1;                         // about four teams a workgroup and four rows a team at the least
  const long long want = (rows + 4 * per - 1) / (4 * per), most = E <= 2048 ? 1024 : 512;      // (512 partial rows of 4 096: 8 MB)
  return (int)(want < 1 ? 1 : want > most ? most : want);
}

extern "C" int rr_add_rms_norm_bwd(int dtype, const void* x, long long ldx, const void* res, long long ldr, const void* w, int w_is_f32, const void* dy, long long lddy,
                                   const void* dh, long long lddh, const float* rstd, void* dx, void* dw, float* workspace, int parts, long long rows, int E,
                                   hipStream_t st) {
  if (rows < 1 || E < 1 || E > 16384 || x == nullptr || dy == nullptr || rstd == nullptr || dx == nullptr || parts < 1 || rows > 0x7fffffffLL ||
      (dw != nullptr && (w == nullptr || workspace == nullptr)) || ldx < 0 || ldr < 0 || lddy < 0 || lddh < 0)
    return RR_EINVAL;
  if (res == nullptr) ldr = 0;
  if (dh == nullptr) lddh = 0;
  switch (dtype) {
    case RR_F32: return norm_bwd<float>(x, ldx, res, ldr, w, w_is_f32, dy, lddy, dh, lddh, rstd, dx, dw, workspace, parts, rows, E, st);
    case RR_F16: return norm_bwd<rr_f16>(x, ldx, res, ldr, w, w_is_f32, dy, lddy, dh, lddh, rstd, dx, dw, workspace, parts, rows, E, st);
    case RR_BF16: return norm_bwd<rr_bf16>(x, ldx, res, ldr, w, w_is_f32, dy, lddy, dh, lddh, rstd, dx, dw, workspace, parts, rows, E, st);
  }
  return RR_EINVAL;
}
