// Token-wise operators of a transformer block (dfcsa.token_ops): the RMS norm of a residual stream
// (training, backward, 8-bit output) and rotary positions with several axes.  All of them move each
// byte once and compute ~10 operations per element, so HBM bandwidth bounds them; every thread loads
// and stores 16-byte words and a row (or a token's angles) stays on chip between its two uses.
#include <cmath>

#include "common.h"
#include "dfcsa_internal.h"

namespace {

// Workgroups of 256 threads in a grid of two dimensions where they are many: a launch counts the
// threads of one dimension in 32 bits.
dim3 grid2(int64_t groups) {
  const int64_t y = (groups + (1 << 22) - 1) >> 22;
  return dim3((unsigned)((groups + y - 1) / y), (unsigned)y);
}
__device__ __forceinline__ int64_t group2() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// ============================================================================ RMS norm
// r = R(x + res); y = T(r * rstd * w), rstd = rsqrt(mean(r^2) + eps).
// The sum of squares, rstd and the products are fp32; r is rounded to the stream's type before the
// statistics because the stream is what the backward (and the next block) reads.
//
// A row is held by WAVES waves of one workgroup (1: C <= 2048, four rows per workgroup and no barrier; 4:
// wider rows), NC chunks of 8 columns per lane, from its one read to its writes.  Measured: 16384 rows of
// 4096 in bf16 87 us forward (537 MB, 6.2 TB/s) and 113 us backward (537 MB, 4.75 TB/s; a large copy moves
// 5.0); 8191 rows of 2560 to 8 bits from an fp32 stream 43 us (231 MB, 5.4 TB/s).
constexpr int kNormMaxC = 16384;
constexpr int kNormMaxRows = 0x7fff0000;   // a row index plus a grid's rows stays an int
constexpr float kE4m3Max = 448.0f;

template <int WAVES>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (WAVES > 1) {
    __syncthreads();   // the previous row's readers are done with red
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}
// |v| as bits: unsigned order is the order of the magnitudes, with NaN above infinity, so a maximum
// over bits keeps a NaN that a float maximum would drop
template <int WAVES>
__device__ __forceinline__ unsigned row_umax(unsigned v, unsigned* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
  if constexpr (WAVES > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = max(max(red[0], red[1]), max(red[2], red[3]));
  }
  return v;
}

__device__ __forceinline__ uint2 pack_e4m3(const float (&v)[8]) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
  return make_uint2((unsigned)lo, (unsigned)hi);
}

// Q8: y8 (e4m3) and scales [rows][C / group] (group == C: one per row) instead of y
template <typename T, typename R, int WAVES, int NC, bool Q8>
__global__ void __launch_bounds__(256) rms_fwd_kernel(int rows, int C, const T* __restrict__ x,
                                                      const R* __restrict__ res, const float* __restrict__ w,
                                                      float eps, T* __restrict__ y, R* __restrict__ r,
                                                      float* __restrict__ rstd_out, unsigned char* __restrict__ y8,
                                                      float* __restrict__ scales, int group) {
  constexpr int LANES = 64 * WAVES, RPW = 4 / WAVES;   // lanes per row, rows per workgroup
  __shared__ float red[4];
  __shared__ unsigned ured[4];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  float wv[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (lane + i * LANES) * 8;
    if (c < C) load8<float>(w + c, wv[i]);
  }
  for (int row = blockIdx.x * RPW + sub; row < rows; row += gridDim.x * RPW) {
    const size_t base = (size_t)row * C;
    float v[NC][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (lane + i * LANES) * 8;
      if (c < C) {
        float a[8];
        load8<T>(x + base + c, a);
        load8<R>(res + base + c, v[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[i][e] = ElemTraits<R>::to_f(ElemTraits<R>::from_f(v[i][e] + a[e]));
          ss += v[i][e] * v[i][e];
        }
        store8<R>(r + base + c, v[i]);
      }
    }
    ss = row_sum<WAVES>(ss, red);
    const float rstd = rsqrtf(ss / (float)C + eps);
    if (rstd_out && lane == 0) rstd_out[row] = rstd;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * rstd * wv[i][e];
    if constexpr (!Q8) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = (lane + i * LANES) * 8;
        if (c < C) store8<T>(y + base + c, v[i]);
      }
    } else {
      unsigned am[NC];
      unsigned all = 0;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        am[i] = 0;
        if ((lane + i * LANES) * 8 < C)
#pragma unroll
          for (int e = 0; e < 8; ++e) am[i] = max(am[i], __float_as_uint(v[i][e]) & 0x7fffffffu);
        all = max(all, am[i]);
      }
      if (group == C) {
        all = row_umax<WAVES>(all, ured);
      } else {   // a group is group / 8 = 4, 8 or 16 neighbouring lanes (C is a multiple of it)
#pragma unroll
        for (int i = 0; i < NC; ++i)
          for (int o = 1; o < group / 8; o <<= 1) am[i] = max(am[i], (unsigned)__shfl_xor((int)am[i], o, 64));
      }
      const int ng = C / group;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = (lane + i * LANES) * 8;
        if (c < C) {
          const float amax = __uint_as_float(group == C ? all : am[i]);
          // a NaN stays a NaN (the comparison is false); a row of zeros keeps a usable scale
          const float sc = (amax < 1e-12f ? 1e-12f : amax) / kE4m3Max;
          const float inv = 1.0f / sc;
          float q[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] = v[i][e] * inv;   // the rounding to e4m3: the operator's output type
          *(uint2*)(y8 + base + c) = pack_e4m3(q);
          if (c % group == 0) scales[(size_t)row * ng + c / group] = sc;
        }
      }
    }
  }
}

// Backward: u = dy * w, xh = r * rstd: d = rstd (u - xh mean(u xh)) + dr; dx = T(d), dres = R(d).
// dw is summed per workgroup over its rows (fp32) into part[gridDim.x][C]; rms_dw_kernel adds those in
// a fixed order, so the result does not depend on the order workgroups run in.  Fetching the next row
// before this one's sum is known measured no faster (115 us): the waves of a CU cover for each other.
template <typename T, typename R, int WAVES, int NC>
__global__ void __launch_bounds__(256) rms_bwd_kernel(int rows, int C, const T* __restrict__ dy,
                                                      const R* __restrict__ dr, const R* __restrict__ r,
                                                      const float* __restrict__ rstd_in, const float* __restrict__ w,
                                                      T* __restrict__ dx, R* __restrict__ dres,
                                                      float* __restrict__ part) {
  constexpr int LANES = 64 * WAVES, RPW = 4 / WAVES;
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) float wred[RPW > 1 ? 512 * NC : 4];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  float wv[NC][8], dw[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (lane + i * LANES) * 8;
    if (c < C) load8<float>(w + c, wv[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
  }
  for (int row = blockIdx.x * RPW + sub; row < rows; row += gridDim.x * RPW) {
    const size_t base = (size_t)row * C;
    const float rstd = rstd_in[row];
    float xh[NC][8], u[NC][8], g[NC][8];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (lane + i * LANES) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) g[i][e] = 0.f;
      if (c < C) {
        load8<R>(r + base + c, xh[i]);
        load8<T>(dy + base + c, u[i]);
        if (dr) load8<R>(dr + base + c, g[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          xh[i][e] *= rstd;
          dw[i][e] += u[i][e] * xh[i][e];
          u[i][e] *= wv[i][e];
          s += u[i][e] * xh[i][e];
        }
      }
    }
    s = row_sum<WAVES>(s, red) / (float)C;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (lane + i * LANES) * 8;
      if (c < C) {
#pragma unroll
        for (int e = 0; e < 8; ++e) g[i][e] += rstd * (u[i][e] - xh[i][e] * s);
        if (dx) store8<T>(dx + base + c, g[i]);
        if (dres) store8<R>(dres + base + c, g[i]);
      }
    }
  }
  if (!part) return;
  if constexpr (RPW > 1) {   // the four waves' sums, one after the other
#pragma unroll 1
    for (int k = 0; k < RPW; ++k) {
      if (sub == k) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          float* p = wred + (lane + i * 64) * 8;
          if (k > 0) {
            float o[8];
            load8<float>(p, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) dw[i][e] += o[e];
          }
          lds_st8(p, dw[i]);
        }
      }
      __syncthreads();
    }
    if (sub != RPW - 1) return;
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (lane + i * LANES) * 8;
    if (c < C) store8<float>(part + (size_t)blockIdx.x * C + c, dw[i]);
  }
}

// out[c] = sum over n rows of part[.][c]: 16 columns per workgroup, 64 row slices of 16 threads with four
// loads in flight each, then the slices in a fixed order (784 rows of 768: 6 us; with 8 slices 29 us)
__global__ void __launch_bounds__(1024) rms_dw_kernel(int n, int C, const float* __restrict__ part,
                                                      float* __restrict__ out) {
  __shared__ float sm[64][17];
  const int cl = threadIdx.x & 15, sl = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < C)
    for (int i = sl; i < n; i += 256)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + 64 * k < n) s[k] += part[(size_t)(i + 64 * k) * C + c];
  sm[sl][cl] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (threadIdx.x < 64) {   // 4 slices of 16 each, then those four
    const int q = threadIdx.x >> 4;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) v += sm[q * 16 + k][cl];
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    if (q == 0 && c < C) out[c] = v;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) dequant_kernel(int64_t n8, int C8, int gsh, int ng,
                                                      const uint2* __restrict__ y8, const float* __restrict__ scales,
                                                      T* __restrict__ out) {
  const int64_t i = group2() * 256 + threadIdx.x;
  if (i >= n8) return;
  const int64_t row = i / C8;
  const int c8 = (int)(i - row * C8);
  const float s = scales[row * ng + (gsh < 0 ? 0 : c8 >> gsh)];
  const uint2 u = y8[i];
  float v[8];
  v[0] = __builtin_amdgcn_cvt_f32_fp8((int)u.x, 0) * s;
  v[1] = __builtin_amdgcn_cvt_f32_fp8((int)u.x, 1) * s;
  v[2] = __builtin_amdgcn_cvt_f32_fp8((int)u.x, 2) * s;
  v[3] = __builtin_amdgcn_cvt_f32_fp8((int)u.x, 3) * s;
  v[4] = __builtin_amdgcn_cvt_f32_fp8((int)u.y, 0) * s;
  v[5] = __builtin_amdgcn_cvt_f32_fp8((int)u.y, 1) * s;
  v[6] = __builtin_amdgcn_cvt_f32_fp8((int)u.y, 2) * s;
  v[7] = __builtin_amdgcn_cvt_f32_fp8((int)u.y, 3) * s;
  store8<T>(out + i * 8, v);
}

// rows one workgroup of the backward walks: one partial dw row per workgroup, so fewer workgroups
// mean fewer partial bytes; 1024 keep four per CU in flight
int bwd_groups(int rows, int C) {
  const int rpw = C <= 2048 ? 4 : 1;
  const int all = (rows + rpw - 1) / rpw;
  return all < 1024 ? all : 1024;
}

template <typename T, typename R, bool Q8>
int launch_fwd(int rows, int C, const void* x, const void* res, const float* w, float eps, void* y, void* r,
               float* rstd, void* y8, float* scales, int group, hipStream_t st) {
  const bool wide = C > 2048;
  const int rpw = wide ? 1 : 4, all = (rows + rpw - 1) / rpw;
  const dim3 grid(all < 4096 ? all : 4096);
  const int chunks = (C / 8 + (wide ? 255 : 63)) / (wide ? 256 : 64);
#define FWD(W, N)                                                                                                  \
  hipLaunchKernelGGL((rms_fwd_kernel<T, R, W, N, Q8>), grid, dim3(256), 0, st, rows, C, (const T*)x, (const R*)res, \
                     w, eps, (T*)y, (R*)r, rstd, (unsigned char*)y8, scales, group)
  if (!wide) {
    if (chunks <= 1) FWD(1, 1);
    else if (chunks <= 2) FWD(1, 2);
    else FWD(1, 4);
  } else {
    if (chunks <= 2) FWD(4, 2);
    else if (chunks <= 4) FWD(4, 4);
    else FWD(4, 8);
  }
#undef FWD
  DFCSA_CHECK_LAUNCH();
  return 0;
}

template <typename T, typename R>
int launch_bwd(int rows, int C, const void* dy, const void* dr, const void* r, const float* rstd, const float* w,
               void* dx, void* dres, float* part, float* dw, hipStream_t st) {
  const bool wide = C > 2048;
  const int n = bwd_groups(rows, C);
  const int chunks = (C / 8 + (wide ? 255 : 63)) / (wide ? 256 : 64);
#define BWD(W, N)                                                                                                 \
  hipLaunchKernelGGL((rms_bwd_kernel<T, R, W, N>), dim3(n), dim3(256), 0, st, rows, C, (const T*)dy, (const R*)dr, \
                     (const R*)r, rstd, w, (T*)dx, (R*)dres, part)
  if (!wide) {
    if (chunks <= 1) BWD(1, 1);
    else if (chunks <= 2) BWD(1, 2);
    else BWD(1, 4);
  } else {
    if (chunks <= 2) BWD(4, 2);
    else if (chunks <= 4) BWD(4, 4);
    else BWD(4, 8);
  }
#undef BWD
  DFCSA_CHECK_LAUNCH();
  if (dw) {
    hipLaunchKernelGGL(rms_dw_kernel, dim3((C + 15) / 16), dim3(1024), 0, st, n, C, part, dw);
    DFCSA_CHECK_LAUNCH();
  }
  return 0;
}

bool norm_shape_ok(int rows, int C) { return rows > 0 && rows <= kNormMaxRows && C >= 8 && C % 8 == 0 && C <= kNormMaxC; }
bool eps_ok(float eps) { return eps >= 0.f && std::isfinite(eps); }
bool types_ok(int t, int r) { return (t == DFCSA_DT_BF16 && (r == DFCSA_DT_BF16 || r == DFCSA_DT_F32)) ||
                                     (t == DFCSA_DT_F32 && r == DFCSA_DT_F32); }

// ============================================================================ rotary positions
// Pair j of a token's channels turns by angle = position[axis(j)] * freq(j):
//   (a, b) -> (a cos - b sin, a sin + b cos);  the backward turns by the negative angle.
// Halves: pair j = channels (j, P + j); interleaved: (2j, 2j + 1); channels from 2P on pass through.
// Positions reach 10^6 and more, where an fp32 angle is off by 0.06: the turn position * freq / 2 pi is
// formed in fp64 and reduced to its fraction exactly; only the fraction goes on in fp32.
//
// A workgroup takes tok tokens: it computes their P angles once into LDS and applies them to all heads,
// V channels of both halves per item.  Bound by the read and the write of q and k: 16384 tokens of 16 + 4
// heads of 128 in bf16 (168 MB) take 29 us, 5.8 TB/s.
struct RotaryArgs {
  const void* src[2];
  void* dst[2];
  int64_t sb[2], sn[2], sh[2];   // source strides in elements (the destination is contiguous)
  int heads[2];
  int B, N, D, P, A, tok, interleaved;
  const void* pos;
  int pos64;
  int64_t pb, pn, pa;
  float sign;
  double turns[DFCSA_ROTARY_MAX_PAIRS];   // freq / 2 pi
  unsigned char axis[DFCSA_ROTARY_MAX_PAIRS];
};

constexpr int kRotLds = 256;   // angles (cos, sin) a workgroup holds

template <typename T, int V>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  __shared__ __attribute__((aligned(16))) float cs[kRotLds], sn[kRotLds];
  const int64_t tokens = (int64_t)a.B * a.N, t0 = group2() * a.tok;
  if (t0 >= tokens) return;
  const int nt = (int)min((int64_t)a.tok, tokens - t0);
  for (int e = threadIdx.x; e < nt * a.P; e += 256) {
    const int tl = e / a.P, j = e - tl * a.P;
    const int64_t t = t0 + tl, b = t / a.N, n = t - b * a.N;
    const int64_t at = b * a.pb + n * a.pn + a.axis[j] * a.pa;
    const double p = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int*)a.pos)[at];
    double turn = p * a.turns[j];
    turn -= rint(turn);
    float s, c;
    sincospif(2.0f * (float)turn, &s, &c);
    cs[e] = c;
    sn[e] = s * a.sign;
  }
  __syncthreads();
  const int heads = a.heads[0] + a.heads[1];
  // items of one head: rotated groups of V pairs (halves) or V/2 pairs (interleaved), then the tail
  const int rot = V == 1 ? a.P : (a.interleaved ? 2 * a.P / V : a.P / V);
  const int items = rot + (a.D - 2 * a.P) / V;
  const int per = heads * items;
  for (int e = threadIdx.x; e < nt * per; e += 256) {
    const int tl = e / per, q = e - tl * per, hh = q / items, it = q - hh * items;
    const int64_t t = t0 + tl, b = t / a.N, n = t - b * a.N;
    const int which = hh >= a.heads[0], h = hh - (which ? a.heads[0] : 0);
    const T* src = (const T*)a.src[which] + b * a.sb[which] + n * a.sn[which] + h * a.sh[which];
    T* dst = (T*)a.dst[which] + (t * a.heads[which] + h) * a.D;
    const float* c = cs + tl * a.P;
    const float* s = sn + tl * a.P;
    if constexpr (V == 1) {
      using E = ElemTraits<T>;
      if (it < rot) {
        const int ia = a.interleaved ? 2 * it : it, ib = a.interleaved ? 2 * it + 1 : a.P + it;
        const float va = E::to_f(src[ia]), vb = E::to_f(src[ib]);
        dst[ia] = E::from_f(va * c[it] - vb * s[it]);
        dst[ib] = E::from_f(va * s[it] + vb * c[it]);
      } else {
        const int i = 2 * a.P + it - rot;
        dst[i] = src[i];
      }
    } else {
      float va[8];
      if (it >= rot) {
        const int i = 2 * a.P + (it - rot) * 8;
        load8<T>(src + i, va);
        store8<T>(dst + i, va);
      } else if (a.interleaved) {
        load8<T>(src + it * 8, va);
        float o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float ck = c[it * 4 + k], sk = s[it * 4 + k];
          o[2 * k] = va[2 * k] * ck - va[2 * k + 1] * sk;
          o[2 * k + 1] = va[2 * k] * sk + va[2 * k + 1] * ck;
        }
        store8<T>(dst + it * 8, o);
      } else {
        float vb[8], oa[8], ob[8];
        load8<T>(src + it * 8, va);
        load8<T>(src + a.P + it * 8, vb);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float ck = c[it * 8 + k], sk = s[it * 8 + k];
          oa[k] = va[k] * ck - vb[k] * sk;
          ob[k] = va[k] * sk + vb[k] * ck;
        }
        store8<T>(dst + it * 8, oa);
        store8<T>(dst + a.P + it * 8, ob);
      }
    }
  }
}

template <typename T>
void launch_rotary(const RotaryArgs& a, bool vec, hipStream_t st) {
  const int64_t tokens = (int64_t)a.B * a.N;
  const dim3 grid = grid2((tokens + a.tok - 1) / a.tok);
  if (vec) hipLaunchKernelGGL((rotary_kernel<T, 8>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((rotary_kernel<T, 1>), grid, dim3(256), 0, st, a);
}

}  // namespace

extern "C" {

int dfcsa_rms_fwd(int dtype, int rdtype, int rows, int C, const void* x, const void* res, const float* w, float eps,
                  void* y, void* r, float* rstd, void* stream) {
  if (!norm_shape_ok(rows, C) || !types_ok(dtype, rdtype) || !x || !res || !w || !y || !r || !eps_ok(eps)) return DFCSA_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DFCSA_DT_F32) return launch_fwd<float, float, false>(rows, C, x, res, w, eps, y, r, rstd, nullptr, nullptr, C, st);
  if (rdtype == DFCSA_DT_F32) return launch_fwd<bf16_t, float, false>(rows, C, x, res, w, eps, y, r, rstd, nullptr, nullptr, C, st);
  return launch_fwd<bf16_t, bf16_t, false>(rows, C, x, res, w, eps, y, r, rstd, nullptr, nullptr, C, st);
}

int dfcsa_rms_fwd_q8(int dtype, int rdtype, int rows, int C, int group, const void* x, const void* res, const float* w,
                     float eps, void* y8, float* scales, void* r, void* stream) {
  if (!norm_shape_ok(rows, C) || !types_ok(dtype, rdtype) || !x || !res || !w || !y8 || !scales || !r || !eps_ok(eps)) return DFCSA_EINVAL;
  if (group == 0) group = C;
  if (group != C && ((group != 32 && group != 64 && group != 128) || C % group)) return DFCSA_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DFCSA_DT_F32) return launch_fwd<float, float, true>(rows, C, x, res, w, eps, nullptr, r, nullptr, y8, scales, group, st);
  if (rdtype == DFCSA_DT_F32) return launch_fwd<bf16_t, float, true>(rows, C, x, res, w, eps, nullptr, r, nullptr, y8, scales, group, st);
  return launch_fwd<bf16_t, bf16_t, true>(rows, C, x, res, w, eps, nullptr, r, nullptr, y8, scales, group, st);
}

int64_t dfcsa_rms_bwd_work_floats(int rows, int C) {
  return norm_shape_ok(rows, C) ? (int64_t)bwd_groups(rows, C) * C : 0;
}

int dfcsa_rms_bwd(int dtype, int rdtype, int rows, int C, const void* dy, const void* dr, const void* r,
                  const float* rstd, const float* w, void* dx, void* dres, float* dw, float* work,
                  int64_t work_floats, void* stream) {
  if (!norm_shape_ok(rows, C) || !types_ok(dtype, rdtype) || !dy || !r || !rstd || !w) return DFCSA_EINVAL;
  if (dw && (!work || work_floats < dfcsa_rms_bwd_work_floats(rows, C))) return DFCSA_EINVAL;
  float* part = dw ? work : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DFCSA_DT_F32) return launch_bwd<float, float>(rows, C, dy, dr, r, rstd, w, dx, dres, part, dw, st);
  if (rdtype == DFCSA_DT_F32) return launch_bwd<bf16_t, float>(rows, C, dy, dr, r, rstd, w, dx, dres, part, dw, st);
  return launch_bwd<bf16_t, bf16_t>(rows, C, dy, dr, r, rstd, w, dx, dres, part, dw, st);
}

int dfcsa_dequant_q8(int dtype, int64_t rows, int C, int group, const void* y8, const float* scales, void* out,
                     void* stream) {
  if (rows <= 0 || C < 8 || C % 8 || C > kNormMaxC || !y8 || !scales || !out) return DFCSA_EINVAL;
  if (group == 0) group = C;
  if (group != C && ((group != 32 && group != 64 && group != 128) || C % group)) return DFCSA_EINVAL;
  const int gsh = group == C ? -1 : (group == 32 ? 2 : group == 64 ? 3 : 4);
  const int64_t n8 = rows * (C / 8), blocks = (n8 + 255) / 256;
  if (blocks > 0x7fffffff) return DFCSA_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DFCSA_DT_F32)
    hipLaunchKernelGGL((dequant_kernel<float>), grid2(blocks), dim3(256), 0, st, n8, C / 8, gsh, C / group,
                       (const uint2*)y8, scales, (float*)out);
  else if (dtype == DFCSA_DT_BF16)
    hipLaunchKernelGGL((dequant_kernel<bf16_t>), grid2(blocks), dim3(256), 0, st, n8, C / 8, gsh,
                       C / group, (const uint2*)y8, scales, (bf16_t*)out);
  else
    return DFCSA_EINVAL;
  DFCSA_CHECK_LAUNCH();
  return 0;
}

int dfcsa_rotary(const dfcsa_rotary_desc* d, void* stream) {
  if (!d || (d->dtype != DFCSA_DT_F32 && d->dtype != DFCSA_DT_BF16)) return DFCSA_EINVAL;
  if (d->B <= 0 || d->N <= 0 || d->D <= 0 || d->D > 1024 || d->npairs <= 0 || d->npairs > DFCSA_ROTARY_MAX_PAIRS ||
      2 * d->npairs > d->D || d->naxes <= 0 || d->naxes > 4 || !d->positions || !d->turns || !d->axis)
    return DFCSA_EINVAL;
  const int64_t tokens = (int64_t)d->B * d->N;
  if (tokens > 0x7fffffff) return DFCSA_EINVAL;
  RotaryArgs a;
  const int es = d->dtype == DFCSA_DT_F32 ? 4 : 2;
  bool vec = d->D % 8 == 0 && (d->interleaved ? (2 * d->npairs) % 8 == 0 : d->npairs % 8 == 0);
  int heads = 0;
  for (int i = 0; i < 2; ++i) {
    a.src[i] = d->src[i];
    a.dst[i] = d->dst[i];
    a.sb[i] = d->src_sb[i];
    a.sn[i] = d->src_sn[i];
    a.sh[i] = d->src_sh[i];
    a.heads[i] = d->heads[i];
    if (d->heads[i] < 0 || d->heads[i] > 4096 || (d->heads[i] > 0 && (!d->src[i] || !d->dst[i]))) return DFCSA_EINVAL;
    heads += d->heads[i];
    if (d->heads[i] > 0 && ((uintptr_t)d->src[i] % 16 || (uintptr_t)d->dst[i] % 16 || (d->src_sb[i] * es) % 16 ||
                            (d->src_sn[i] * es) % 16 || (d->src_sh[i] * es) % 16))
      vec = false;
  }
  if (heads == 0) return DFCSA_EINVAL;
  a.B = d->B; a.N = d->N; a.D = d->D; a.P = d->npairs; a.A = d->naxes; a.interleaved = d->interleaved;
  a.pos = d->positions; a.pos64 = d->pos64; a.pb = d->pos_sb; a.pn = d->pos_sn; a.pa = d->pos_sa;
  a.sign = d->inverse ? -1.f : 1.f;
  for (int j = 0; j < d->npairs; ++j) {
    a.turns[j] = d->turns[j];
    a.axis[j] = d->axis[j];
    if (d->axis[j] >= d->naxes) return DFCSA_EINVAL;
  }
  // one angle per thread of a workgroup, as far as that leaves a workgroup for each CU
  int tok = 256 / a.P;
  tok = tok < 1 ? 1 : tok;
  while (tok > 1 && ((tokens + tok - 1) / tok < 512 || (int64_t)heads * a.D * tok > 1 << 28)) tok >>= 1;
  a.tok = tok;
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == DFCSA_DT_F32) launch_rotary<float>(a, vec, st);
  else launch_rotary<bf16_t>(a, vec, st);
  DFCSA_CHECK_LAUNCH();
  return 0;
}

}  // extern "C"
