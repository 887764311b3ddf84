// Rows to microscaled blocks (mx.h), on their own or as the end of a norm, and back.
//
//   block of 32 values v:   X = clamp(floor(log2 max|v|) - emax, -127, 127)      emax = 2 (e2m1), 8 (e4m3)
//                           element = round_to_nearest_even(v / 2^X), at most the format's largest value (6, 448)
//   (the OCP MX conversion).  max|v| and its exponent come from the bits of the floats, v / 2^X is exact, so a call rounds each value
//   once and its codes are those of the formula in any precision.  A block that holds an infinity or a NaN gets the scale 0xff and
//   zero elements: NaN wherever it is read.
//
// All of these kernels move each byte once and are bound by HBM (quantise: 2 bytes in, 0.53 / 1.03 out per value of a 16-bit row).
// A thread owns 8 consecutive columns -- 16 bytes of a 16-bit row -- and keeps them from row to row, so nothing is divided in the loop;
// four neighbouring threads share a block (its maximum: two DPP steps), sixteen share the scale word of 128 columns.
#include "common.h"
#include "mx.h"

namespace {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
// rows start at any element: the vector accesses promise no more than the element's own alignment (gfx950 takes them all)
struct __attribute__((packed, aligned(2))) Pack16 { u32x4_t v; };
struct __attribute__((packed, aligned(4))) Pack32 { u32x4_t v[2]; };

template <typename T> struct Elem;
template <> struct Elem<__bf16> {
  static __device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ void load8(const __bf16* p, float (&v)[8]) {
    const u32x4_t r = ((const Pack16*)p)->v;
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(r[i] << 16); v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ void store8(__bf16* p, const float (&v)[8]) {
    Pack16 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    *(Pack16*)p = r;
  }
};
template <> struct Elem<_Float16> {
  static __device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ void load8(const _Float16* p, float (&v)[8]) {
    const f16x8_t r = __builtin_bit_cast(f16x8_t, ((const Pack16*)p)->v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)r[i];
  }
  static __device__ __forceinline__ void store8(_Float16* p, const float (&v)[8]) {
    f16x8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)v[i];
    ((Pack16*)p)->v = __builtin_bit_cast(u32x4_t, r);
  }
};
template <> struct Elem<float> {
  static __device__ __forceinline__ float to_f32(float v) { return v; }
  static __device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const Pack32 r = *(const Pack32*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.v[i >> 2][i & 3]);
  }
  static __device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    Pack32 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i >> 2][i & 3] = __float_as_uint(v[i]);
    *(Pack32*)p = r;
  }
};

// the columns c .. c + 7 of a row of k; zeros behind its end
template <typename T>
__device__ __forceinline__ void load_cols(const T* row, int c, int k, float (&v)[8]) {
  if (c + 8 <= k) { Elem<T>::load8(row + c, v); return; }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = c + i < k ? Elem<T>::to_f32(row[c + i]) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void store_cols(T* row, int c, int k, const float (&v)[8]) {
  if (c + 8 <= k) { Elem<T>::store8(row + c, v); return; }
#pragma unroll
  for (int i = 0; i < 8; ++i) if (c + i < k) row[c + i] = (T)v[i];
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
#define DPP_XOR1 0xB1            // quad_perm [1,0,3,2]
#define DPP_XOR2 0x4E            // quad_perm [2,3,0,1]
#define DPP_HALF_MIRROR 0x141    // lane i of 8 -> 7 - i
#define DPP_MIRROR 0x140         // lane i of 16 -> 15 - i

__device__ __forceinline__ uint32_t abs_bits8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// eight values times `inv` (a power of two, or the row's 448 / max) to e4m3 / e2m1; v_cvt_pk_fp8_f32 does not saturate, the e2m1 one does
__device__ __forceinline__ u32x2_t to_e4m3(const float (&v)[8], float inv) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = __builtin_amdgcn_fmed3f(v[i] * inv, -448.0f, 448.0f);
  int a = 0, b = 0;
  a = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], a, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], a, true);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], b, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], b, true);
  return u32x2_t{(uint32_t)a, (uint32_t)b};
}
__device__ __forceinline__ uint32_t to_e2m1(const float (&v)[8], float inv) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0] * inv, v[1] * inv, 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2] * inv, v[3] * inv, 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4] * inv, v[5] * inv, 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6] * inv, v[7] * inv, 1.0f, 3);
  return w;
}

// The scale byte and 1 / 2^X of a block whose largest magnitude has the bits `m`.
__device__ __forceinline__ uint32_t block_scale(uint32_t m, int emax, float& inv) {
  if (m >= 0x7f800000u) { inv = 0.0f; return 0xffu; }
  int e = (int)(m >> 23) - 127;
  if (m < 0x00800000u) e = m ? (31 - __clz((int)m)) - 149 : -127;   // subnormal maxima: fp32 inputs only
  const int x = max(e - emax, -127);                                 // <= 125
  inv = __uint_as_float((uint32_t)(127 - x) << 23);                  // 2^-X, X in [-127, 125]: a normal float
  return (uint32_t)(x + 127);
}

// Quantises the thread's 8 columns; the 16 threads of 128 columns take part together.  Non-finite blocks: inf * 0 would be NaN, so
// their elements are cleared.
__device__ __forceinline__ void store_block(const float (&v)[8], int fmt, uint8_t* q_row, uint8_t* s_row, int c) {
  uint32_t m = abs_bits8(v);
  m = max(m, dpp<DPP_XOR1>(m));
  m = max(m, dpp<DPP_XOR2>(m));
  float inv;
  const uint32_t x = block_scale(m, fmt == MX_E2M1 ? 2 : 8, inv);
  uint32_t word = x << (8 * ((threadIdx.x >> 2) & 3));
  word |= dpp<DPP_HALF_MIRROR>(word);
  word |= dpp<DPP_MIRROR>(word);
  if (fmt == MX_E2M1) {
    const uint32_t w = to_e2m1(v, inv);
    *(uint32_t*)(q_row + c / 2) = x == 0xffu ? 0u : w;
  } else {
    u32x2_t w = to_e4m3(v, inv);
    if (x == 0xffu) w = u32x2_t{0u, 0u};
    *(u32x2_t*)(q_row + c) = w;
  }
  if ((threadIdx.x & 15) == 0) *(uint32_t*)(s_row + c / 32) = word;
}

// Threads 0 .. active - 1 own (row, 8 columns) pairs, row by row; active is a multiple of kp / 8, so that a step of the loop moves
// every thread by `step` = active / (kp / 8) whole rows.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_quant_kernel(const T* __restrict__ x, long n_rows, int k, int kp, long ld_x, uint8_t* __restrict__ q,
                                                       uint8_t* __restrict__ scale, long active, long step) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= active) return;                       // in whole groups of 16 threads
  const int per_row = kp >> 3;
  const long row0 = id / per_row;
  const int c = (int)(id - row0 * per_row) * 8;
  const size_t q_ld = FMT == MX_E2M1 ? kp / 2 : kp, s_ld = kp / 32;
  for (long row = row0; row < n_rows; row += step) {
    float v[8];
    load_cols<T>(x + row * ld_x, c, k, v);
    store_block(v, FMT, q + (size_t)row * q_ld, scale + (size_t)row * s_ld, c);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void mx_dequant_kernel(const uint8_t* __restrict__ q, const void* __restrict__ scale, int fmt, long n_rows, int k,
                                                         int kp, T* __restrict__ out, long active, long step) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= active) return;
  const int per_row = kp >> 3;
  const long row0 = id / per_row;
  const int c = (int)(id - row0 * per_row) * 8;
  const size_t q_ld = fmt == MX_E2M1 ? kp / 2 : kp;
  for (long row = row0; row < n_rows; row += step) {
    float s;
    if (fmt == MX_ROW_E4M3) s = ((const float*)scale)[row];
    else {
      const uint32_t x = ((const uint8_t*)scale)[(size_t)row * (kp / 32) + c / 32];
      s = x == 0xffu ? __builtin_nanf("") : x ? __uint_as_float(x << 23) : 0x1p-127f;
    }
    float v[8];
    const uint8_t* src = q + (size_t)row * q_ld;
    if (fmt == MX_E2M1) {
      const uint32_t w = *(const uint32_t*)(src + c / 2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // the 3-bit magnitude as a float: 0.5 is the format's one subnormal, codes 2 .. 7 are (1 + m / 2) 2^(e - 1)
        const uint32_t code = (w >> (4 * i)) & 15u, mag = code & 7u;
        const float a = mag < 2u ? 0.5f * (float)mag : __uint_as_float((126u << 23) + (mag << 22));
        v[i] = (code & 8u ? -a : a) * s;
      }
    } else {
      const u32x2_t w = *(const u32x2_t*)(src + c);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 0) * s;
        v[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 1) * s;
        v[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 2) * s;
        v[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 3) * s;
      }
    }
    if (c < k) store_cols<T>(out + (size_t)row * k, c, k, v);
  }
}

// ---- norm --------------------------------------------------------------------------------------------------------------------------
//   h = x + resid (rounded to the rows' type, as it is stored);  RMS: y = h / sqrt(mean(h^2) + eps) * gamma + beta,
//   LAYER: the same of h - mean(h);  then y in blocks, or in e4m3 with one scale a row, max|y| / 448
// The row stays in the registers of NT threads, CH chunks of 8 columns each.  Sums and the factor are held in 64 bits: fp64 runs
// at the rate of single fp32 operations here and hides behind the row's bytes, squares cannot overflow, and y is rounded to fp32 once,
// so that codes differ from the formula's only where y lies within 2^-24 of a rounding border.
template <int NT>
__device__ __forceinline__ double sum_over(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (NT > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) v += red[i];
    __syncthreads();
  }
  return v;
}
template <int NT>
__device__ __forceinline__ uint32_t max_over(uint32_t v, uint32_t* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  if constexpr (NT > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) v = max(v, red[i]);
    __syncthreads();
  }
  return v;
}

// NT = 64: four rows a workgroup, one wave each, no barrier;  NT > 64: a row a workgroup
template <typename T, int NT, int CH>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void mx_norm_kernel(const MxNormParams p) {
  __shared__ double red[NT / 64];
  const int t = NT == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const long per_step = NT == 64 ? (long)gridDim.x * 4 : (long)gridDim.x;
  long row = NT == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x;
  for (; row < p.n_rows; row += per_step) {
    float v[CH][8];
#pragma unroll
    for (int i = 0; i < CH; ++i) load_cols<T>((const T*)p.x + row * p.ld_x, (i * NT + t) * 8, p.k, v[i]);
    if (p.resid) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = (i * NT + t) * 8;
        float r[8];
        load_cols<T>((const T*)p.resid + row * p.ld_r, c, p.k, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = (float)(T)(v[i][j] + r[j]);
        if (c < p.k) store_cols<T>((T*)p.h + (size_t)row * p.k, c, p.k, v[i]);
      }
    }
    double mean = 0;
    if (p.norm == MX_NORM_LAYER) {
      double s = 0;
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s += (double)v[i][j];
      mean = sum_over<NT>(s, red) / p.k;
    }
    double ss = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double d = (i * NT + t) * 8 + j < p.k ? (double)v[i][j] - mean : 0.0;
        ss = fma(d, d, ss);
      }
    const double factor = 1.0 / sqrt(sum_over<NT>(ss, red) / p.k + (double)p.eps);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = (i * NT + t) * 8;
      float g[8], b[8];
      load_cols<float>(p.gamma, c, p.k, g);
      if (p.beta) load_cols<float>(p.beta, c, p.k, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double y = ((double)v[i][j] - mean) * factor * (double)g[j] + (p.beta ? (double)b[j] : 0.0);
        v[i][j] = c + j < p.k ? (float)y : 0.0f;
      }
      m = max(m, abs_bits8(v[i]));
    }
    if (p.fmt == MX_ROW_E4M3) {
      m = max_over<NT>(m, (uint32_t*)red);
      const float amax = __uint_as_float(m);
      const bool fine = m < 0x7f800000u;
      const double inv = m && fine ? 448.0 / (double)amax : 0.0;   // a zero row: scale 0.  In 64 bits: 448 / max may pass fp32's range
      if (t == 0) ((float*)p.scale)[row] = fine ? amax / 448.0f : __builtin_nanf("");
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = (i * NT + t) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = (float)((double)v[i][j] * inv);
        u32x2_t w = to_e4m3(v[i], 1.0f);
        if (!fine) w = u32x2_t{0u, 0u};
        if (c < p.kp) *(u32x2_t*)(p.q + (size_t)row * p.kp + c) = w;
      }
    } else {
      const size_t q_ld = p.fmt == MX_E2M1 ? p.kp / 2 : p.kp;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = (i * NT + t) * 8;
        if (c < p.kp) store_block(v[i], p.fmt, p.q + (size_t)row * q_ld, (uint8_t*)p.scale + (size_t)row * (p.kp / 32), c);
      }
    }
  }
}

// how many threads own (row, 8 columns) pairs, at most `blocks` workgroups of 256, and how many rows a step moves them
struct Spread { long active, step; int blocks; };
Spread spread_rows(long n_rows, int kp, int blocks) {
  const long per_row = kp / 8;
  long rows = (long)blocks * 256 / per_row;
  if (rows < 1) rows = 1;
  if (rows > n_rows) rows = n_rows;
  return Spread{rows * per_row, rows, (int)((rows * per_row + 255) / 256)};
}
constexpr int STREAM_BLOCKS = 256 * 16;

template <typename T>
void launch_quant(const T* x, long n_rows, int k, long ld_x, int fmt, uint8_t* q, uint8_t* scale, hipStream_t stream) {
  const int kp = mx_kp(k);
  const Spread s = spread_rows(n_rows, kp, STREAM_BLOCKS);
  if (fmt == MX_E2M1) hipLaunchKernelGGL((mx_quant_kernel<T, MX_E2M1>), dim3(s.blocks), dim3(256), 0, stream, x, n_rows, k, kp, ld_x, q, scale, s.active, s.step);
  else hipLaunchKernelGGL((mx_quant_kernel<T, MX_E4M3>), dim3(s.blocks), dim3(256), 0, stream, x, n_rows, k, kp, ld_x, q, scale, s.active, s.step);
}

template <typename T>
hipError_t launch_norm(const MxNormParams& p, hipStream_t stream) {
  const long waves = (p.n_rows + 3) / 4;
  const int g4 = (int)(waves < 256 * 8 ? waves : 256 * 8), g1 = (int)(p.n_rows < 256 * 8 ? p.n_rows : 256 * 8);
#define NORM_LAUNCH(NT, CH) hipLaunchKernelGGL((mx_norm_kernel<T, NT, CH>), dim3(NT == 64 ? g4 : g1), dim3(NT == 64 ? 256 : NT), 0, stream, p)
  if (p.kp <= 512) NORM_LAUNCH(64, 1);
  else if (p.kp <= 1024) NORM_LAUNCH(64, 2);
  else if (p.kp <= 2048) NORM_LAUNCH(64, 4);
  else if (p.kp <= 4096) NORM_LAUNCH(256, 2);
  else if (p.kp <= 8192) NORM_LAUNCH(256, 4);
  else if (p.kp <= MX_NORM_MAX_K) NORM_LAUNCH(512, 4);
  else return hipErrorInvalidValue;
#undef NORM_LAUNCH
  return hipGetLastError();
}

}  // namespace

hipError_t ce_mx_quant(const void* x, int dtype, long n_rows, int k, long ld_x, int fmt, uint8_t* q, uint8_t* scale, hipStream_t stream) {
  if (dtype == MX_DT_BF16) launch_quant((const __bf16*)x, n_rows, k, ld_x, fmt, q, scale, stream);
  else if (dtype == MX_DT_F16) launch_quant((const _Float16*)x, n_rows, k, ld_x, fmt, q, scale, stream);
  else launch_quant((const float*)x, n_rows, k, ld_x, fmt, q, scale, stream);
  return hipGetLastError();
}

hipError_t ce_mx_dequant(const uint8_t* q, const void* scale, int fmt, long n_rows, int k, void* out, int out_dtype, hipStream_t stream) {
  const int kp = mx_kp(k);
  const Spread s = spread_rows(n_rows, kp, STREAM_BLOCKS);
#define DEQUANT_LAUNCH(T) hipLaunchKernelGGL((mx_dequant_kernel<T>), dim3(s.blocks), dim3(256), 0, stream, q, scale, fmt, n_rows, k, kp, (T*)out, s.active, s.step)
  if (out_dtype == MX_DT_BF16) DEQUANT_LAUNCH(__bf16);
  else if (out_dtype == MX_DT_F16) DEQUANT_LAUNCH(_Float16);
  else DEQUANT_LAUNCH(float);
#undef DEQUANT_LAUNCH
  return hipGetLastError();
}

hipError_t ce_mx_norm(const MxNormParams& p, int dtype, hipStream_t stream) {
  return dtype == MX_DT_BF16 ? launch_norm<__bf16>(p, stream) : dtype == MX_DT_F16 ? launch_norm<_Float16>(p, stream) : launch_norm<float>(p, stream);
}
