// Microscaled (OCP MX) rows and their operators: quant_mx.hip (quantise, norm + quantise, read back), gemm_mx.hip (products).
//
// A quantised matrix of n_rows x k:  every row in whole groups of 128 columns (kp = k rounded up to 128, the added columns zero)
//   elements  e2m1: kp / 2 bytes a row, the lower column in the low half of a byte;   e4m3: kp bytes a row
//   scales    kp / 32 bytes a row, the biased exponents X + 127 of the blocks of 32 columns (E8M0);  0xff: the block is NaN
// so that the four scales of 128 columns -- one K step of the scaled MFMA -- are one aligned 32-bit word.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

enum { MX_E2M1 = 0, MX_E4M3 = 1, MX_ROW_E4M3 = 2 };
enum { MX_DT_BF16 = 0, MX_DT_F16 = 1, MX_DT_F32 = 2 };
enum { MX_NORM_RMS = 0, MX_NORM_LAYER = 1 };
#define MX_NORM_MAX_K 16384             // widest row of the norm: 512 threads hold it in registers, 32 values each

static inline int mx_kp(int k) { return (k + 127) / 128 * 128; }
// Whether a product quantises its rows itself, one launch instead of two, in every workgroup again: up to 16 rows, and up to 64 while the
// workgroups of 16 x 16 results are two a CU or fewer (4096 x 1024, e4m3, GPU time of 1 / 32 rows: 3.9 / 6.0 us, in two launches 5.0 / 6.6;
// 5120 x 1280, 24 rows: 9.8 against 7.5) -- and fewer than 2^26 weights, whose sweep would be held up by it (12 800 x 5120, 1 / 16 rows:
// 15 / 16 us against 14 / 21; 8192 x 8192: 21 / 26 against 12 / 18).
static inline bool mx_takes_values(int m, int n, int k) {
  return (m <= 16 || (m <= 64 && (long)((m + 15) / 16) * ((n + 15) / 16) <= 512)) && (long)n * k < 1l << 26;
}

struct MxNormParams {
  const void* x; long ld_x;             // [n_rows] rows of k elements, ld_x elements apart
  const void* resid; long ld_r;         // NULL: none
  const float* gamma; const float* beta;   // [k]; beta NULL: 0
  void* h;                              // [n_rows][k] x + resid as it is stored (NULL with resid NULL)
  uint8_t* q; void* scale;              // MX_ROW_E4M3: scale is float [n_rows]
  long n_rows; int k, kp;
  int norm, fmt;
  float eps;
};

struct MxGemmParams {
  const uint8_t* a; const uint8_t* a_scale;   // [M] quantised rows
  const uint8_t* w; const uint8_t* w_scale;   // [N] e2m1 rows
  int M, N, nk;                               // nk: K steps of 128 columns
  const float* bias;                          // [N] or NULL
  const void* resid;                          // [M][N] of the output's type, or NULL; may be `out`
  void* out;                                  // [M][N]
  int act, out_dtype;                         // CE_ACT_* or -1; MX_DT_*
  bool streamed;                              // set by ce_mx_gemm: 16-bit results leave with the streaming cache policy
};

#ifdef __HIPCC__
typedef __attribute__((ext_vector_type(2))) uint32_t mx_u32x2_t;
// eight values times `inv` (a power of two, or the row's 448 / max) to e4m3 / e2m1; v_cvt_pk_fp8_f32 does not saturate, the e2m1 one does
__device__ __forceinline__ mx_u32x2_t mx_to_e4m3(const float* v, float inv) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = __builtin_amdgcn_fmed3f(v[i] * inv, -448.0f, 448.0f);
  int a = 0, b = 0;
  a = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], a, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], a, true);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], b, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], b, true);
  return mx_u32x2_t{(uint32_t)a, (uint32_t)b};
}
__device__ __forceinline__ uint32_t mx_to_e2m1(const float* v, float inv) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0] * inv, v[1] * inv, 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2] * inv, v[3] * inv, 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4] * inv, v[5] * inv, 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6] * inv, v[7] * inv, 1.0f, 3);
  return w;
}

// The scale byte and 1 / 2^X of a block whose largest magnitude has the bits `m`.
__device__ __forceinline__ uint32_t mx_block_scale(uint32_t m, int emax, float& inv) {
  if (m >= 0x7f800000u) { inv = 0.0f; return 0xffu; }
  int e = (int)(m >> 23) - 127;
  if (m < 0x00800000u) e = m ? (31 - __clz((int)m)) - 149 : -127;   // subnormal maxima: fp32 inputs only
  const int x = max(e - emax, -127);                                 // <= 125
  inv = __uint_as_float((uint32_t)(127 - x) << 23);                  // 2^-X, X in [-127, 125]: a normal float
  return (uint32_t)(x + 127);
}
#endif

hipError_t ce_mx_quant(const void* x, int dtype, long n_rows, int k, long ld_x, int fmt, uint8_t* q, uint8_t* scale, hipStream_t stream);
hipError_t ce_mx_dequant(const uint8_t* q, const void* scale, int fmt, long n_rows, int k, void* out, int out_dtype, hipStream_t stream);
hipError_t ce_mx_norm(const MxNormParams& p, int dtype, hipStream_t stream);
hipError_t ce_mx_gemm(MxGemmParams p, int a_fmt, hipStream_t stream);
// mx_takes_values: the rows of p.a are quantised from x inside
hipError_t ce_mx_gemm_values(const MxGemmParams& p, const void* x, int dtype, long ld_x, int k, int fmt, hipStream_t stream);
