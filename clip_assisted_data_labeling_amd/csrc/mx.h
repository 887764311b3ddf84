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
#define MX_NORM_MAX_K 16384             // widest row of the norm: 1024 threads hold it in registers, 16 values each

static inline int mx_kp(int k) { return (k + 127) / 128 * 128; }

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

hipError_t ce_mx_quant(const void* x, int dtype, long n_rows, int k, long ld_x, int fmt, uint8_t* q, uint8_t* scale, hipStream_t stream);
hipError_t ce_mx_dequant(const uint8_t* q, const void* scale, int fmt, long n_rows, int k, void* out, int out_dtype, hipStream_t stream);
hipError_t ce_mx_norm(const MxNormParams& p, int dtype, hipStream_t stream);
hipError_t ce_mx_gemm(MxGemmParams p, int a_fmt, hipStream_t stream);
