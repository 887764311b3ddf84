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
#include <type_traits>

#include "common.h"
#include "mx.h"

namespace {

// 65 792 x 4096 of bf16 to e2m1 and back, 682 MB each, one pass behind the other: 116 us (5.9 TB/s) and 136 us (5.0).  Quantising wants many short
// workgroups -- one row a thread and step: 256 workgroups a CU 116 us, 64 131; four rows in flight and 16 a CU 154 --, reading back few long
// ones: four rows in flight and 8 a CU 136 us, 16 a CU 141, one row 174 (e4m3: 159, 164, 151).
constexpr int QUANT_BLOCKS = 256 * 256, DEQUANT_ROWS = 4, DEQUANT_BLOCKS = 256 * 8;

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
typedef mx_u32x2_t u32x2_t;
// rows start at any element: the vector accesses promise no more than the element's own alignment (gfx950 takes them all)
struct __attribute__((packed, aligned(2))) Pack16 { u32x4_t v; };
struct __attribute__((packed, aligned(4))) Pack32 { u32x4_t v[2]; };

// Eight values of a row as they lie in memory: 16 or 32 bytes
template <typename T> struct Raw { u32x4_t v[sizeof(T) / 2]; };
template <typename T> using Pack = typename std::conditional<sizeof(T) == 2, Pack16, Pack32>::type;

// The columns c .. c + 7 of a row of k; zeros behind its end.  WHOLE: k % 8 == 0, no chunk is partly behind it.
template <typename T, bool WHOLE>
__device__ __forceinline__ Raw<T> load_raw(const T* row, int c, int k) {
  Raw<T> r;
  if (c + 8 <= k) {
    const Pack<T> p = *(const Pack<T>*)(row + c);
    __builtin_memcpy(&r, &p, sizeof(r));
    return r;
  }
  r = Raw<T>{};
  if constexpr (!WHOLE) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = c + i < k ? row[c + i] : (T)0.0f;
    __builtin_memcpy(&r, e, sizeof(r));
  }
  return r;
}
__device__ __forceinline__ void values_of(const Raw<__bf16>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(r.v[0][i] << 16); v[2 * i + 1] = __uint_as_float(r.v[0][i] & 0xffff0000u); }
}
__device__ __forceinline__ void values_of(const Raw<_Float16>& r, float (&v)[8]) {
  const f16x8_t h = __builtin_bit_cast(f16x8_t, r.v[0]);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
}
__device__ __forceinline__ void values_of(const Raw<float>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.v[i >> 2][i & 3]);
}
template <typename T>
__device__ __forceinline__ Raw<T> raw_of(const float (&v)[8]) {
  Raw<T> r;
  if constexpr (std::is_same<T, __bf16>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[0][i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  } else {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = (T)v[i];
    __builtin_memcpy(&r, e, sizeof(r));
  }
  return r;
}
template <typename T, bool WHOLE>
__device__ __forceinline__ void store_raw(T* row, int c, int k, const Raw<T>& r) {
  if (c + 8 <= k) {
    Pack<T> p;
    __builtin_memcpy(&p, &r, sizeof(r));
    *(Pack<T>*)(row + c) = p;
  } else if constexpr (!WHOLE) {
    T e[8];
    __builtin_memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < 8; ++i) if (c + i < k) row[c + i] = e[i];
  }
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

// Quantises the thread's 8 columns; the 16 threads of 128 columns take part together.  Non-finite blocks: inf * 0 would be NaN, so
// their elements are cleared.
__device__ __forceinline__ void store_block(const float (&v)[8], int fmt, uint8_t* q_row, uint8_t* s_row, int c) {
  uint32_t m = abs_bits8(v);
  m = max(m, dpp<DPP_XOR1>(m));
  m = max(m, dpp<DPP_XOR2>(m));
  float inv;
  const uint32_t x = mx_block_scale(m, fmt == MX_E2M1 ? 2 : 8, inv);
  uint32_t word = x << (8 * ((threadIdx.x >> 2) & 3));
  word |= dpp<DPP_HALF_MIRROR>(word);
  word |= dpp<DPP_MIRROR>(word);
  if (fmt == MX_E2M1) {
    const uint32_t w = mx_to_e2m1(v, inv);
    *(uint32_t*)(q_row + c / 2) = x == 0xffu ? 0u : w;
  } else {
    u32x2_t w = mx_to_e4m3(v, inv);
    if (x == 0xffu) w = u32x2_t{0u, 0u};
    *(u32x2_t*)(q_row + c) = w;
  }
  if ((threadIdx.x & 15) == 0) *(uint32_t*)(s_row + c / 32) = word;
}

// Threads 0 .. active - 1 own (row, 8 columns) pairs, row by row; active is a multiple of kp / 8, so that a step of the loop moves
// every thread by `step` = active / (kp / 8) whole rows.
template <typename T, int FMT, bool WHOLE>
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
    values_of(load_raw<T, WHOLE>(x + row * ld_x, c, k), v);
    store_block(v, FMT, q + (size_t)row * q_ld, scale + (size_t)row * s_ld, c);
  }
}

__device__ __forceinline__ float scale_value(uint32_t x) {
  return x == 0xffu ? __builtin_nanf("") : x ? __uint_as_float(x << 23) : 0x1p-127f;
}

// (row, 8 columns) pairs as above; the elements and scales of DEQUANT_ROWS rows are in flight
template <typename T, int FMT, bool WHOLE>
__global__ __launch_bounds__(256) void mx_dequant_kernel(const uint8_t* __restrict__ q, const void* __restrict__ scale, long n_rows, int k, int kp,
                                                         T* __restrict__ out, long active, long step) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= active) return;
  const int per_row = kp >> 3;
  const long row0 = id / per_row;
  const int c = (int)(id - row0 * per_row) * 8;
  if (c >= k) return;
  const size_t q_ld = FMT == MX_E2M1 ? kp / 2 : kp;
  auto load = [&](long row, u32x2_t& w, float& s) {
    const uint8_t* src = q + (size_t)row * q_ld;
    if constexpr (FMT == MX_E2M1) w = u32x2_t{*(const uint32_t*)(src + c / 2), 0u};
    else w = *(const u32x2_t*)(src + c);
    if constexpr (FMT == MX_ROW_E4M3) s = ((const float*)scale)[row];
    else s = scale_value(((const uint8_t*)scale)[(size_t)row * (kp / 32) + c / 32]);
  };
  // A block's scale is a power of two and the product exact; with a row's it has up to 28 bits, which reach 16 through an fp32 value rounded to
  // odd: of the two neighbours the one whose last bit is set.
  auto times = [](float a, float s) {
    const float p = a * s;
    if constexpr (FMT != MX_ROW_E4M3 || sizeof(T) == 4) return p;
    const float rest = __builtin_fmaf(a, s, -p);
    uint32_t b = __float_as_uint(p);
    if ((rest > 0.0f || rest < 0.0f) && !(b & 1u)) b += (rest > 0.0f) == (p > 0.0f) ? 1u : 0xffffffffu;
    return __uint_as_float(b);
  };
  auto store = [&](long row, u32x2_t w, float s) {
    float v[8];
    if constexpr (FMT == MX_E2M1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // the 3-bit magnitude as a float: 0.5 is the format's one subnormal, codes 2 .. 7 are (1 + m / 2) 2^(e - 1)
        const uint32_t code = (w[0] >> (4 * i)) & 15u, mag = code & 7u;
        const float a = mag < 2u ? 0.5f * (float)mag : __uint_as_float((126u << 23) + (mag << 22));
        v[i] = (code & 8u ? -a : a) * s;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[4 * i] = times(__builtin_amdgcn_cvt_f32_fp8((int)w[i], 0), s);
        v[4 * i + 1] = times(__builtin_amdgcn_cvt_f32_fp8((int)w[i], 1), s);
        v[4 * i + 2] = times(__builtin_amdgcn_cvt_f32_fp8((int)w[i], 2), s);
        v[4 * i + 3] = times(__builtin_amdgcn_cvt_f32_fp8((int)w[i], 3), s);
      }
    }
    store_raw<T, WHOLE>(out + (size_t)row * k, c, k, raw_of<T>(v));
  };
  constexpr int R = DEQUANT_ROWS;
  long row = row0;
  for (; row + (R - 1) * step < n_rows; row += R * step) {
    u32x2_t w[R];
    float s[R];
#pragma unroll
    for (int i = 0; i < R; ++i) load(row + i * step, w[i], s[i]);
#pragma unroll
    for (int i = 0; i < R; ++i) store(row + i * step, w[i], s[i]);
  }
  for (; row < n_rows; row += step) {
    u32x2_t w;
    float s;
    load(row, w, s);
    store(row, w, s);
  }
}

// ---- norm --------------------------------------------------------------------------------------------------------------------------
//   h = x + resid (rounded to the rows' type, as it is stored);  RMS: y = h / sqrt(mean(h^2) + eps) * gamma + beta,
//   LAYER: the same of h - mean(h);  then y in blocks, or in e4m3 with one scale a row, max|y| / 448
// The row stays in the registers of NT threads, CH chunks of 8 columns each, and so does its share of gamma; the next row's loads are
// under way while a row is worked on.  Sums, the factor and y are formed in 64 bits, so that no square overflows and beta may cancel; y
// reaches its few bits through an fp32 value rounded to ODD, so that codes are those of the 64-bit y and no value next to a border
// between two of them is rounded twice.
// 65 536 rows of 1024, bf16, with residual and h: 470 MB in 93 us (5.1 TB/s, what a copy reaches); of 1280 without: 254 MB in 76 us.
__device__ __forceinline__ float to_odd(double d) {
  // what lies below the 23 bits of an fp32 mantissa, as their last bit: the conversion has nothing left to round (normal results)
  const uint64_t b = (uint64_t)__double_as_longlong(d);
  const uint32_t lo = (uint32_t)b, sticky = (lo & 0x1fffffffu) + 0x1fffffffu;
  return (float)__longlong_as_double((long long)((b >> 32 << 32) | ((lo | sticky) & 0xe0000000u)));
}

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
__device__ __forceinline__ double max_over(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o));
  if constexpr (NT > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) v = fmax(v, red[i]);
    __syncthreads();
  }
  return v;
}

// NT = 64: four rows a workgroup, one wave each, no barrier;  NT > 64: a row a workgroup
template <typename T, int NT, int CH, bool WHOLE, bool ROW>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void mx_norm_kernel(const MxNormParams p) {
  __shared__ double red[NT / 64];
  const int t = NT == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const long per_step = NT == 64 ? (long)gridDim.x * 4 : (long)gridDim.x;
  long row = NT == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x;
  if (row >= p.n_rows) return;                                                  // NT = 64: a whole wave; else the workgroup
  float g[CH][8];
#pragma unroll
  for (int i = 0; i < CH; ++i) values_of(load_raw<float, WHOLE>(p.gamma, (i * NT + t) * 8, p.k), g[i]);
  auto inside = [&](int i, int j) { return (i * NT + t) * 8 + (WHOLE ? 0 : j) < p.k; };
  Raw<T> rx[CH], rr[CH];
  auto fetch = [&](long r) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      rx[i] = load_raw<T, WHOLE>((const T*)p.x + r * p.ld_x, (i * NT + t) * 8, p.k);
      if (p.resid) rr[i] = load_raw<T, WHOLE>((const T*)p.resid + r * p.ld_r, (i * NT + t) * 8, p.k);
    }
  };
  fetch(row);
  for (; row < p.n_rows; row += per_step) {
    float v[CH][8];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      values_of(rx[i], v[i]);
      if (p.resid) {
        float r[8];
        values_of(rr[i], r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += r[j];
        const Raw<T> h = raw_of<T>(v[i]);
        store_raw<T, WHOLE>((T*)p.h + (size_t)row * p.k, (i * NT + t) * 8, p.k, h);
        values_of(h, v[i]);
      }
    }
    if (row + per_step < p.n_rows) fetch(row + per_step);
    double mean = 0;
    const bool layer = p.norm == MX_NORM_LAYER;
    if (layer) {
      double s = 0;
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s += (double)v[i][j];
      mean = sum_over<NT>(s, red) / p.k;
    }
    double ss = 0;
    if (layer) {
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const double d = inside(i, j) ? (double)v[i][j] - mean : 0.0;
          ss = fma(d, d, ss);
        }
    } else {
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fma((double)v[i][j], (double)v[i][j], ss);   // (behind the row: zeros)
    }
    const double factor = 1.0 / sqrt(sum_over<NT>(ss, red) / p.k + (double)p.eps);
    auto y_of = [&](int i, double (&y)[8]) {
      auto of = [&](int j) {
        float gj = g[i][j];
        asm("" : "+v"(gj));                                                     // kept as fp32: its conversion is not to leave the loop
        return (double)gj * factor;
      };
      if (layer) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = inside(i, j) ? ((double)v[i][j] - mean) * of(j) : 0.0;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (double)v[i][j] * of(j);
      }
      if (p.beta) {
        float b[8];
        values_of(load_raw<float, WHOLE>(p.beta, (i * NT + t) * 8, p.k), b);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] += (double)b[j];
      }
    };
    if constexpr (ROW) {
      double most = 0, bad = 0;                                                 // fmax drops NaN: it is kept in `bad`
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        double y[8];
        y_of(i, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) { most = fmax(most, fabs(y[j])); bad = y[j] - y[j] == 0.0 ? bad : 1.0; }
      }
      most = max_over<NT>(most, red);
      bad = max_over<NT>(bad, red);
      const bool fine = bad == 0.0 && most <= 3.4028234663852886e38;            // what fp32 holds
      const double inv = fine && most > 0.0 ? 448.0 / most : 0.0;               // a zero row: scale 0
      if (t == 0) ((float*)p.scale)[row] = fine ? (float)(most / 448.0) : __builtin_nanf("");
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = (i * NT + t) * 8;
        double y[8];
        y_of(i, y);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = to_odd(y[j] * inv);
        u32x2_t w = mx_to_e4m3(f, 1.0f);
        if (!fine) w = u32x2_t{0u, 0u};
        if (c < p.kp) *(u32x2_t*)(p.q + (size_t)row * p.kp + c) = w;
      }
    } else {
      const size_t q_ld = p.fmt == MX_E2M1 ? p.kp / 2 : p.kp;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = (i * NT + t) * 8;
        double y[8];
        y_of(i, y);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = to_odd(y[j]);
        if (c < p.kp) store_block(f, p.fmt, p.q + (size_t)row * q_ld, (uint8_t*)p.scale + (size_t)row * (p.kp / 32), c);
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

template <typename T>
void launch_quant(const T* x, long n_rows, int k, long ld_x, int fmt, uint8_t* q, uint8_t* scale, hipStream_t stream) {
  const int kp = mx_kp(k);
  const Spread s = spread_rows(n_rows, kp, QUANT_BLOCKS);
#define QUANT_LAUNCH(F, W) hipLaunchKernelGGL((mx_quant_kernel<T, F, W>), dim3(s.blocks), dim3(256), 0, stream, x, n_rows, k, kp, ld_x, q, scale, s.active, s.step)
  if (k % 8 == 0) { if (fmt == MX_E2M1) QUANT_LAUNCH(MX_E2M1, true); else QUANT_LAUNCH(MX_E4M3, true); }
  else { if (fmt == MX_E2M1) QUANT_LAUNCH(MX_E2M1, false); else QUANT_LAUNCH(MX_E4M3, false); }
#undef QUANT_LAUNCH
}

template <typename T>
void launch_dequant(const uint8_t* q, const void* scale, int fmt, long n_rows, int k, T* out, hipStream_t stream) {
  const int kp = mx_kp(k);
  const Spread s = spread_rows(n_rows, kp, DEQUANT_BLOCKS);
#define DEQUANT_LAUNCH(F) \
  if (k % 8 == 0) hipLaunchKernelGGL((mx_dequant_kernel<T, F, true>), dim3(s.blocks), dim3(256), 0, stream, q, scale, n_rows, k, kp, out, s.active, s.step); \
  else hipLaunchKernelGGL((mx_dequant_kernel<T, F, false>), dim3(s.blocks), dim3(256), 0, stream, q, scale, n_rows, k, kp, out, s.active, s.step)
  if (fmt == MX_E2M1) { DEQUANT_LAUNCH(MX_E2M1); }
  else if (fmt == MX_E4M3) { DEQUANT_LAUNCH(MX_E4M3); }
  else { DEQUANT_LAUNCH(MX_ROW_E4M3); }
#undef DEQUANT_LAUNCH
}

// Threads of a row: as few as hold it in 16 .. 32 values each, since every wave more costs a turn of the sums (65 536 rows of 1280 / 2048 / 4096 /
// 8192, bf16 to e4m3: 76 / 118 / 212 / 387 us; in 256 / 256 / 512 / 1024 threads of 8 values 8 to 70 % more; 512 columns in 64 threads 36
// us, in 256 97).  Up to NORM_FEW rows of up to 2048 the latency of one row counts: 256 threads of 8 values (one row of 1280 3.8 us instead
// of 4.4, 1024 rows 5.3 both, 2048 rows 7.3 instead of 6.1).
constexpr long NORM_FEW = 1024;
template <typename T, bool WHOLE>
hipError_t launch_norm(const MxNormParams& p, hipStream_t stream) {
  const long waves = (p.n_rows + 3) / 4;
  const int g4 = (int)(waves < 256 * 8 ? waves : 256 * 8), g1 = (int)(p.n_rows < 256 * 8 ? p.n_rows : 256 * 8);
#define NORM_LAUNCH(NT, CH) \
  if (p.fmt == MX_ROW_E4M3) hipLaunchKernelGGL((mx_norm_kernel<T, NT, CH, WHOLE, true>), dim3(NT == 64 ? g4 : g1), dim3(NT == 64 ? 256 : NT), 0, stream, p); \
  else hipLaunchKernelGGL((mx_norm_kernel<T, NT, CH, WHOLE, false>), dim3(NT == 64 ? g4 : g1), dim3(NT == 64 ? 256 : NT), 0, stream, p)
  if (p.kp <= 512) { NORM_LAUNCH(64, 1); }
  else if (p.kp <= 1024) { NORM_LAUNCH(64, 2); }
  else if (p.kp <= 2048 && p.n_rows <= NORM_FEW) { NORM_LAUNCH(256, 1); }
  else if (p.kp <= 1536) { NORM_LAUNCH(64, 3); }
  else if (p.kp <= 2048) { NORM_LAUNCH(128, 2); }
  else if (p.kp <= 4096) { NORM_LAUNCH(256, 2); }
  else if (p.kp <= 8192) { NORM_LAUNCH(256, 4); }
  else if (p.kp <= MX_NORM_MAX_K) { NORM_LAUNCH(512, 4); }
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
  if (out_dtype == MX_DT_BF16) launch_dequant(q, scale, fmt, n_rows, k, (__bf16*)out, stream);
  else if (out_dtype == MX_DT_F16) launch_dequant(q, scale, fmt, n_rows, k, (_Float16*)out, stream);
  else launch_dequant(q, scale, fmt, n_rows, k, (float*)out, stream);
  return hipGetLastError();
}

template <typename T>
static hipError_t norm_of(const MxNormParams& p, hipStream_t stream) {
  return p.k % 8 == 0 ? launch_norm<T, true>(p, stream) : launch_norm<T, false>(p, stream);
}
hipError_t ce_mx_norm(const MxNormParams& p, int dtype, hipStream_t stream) {
  return dtype == MX_DT_BF16 ? norm_of<__bf16>(p, stream) : dtype == MX_DT_F16 ? norm_of<_Float16>(p, stream) : norm_of<float>(p, stream);
}
