// Products of microscaled rows (mx.h):  out[M][N] = act(A . W^T + bias) (+ resid),  A e2m1 or e4m3, W e2m1, on the scaled MFMA
// v_mfma_scale_f32_16x16x128_f8f6f4, which takes both operands as they lie -- 4 or 8 bits -- and applies the block scales itself.
// Sums are fp32; the result is rounded once, after bias, activation and residual.
//
// Operand maps (measured):  a lane holds row l & 15 of an operand and, g = l >> 4, of its 128 columns
//   4 bits: columns 32 g .. 32 g + 31 (16 bytes);      8 bits: 16 g .. 16 g + 15 and 64 + 16 g .. 64 + 16 g + 15 (two times 16 bytes)
// the scale byte of lane (row, g) is that of the BLOCK 32 g .. 32 g + 31 in both cases; `opsel` picks the byte of the lane's word.
// W is the MFMA's first operand, so a lane's four results are four neighbouring columns n of one row m.
//
// What the matrix pipe keeps (measured): the products of 8 neighbouring columns are added at fixed point, cut below 2^(E - 13), 2^E the
// largest product's power of two; everything above that is added in fp32.  e2m1 products span 6 bits and lose nothing.  e4m3 x e2m1
// products span 22, so that two large ones of opposite signs among eight neighbours would leave nothing of the six others.  They are
// therefore added in two BANDS of the e4m3 codes, exponent fields 8 .. 15 and 0 .. 7: a band's products span at most 14 bits (2^-3 .. 2^11,
// 2^-10 .. 2^3), so nothing is cut, at two MFMAs a fragment pair.
//
// Persistent tiles of BM x BN, WM x WN waves.  LDS holds two stages of 128-byte rows of A (256 columns of e2m1, 128 of e4m3) and two of W
// (256 columns), brought in by LDS-DMA in pieces of 8 rows x 128 bytes.  The walk is one sequence of stages over all of a workgroup's
// tiles: a stage's last fragments are in registers before its end, so the barrier there frees its buffer, the stage after next is asked
// for -- of this tile or the next one --, the next stage's first fragments are read under the last products, and a finished tile's
// results leave straight from the registers while the next tile's rows arrive.  The 16-byte chunk c of tile row r lies at chunk
// c ^ ((r >> 1) & 7) of its row, by the choice of the DMA's source addresses, so that 16 lanes reading one chunk column of 16 rows meet no
// bank twice.  K steps are counted in pairs; an odd number of them is led by an empty one, which e4m3 rows skip and e2m1 rows multiply
// with both scales at 2^-127: products below 2^-240, zeros in fp32.
// Scales come by periods of 512 columns, the four words of a row turned round -- word g: the scales of block g in the period's four K
// steps -- so that a lane holds the scales of 16 rows and a period in ONE word.
//
// Measured, 256 x 256 tiles:  16 384 x 8192 -> 4096  e2m1 271 us (4.05 PFLOP/s), e4m3 784 us (1.4, of MFMAs in two bands 2.8);  65 536 x 4096
// -> 1024 in e2m1 160 us (3.4), 65 792 in e4m3 434 us (1.27); the bare instruction reaches 7.7 and 4.5.  Over long e4m3 rows the matrix pipe is
// busy 0.53 of the time, and waits at the barriers and for a stage's first fragments; one MFMA a fragment pair, whose sums the cut above
// would hold in 14 bits, took 402 and 242 us.  A short K is bound by the way out: 65 792 x 1024 -> 4096 in e2m1 with QuickGELU 255 us, 539 MB
// of results.
#include <type_traits>

#include "common.h"
#include "mx.h"

namespace {

enum { A_E2M1 = 0, A_E4M3 = 1 };   // the kernels' A

typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;

// Activations of fp32 arguments, whose errors are relative to their results -- into the tails, down to 2^-120.  WIDE: a few units of fp32's last
// bit; else 2^-14, well under what 16 bits round, for whole tiles' 16-bit results (65 792 x 1024 -> 4096 in e2m1, GELU: 322 us, without
// an activation 231; fp32 results 412 and 321).
//   QuickGELU(u) = u / (1 + exp(-1.702 u))
//   GELU(u) = u Phi(u):  q = Phi(-|u|) = exp(-u^2 / 2) g(|u|), and u q where u < 0, u (1 - q) elsewhere -- no difference of two numbers near 1.
//   g(x) = exp(x^2 / 2) erfc(x / sqrt 2) / 2 is taken as t P(t), t = 1 / (1 + p x), P fitted to the least relative error over x = 0 .. 13.5, where
//   q leaves fp32's normal numbers: degree 4, 2.9e-5; degree 8, 2.0e-8.  A fit of the absolute error of erfc (1.5e-7) is 2 % off at u = -4.5.
// An exponential of a large argument carries the argument's own rounding: WIDE has it in two floats.
// N vectors at once, stage by stage: the exp2s and rcps stand apart from their consumers, one branch for all.
template <bool WIDE, int N>
__device__ __forceinline__ void activate(f32x4_t (&v)[N], int act) {
#define EACH for (int j = 0; j < N; ++j) _Pragma("unroll") for (int e = 0; e < 4; ++e)
  constexpr float LN2 = 0.69314718056f;
  if (act == CE_ACT_QUICK_GELU) {
    constexpr float C = -2.4554669595930157f, C_LOW = (float)(-2.4554669595930157 - (double)C);      // -1.702 / ln 2
    f32x4_t t[N];
    if constexpr (WIDE) {
#pragma unroll
      EACH {
        const float x = __builtin_amdgcn_fmed3f(v[j][e], -200.0f, 200.0f), a = x * C;                // (beyond: 0 or infinity all the same)
        const float low = __builtin_fmaf(x, C_LOW, __builtin_fmaf(x, C, -a));
        t[j][e] = __builtin_amdgcn_exp2f(a) * __builtin_fmaf(low, LN2, 1.0f);
      }
    } else {
#pragma unroll
      EACH t[j][e] = __builtin_amdgcn_exp2f(v[j][e] * C);
    }
#pragma unroll
    EACH t[j][e] = __builtin_amdgcn_rcpf(1.0f + t[j][e]);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] *= t[j];
  } else if (act == CE_ACT_GELU_ERF) {
    constexpr float K = -0.72134752044448170f, K_LOW = (float)(-0.72134752044448170 - (double)K);    // -1 / (2 ln 2)
    constexpr float P[2][9] = {{0.14904113113880157f, 0.15792009234428406f, 0.08297396451234818f, 0.20104342699050903f, -0.09098529070615768f},
                               {0.13761912286281586f, 0.1380240023136139f, 0.11721379309892654f, 0.1119045689702034f, -0.03787023574113846f,
                                0.1876179724931717f, -0.2715700566768646f, 0.14548806846141815f, -0.028427232056856155f}};
    constexpr int DEGREE = WIDE ? 8 : 4;
    f32x4_t t[N], q[N];
#pragma unroll
    EACH t[j][e] = __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_fminf(__builtin_fabsf(v[j][e]), 20.0f), WIDE ? 0.345f : 0.375f, 1.0f));   // (beyond: q = 0)
#pragma unroll
    EACH {
      const float x = __builtin_fminf(__builtin_fabsf(v[j][e]), 20.0f), s = x * x, a = s * K;
      q[j][e] = __builtin_amdgcn_exp2f(a);
      if constexpr (WIDE) {
        const float low = __builtin_fmaf(s, K_LOW, __builtin_fmaf(__builtin_fmaf(x, x, -s), K, __builtin_fmaf(s, K, -a)));
        q[j][e] *= __builtin_fmaf(low, LN2, 1.0f);
      }
    }
#pragma unroll
    EACH {
      float g = P[WIDE][DEGREE];
#pragma unroll
      for (int i = DEGREE - 1; i >= 0; --i) g = __builtin_fmaf(g, t[j][e], P[WIDE][i]);
      const float phi = g * t[j][e] * q[j][e];
      v[j][e] *= v[j][e] < 0.0f ? phi : 1.0f - phi;
    }
  }
#undef EACH
}

// 64 lanes x 16 (4) bytes from base + offset (per lane) to the 1 KiB (256 bytes) of LDS at lds_addr.  Inline asm: behind the builtin every
// later LDS read would first wait for all pieces in flight.  m0 is written; nothing else here uses it.
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t b = (uint64_t)p;
  return (const uint8_t*)((uint64_t)__builtin_amdgcn_readfirstlane((unsigned)(b >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((unsigned)b));
}
__device__ __forceinline__ void dma16(const uint8_t* base, unsigned off, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(lds_addr) : "memory");
}
__device__ __forceinline__ void dma4(const uint8_t* base, unsigned off, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds_addr)) : "memory");
}
#define WAIT_LDS() asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory")
#define WAIT_ALL() asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory")
#define BARRIER() asm volatile("s_barrier" : : : "memory")

__device__ __forceinline__ float load_elem(const void* p, size_t i, int dtype) {
  if (dtype == MX_DT_F32) return ((const float*)p)[i];
  if (dtype == MX_DT_BF16) return bf16_to_f32(((const bf16_t*)p)[i]);
  return (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ void store_elem(void* p, size_t i, int dtype, float v) {
  if (dtype == MX_DT_F32) ((float*)p)[i] = v;
  else if (dtype == MX_DT_BF16) ((bf16_t*)p)[i] = f32_to_bf16(v);
  else ((_Float16*)p)[i] = (_Float16)v;
}

// rows of `out` start at any element: no more than its own alignment is promised
struct __attribute__((packed, aligned(2))) Pack16 { u32x4_t v; };
struct __attribute__((packed, aligned(4))) Pack32 { u32x4_t v; };
typedef uint32_t stream16_t __attribute__((ext_vector_type(4), aligned(2)));

// 8 values + 8 of 16 bits (r, if with), rounded once to 16 bits
__device__ __forceinline__ u32x4_t to_16bit(f32x4_t a, f32x4_t b, u32x4_t r, bool with, int dtype) {
  u32x4_t o;
  if (dtype == MX_DT_BF16) {
    if (with) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[2 * i] += __uint_as_float(r[i] << 16); a[2 * i + 1] += __uint_as_float(r[i] & 0xffff0000u);
        b[2 * i] += __uint_as_float(r[i + 2] << 16); b[2 * i + 1] += __uint_as_float(r[i + 2] & 0xffff0000u);
      }
    }
    o[0] = pack_bf16x2(a[0], a[1]); o[1] = pack_bf16x2(a[2], a[3]); o[2] = pack_bf16x2(b[0], b[1]); o[3] = pack_bf16x2(b[2], b[3]);
  } else {
    const f16x8_t s = __builtin_bit_cast(f16x8_t, r);
    f16x8_t h;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = (_Float16)(with ? a[i] + (float)s[i] : a[i]);
      h[i + 4] = (_Float16)(with ? b[i] + (float)s[i + 4] : b[i]);
    }
    o = __builtin_bit_cast(u32x4_t, h);
  }
  return o;
}
// The fragments of two neighbouring column groups (a: columns 4 g .. 4 g + 3 of the first, b: of the second) -> eight neighbouring columns
// a lane, from column 16 (g & 1) + 8 (g >> 1) of the pair: odd rows of 16 lanes change places between the two registers.
__device__ __forceinline__ void pair_columns(f32x4_t& a, f32x4_t& b) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[e]), __float_as_uint(b[e]), false, false);
    a[e] = __uint_as_float(s[0]);
    b[e] = __uint_as_float(s[1]);
  }
}

// the e4m3 codes with exponent fields 8 .. 15 (bit 6 of the byte), zeros in the place of the others
__device__ __forceinline__ i32x8_t high_band(i32x8_t v) {
  i32x8_t r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = (uint32_t)v[i], one = (w >> 6) & 0x01010101u;
    r[i] = (int)(w & ((one << 8) - one));
  }
  return r;
}

template <int CTRL>   // CTRL: quad_perm
__device__ __forceinline__ uint32_t dpp_quad(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }

template <int I, int N, typename F>
__device__ __forceinline__ void for_each_int(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    for_each_int<I + 1, N>(f);
  }
}

// NS: stages of A in LDS, NS - 1 of them under way.  DIRECT: scales come with each stage, a word a row and K step, and lanes read their byte
// of it; else by periods, turned.
template <int AF, int BM_, int BN_, int WM_, int WN_, int NS_, bool DIRECT_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int NS = NS_, NB = NS + 1;                      // NB: biases held -- a tile may be one stage, and that many are under way
  static constexpr bool DIRECT = DIRECT_;
  static constexpr int NW = WM * WN, THREADS = NW * 64;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;       // 16 x 16 fragments of a wave
  static constexpr int STEPS = AF == A_E2M1 ? 2 : 1;               // K steps of a stage of A
  static constexpr int A_BYTES = BM * 128, W_BYTES = BN * 128;
  static constexpr int A_PER = BM / 8 / NW, W_PER = BN / 8 / NW;   // DMA pieces a wave
  static constexpr int W_OFF = NS * A_BYTES, SC_OFF = W_OFF + NS * W_BYTES;
  static constexpr int SC_ROWS = BM + BN, SC_BYTES = SC_ROWS * (DIRECT ? 4 * STEPS : 16), SC_PER = SC_ROWS * 4 / THREADS;
  static constexpr int RAW_OFF = SC_OFF + (DIRECT ? NS : 2) * SC_BYTES, BIAS_OFF = RAW_OFF + (DIRECT ? 0 : SC_BYTES), LDS = BIAS_OFF + NB * BN * 4;
  static constexpr int YOUNGER = (NS - 2) * (A_PER + (AF == A_E2M1 ? W_PER : 0));   // DMAs at least that are younger than the next stage's
  static constexpr int STORES = FM * FN / 2;                       // of a wave's whole 16-bit tile, 16 bytes a lane each
  static_assert(A_PER >= W_PER && FM >= 2 && FN % 2 == 0 && A_PER * NW * 8 == BM && W_PER * NW * 8 == BN && NW % 2 == 0, "pieces");
  static_assert(BM % 64 == 0 && NS >= 2 && YOUNGER + STORES < 64, "ring");
  static_assert(DIRECT || NS == 2, "turned scales are one stage ahead");
  static_assert(SC_PER * THREADS == SC_ROWS * 4 && BM % (THREADS / 4) == 0 && BN % 64 == 0 && BN <= THREADS, "scales, bias");
  static_assert(LDS <= 163840, "LDS");
};

template <int AF, int BM, int BN, int WM, int WN, int NS, bool DIRECT>
__global__ __launch_bounds__(WM * WN * 64, 2) void mx_gemm_kernel(const MxGemmParams p) {
  using T = Tile<AF, BM, BN, WM, WN, NS, DIRECT>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w / WN, wn = w % WN;
  const int r16 = lane & 15, g = lane >> 4;
  const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)smem);

  // tile i of the walk: neighbouring workgroups of one XCD (i mod 8) walk neighbouring tiles, 8 row tiles deep
  const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
  const int nwg = tiles_m * tiles_n;
  auto tile_at = [&](int i, int& m0, int& n0) __attribute__((always_inline)) {
    const int q = nwg >> 3, rem = nwg & 7, xcd = i & 7, pos = i >> 3;
    const int bid = (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + pos;
    constexpr int GM = 8;
    const int first = bid / (GM * tiles_n) * GM, depth = min(tiles_m - first, GM), in_group = bid % (GM * tiles_n);
    m0 = (first + in_group % depth) * BM;
    n0 = in_group / depth * BN;
  };

  const int odd = p.nk & 1, steps = p.nk + odd;                     // K steps counted with the empty one in front
  const unsigned a_ld = (unsigned)p.nk * (AF == A_E2M1 ? 64u : 128u), w_ld = (unsigned)p.nk * 64u;

  // DMA of a piece: the lane's row is lane >> 3 of its 8, its chunk (lane & 7) ^ swizzle -- the same of all of a wave's pieces, whose
  // blocks of 8 rows are w, w + NW, ...: of w's parity.  Rows behind the matrix repeat its last one (their results are not stored).
  // Where the first step is the empty one (lead_in), its half of the row is read from the second one's columns.
  const int lr = lane >> 3, chunk = (lane & 7) ^ ((w & 1) << 2 | lr >> 1);
  const unsigned a_off = (unsigned)(w * 8 + lr) * a_ld + (unsigned)(chunk * 16), w_off = (unsigned)(w * 8 + lr) * w_ld + (unsigned)(chunk * 16);
  const unsigned lead = chunk < 4 ? 64u : 0u, low = (unsigned)(chunk * 16);
  const uint64_t a_hop = (uint64_t)(T::NW * 8) * a_ld, w_hop = (uint64_t)(T::NW * 8) * w_ld;
  auto issue = [&](const uint8_t* base, unsigned off, uint64_t hop, unsigned last, bool whole, bool lead_in, auto per_, unsigned dst) {
    constexpr int PER = decltype(per_)::value;       // last: the offset of the last row
    const unsigned plus = lead_in ? lead : 0u;
    if (whole) {
#pragma unroll
      for (int i = 0; i < PER; ++i) dma16(base + i * hop, off + plus, dst + (unsigned)(i * T::NW * 1024));
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) dma16(base, min(off - low + i * (unsigned)hop, last) + low + plus, dst + (unsigned)(i * T::NW * 1024));
    }
  };

  // Scales: four neighbouring lanes bring the period's four words of a row (16 rows an instruction: a lane a word of 64 rows would
  // touch four times the lines), rows of A first, then those of W; words before a row's first and behind its last one repeat a
  // neighbour.  They land as they are; each thread then turns the 4 x 4 bytes round with its neighbours -- words that its own wave has
  // brought -- and leaves its word where the fragments' lanes read it.
  const unsigned s_ld = (unsigned)p.nk * 4u;
  const int periods = (steps + 3) >> 2;
  auto issue_scales = [&](const uint8_t* a_at, const uint8_t* w_at, int a_rows, int w_rows, int period) __attribute__((always_inline)) {
    // (a_at, w_at: where the period's words of the tile's first rows would begin)
    unsigned j = (unsigned)(tid & 3) * 4u;
    if (period == 0 && odd) j = max(j, 4u);
    if (period == periods - 1 && (steps & 2)) j = min(j, 4u);
#pragma unroll
    for (int i = 0; i < T::SC_PER; ++i) {
      const bool is_a = i * (T::THREADS / 4) < BM;
      const int row = i * (T::THREADS / 4) + (tid >> 2) - (is_a ? 0 : BM);
      dma4(is_a ? a_at : w_at, (unsigned)min(row, (is_a ? a_rows : w_rows) - 1) * s_ld + j, lds0 + (unsigned)(T::RAW_OFF + (i * T::THREADS + w * 64) * 4));
    }
  };
  // (DIRECT) the words of a stage's steps from K step ks on: step by step, rows of A, then of W
  auto issue_words = [&](int m0, int n0, int ks, int buf) {
#pragma unroll
    for (int i = 0; i < (T::SC_ROWS * T::STEPS + T::THREADS - 1) / T::THREADS; ++i) {
      const int at = i * T::THREADS + w * 64;                       // the wave's first word
      if (at >= T::SC_ROWS * T::STEPS) break;
      const int step = at / T::SC_ROWS, row = at % T::SC_ROWS;
      const bool is_a = row < BM;
      const int r = row - (is_a ? 0 : BM) + lane;
      const int dst = T::SC_OFF + buf * T::SC_BYTES + at * 4;
      if (ks + step < 0) { *(uint32_t*)(smem + dst + lane * 4) = 0u; continue; }     // the empty step
      const uint8_t* base = uniform(is_a ? p.a_scale + (long)m0 * s_ld : p.w_scale + (long)n0 * s_ld) + (ks + step) * 4;
      dma4(base, (unsigned)min(r, (is_a ? p.M - m0 : p.N - n0) - 1) * s_ld, lds0 + (unsigned)dst);
    }
  };
  const uint32_t sc_sel = 0x01010101u * (uint32_t)(tid & 3) + 0x00000400u;      // bytes (own, own + 4) of a register pair
  auto turn_scales = [&](int period, int buf) __attribute__((always_inline)) {
    const uint32_t keep = AF == A_E2M1 && odd && period == 0 && (tid & 3) == 0 ? 0u : 0xffffffffu;   // the empty step's word
#pragma unroll
    for (int i = 0; i < T::SC_PER; ++i) {
      const int at = (i * T::THREADS + tid) * 4;
      const uint32_t s = *(volatile const uint32_t*)(smem + T::RAW_OFF + at) & keep;
      const uint32_t w0 = dpp_quad<0x00>(s), w1 = dpp_quad<0x55>(s), w2 = dpp_quad<0xAA>(s), w3 = dpp_quad<0xFF>(s);
      const uint32_t lo = __builtin_amdgcn_perm(w1, w0, sc_sel), hi = __builtin_amdgcn_perm(w3, w2, sc_sel);
      *(uint32_t*)(smem + T::SC_OFF + buf * T::SC_BYTES + at) = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
  };

  f32x4_t acc[T::FM][T::FN];
  const int rd = (r16 >> 3) * 1024 + (r16 & 7) * 128 + ((g ^ ((r16 >> 1) & 7)) << 4);   // chunk g of row r16; chunk g + 4: ^ 64
  // Fragments of a stage whose first K step is number `in_period` (0 .. 3) of its period
  auto load_w = [&](int wbuf, int in_period, int step, int j) __attribute__((always_inline)) {
    const int at = AF == A_E2M1 ? rd : rd ^ ((in_period & 1) * 64);
    const i32x4_t v = *(const i32x4_t*)(smem + T::W_OFF + wbuf * T::W_BYTES + (wn * T::FN + j) * 2048 + (at ^ (step * 64)));
    return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
  };
  auto load_a = [&](int abuf, int step, int i) __attribute__((always_inline)) {
    const char* at = smem + abuf * T::A_BYTES + (wm * T::FM + i) * 2048;
    if constexpr (AF != A_E2M1) {
      const i32x4_t lo = *(const i32x4_t*)(at + rd), hi = *(const i32x4_t*)(at + (rd ^ 64));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const i32x4_t v = *(const i32x4_t*)(at + (rd ^ (step * 64)));
      return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
    }
  };
  // (turned) the one or two bytes of a stage in the lane's word of the period;  (DIRECT) the byte of the stage's step
  auto load_scale = [&](int sbuf, int in_period, int step, int row16) __attribute__((always_inline)) -> uint32_t {
    const char* at = smem + T::SC_OFF + sbuf * T::SC_BYTES;
    if constexpr (DIRECT) return *(const uint8_t*)(at + (step * T::SC_ROWS + row16 * 16 + r16) * 4 + g);
    at += r16 * 16 + g * 4 + row16 * 256 + in_period;
    return T::STEPS == 2 ? (uint32_t)*(const uint16_t*)at : (uint32_t)*(const uint8_t*)at;
  };
  constexpr int FM = T::FM, FN = T::FN, N = T::STEPS * FM;          // N row fragments a stage

  // The stage to ask for next (f_): where its rows begin, its buffers, and which period it opens, whose scales are then to be turned
  const int v0 = AF == A_E2M1 ? 0 : odd;           // a tile's first stage's step (of e4m3 rows the empty step is no stage)
  int f_idx = blockIdx.x, f_v = v0, f_ab = 0, f_wb = 0, f_bias = 0, f_period = -1, f_m0, f_n0;
  auto after = [](int buf, int of) __attribute__((always_inline)) { return buf + 1 == of ? 0 : buf + 1; };
  const uint8_t *f_a, *f_w, *f_sa, *f_sw;
  auto fetch_tile = [&]() {
    tile_at(f_idx, f_m0, f_n0);
    f_v = v0;
    f_a = uniform(p.a + ((long)f_m0 * a_ld + (long)(v0 - odd) * (AF == A_E2M1 ? 64 : 128)));
    f_w = uniform(p.w + ((long)f_n0 * w_ld - odd * 64));
    f_sa = uniform(p.a_scale + ((long)f_m0 * s_ld - odd * 4));
    f_sw = uniform(p.w_scale + ((long)f_n0 * s_ld - odd * 4));
  };
  fetch_tile();
  auto fetch = [&]() {
    f_period = -1;
    if (f_idx >= nwg) return;
    const bool first = f_v == v0;
    issue(f_a, a_off, a_hop, (unsigned)(p.M - 1 - f_m0) * a_ld, f_m0 + BM <= p.M, AF == A_E2M1 && first && odd, std::integral_constant<int, T::A_PER>{},
          lds0 + (unsigned)(f_ab * T::A_BYTES + w * 1024));
    f_a += 128;
    if constexpr (DIRECT) issue_words(f_m0, f_n0, f_v - odd, f_ab);
    f_ab = after(f_ab, NS);
    if (AF == A_E2M1 || (f_v & 1) == 0 || first) {
      issue(f_w, w_off, w_hop, (unsigned)(p.N - 1 - f_n0) * w_ld, f_n0 + BN <= p.N, first && odd, std::integral_constant<int, T::W_PER>{},
            lds0 + (unsigned)(T::W_OFF + f_wb * T::W_BYTES + w * 1024));
      f_w += 128;
      f_wb = after(f_wb, NS);
    }
    if (!DIRECT && ((f_v & 3) == 0 || first)) {
      f_period = f_v >> 2;
      issue_scales(f_sa, f_sw, p.M - f_m0, p.N - f_n0, f_period);
      f_sa += 16;
      f_sw += 16;
    }
    if (first) {
      if (p.bias && w < BN / 64)
        dma4((const uint8_t*)p.bias, (unsigned)min(f_n0 + tid, p.N - 1) * 4u, lds0 + (unsigned)(T::BIAS_OFF + f_bias * BN * 4 + w * 256));
      f_bias = after(f_bias, T::NB);
    }
    f_v += T::STEPS;
    if (f_v >= steps) {
      f_idx += (int)gridDim.x;
      if (f_idx < nwg) fetch_tile();
    }
  };

  int idx = blockIdx.x, m0, n0;
  tile_at(idx, m0, n0);
  int ab = 0, wb = 0, sb = 0, bias_buf = 0;        // the buffers of the current stage, of the current tile's bias
  // What was asked for NS - 1 stages ago has to be there; younger are the stages since then (in the order of the asking), and a finished
  // tile's results, which need not have left.
  auto wait_stage = [&](bool stored) __attribute__((always_inline)) {
    const bool more = f_idx < nwg;                 // else fewer stages are younger
    if (NS > 2 && more && stored) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "i"(T::YOUNGER + T::STORES) : "memory");
    else if (NS > 2 && more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "i"(T::YOUNGER) : "memory");
    else if (stored) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "i"(T::STORES) : "memory");
    else WAIT_ALL();
  };
  bool stored = false;                             // the previous tile's STORES stores may still be on their way, issued after the loads
  // Out, straight from the registers: of two neighbouring fragments a lane gets eight neighbouring columns of a row (16 bits), of one
  // four (fp32); 16 rows x 64 bytes a store
  auto results = [&]() __attribute__((always_inline)) {
    int out_lane = lane;
    asm volatile("" : "+v"(out_lane));             // what follows from it is worked out here, not held in registers over the K loop
    const int row = m0 + wm * FM * 16 + (out_lane & 15), go = out_lane >> 4;
    const int col = n0 + wn * FN * 16;
    const bool whole = m0 + BM <= p.M && n0 + BN <= p.N;
    f32x4_t bs[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) bs[j] = p.bias ? *(const f32x4_t*)(smem + T::BIAS_OFF + bias_buf * BN * 4 + (wn * FN * 16 + j * 16 + go * 4) * 4) : f32x4_t{0, 0, 0, 0};
    if (whole && p.out_dtype != MX_DT_F32) {
      const int c8 = col + 16 * (go & 1) + 8 * (go >> 1);
      constexpr int HALF = FM / 2;                 // the residual of half the fragments at a time, asked for before any of them is stored
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4_t r[HALF][FN / 2];
        if (p.resid) {
#pragma unroll
          for (int i = 0; i < HALF; ++i)
#pragma unroll
            for (int j = 0; j < FN / 2; ++j)
              r[i][j] = ((const Pack16*)((const uint16_t*)p.resid + (size_t)(row + (h * HALF + i) * 16) * p.N + c8 + j * 32))->v;
        } else {
#pragma unroll
          for (int i = 0; i < HALF; ++i)
#pragma unroll
            for (int j = 0; j < FN / 2; ++j) r[i][j] = u32x4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
          f32x4_t u[FN];
#pragma unroll
          for (int j = 0; j < FN; ++j) u[j] = acc[h * HALF + i][j] + bs[j];
          activate<false>(u, p.act);
#pragma unroll
          for (int j = 0; j < FN / 2; ++j) {
            pair_columns(u[2 * j], u[2 * j + 1]);
            Pack16 o;
            o.v = to_16bit(u[2 * j], u[2 * j + 1], r[i][j], p.resid != nullptr, p.out_dtype);
            uint16_t* to = (uint16_t*)p.out + (size_t)(row + (h * HALF + i) * 16) * p.N + c8 + j * 32;
            if (p.streamed) __builtin_nontemporal_store((stream16_t)o.v, (stream16_t*)to);
            else *(Pack16*)to = o;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      stored = true;
    } else {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        f32x4_t u[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) u[j] = acc[i][j] + bs[j];
        activate<true>(u, p.act);
        const int m = row + i * 16;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int n = col + j * 16 + go * 4;
          if (m < p.M && n < p.N) {
            const size_t at = (size_t)m * p.N + n;
            if (p.out_dtype == MX_DT_F32 && n + 4 <= p.N) {
              if (p.resid) u[j] += __builtin_bit_cast(f32x4_t, ((const Pack32*)((const float*)p.resid + at))->v);
              Pack32 o;
              o.v = __builtin_bit_cast(u32x4_t, u[j]);
              *(Pack32*)((float*)p.out + at) = o;
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (n + e < p.N) store_elem(p.out, at + e, p.out_dtype, p.resid ? u[j][e] + load_elem(p.resid, at + e, p.out_dtype) : u[j][e]);
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

#pragma unroll
  for (int i = 0; i < NS - 1; ++i) fetch();
  wait_stage(false);
  if (!DIRECT) turn_scales(0, 0);
  WAIT_LDS();
  BARRIER();
  fetch();
  i32x8_t wf[2][FN], af[3];
  uint32_t sa[3], sw[FN], sw1[FN];               // sw1 (DIRECT): of the second step
  auto first_fragments = [&](int in_period, i32x8_t (&w_)[FN], i32x8_t& a0, i32x8_t& a1, uint32_t (&sw_)[FN], uint32_t& s0, uint32_t& s1) {
#pragma unroll
    for (int j = 0; j < FN; ++j) w_[j] = load_w(wb, in_period, 0, j);
    a0 = load_a(ab, 0, 0);
#pragma unroll
    for (int j = 0; j < FN; ++j) sw_[j] = load_scale(sb, in_period, 0, FM * WM + wn * FN + j);
    s0 = load_scale(sb, in_period, 0, wm * FM);
    a1 = load_a(ab, 0, 1);
    s1 = load_scale(sb, in_period, 0, wm * FM + 1);
  };
  while (true) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4_t{0, 0, 0, 0};
    int v = v0;
    bool last;
    first_fragments(v0 & 3, wf[0], af[0], af[1], sw, sa[0], sa[1]);   // (not held over the results' way out)
#pragma clang loop unroll(disable)
    do {
      auto products = [&](auto t_) {
        constexpr int t = decltype(t_)::value, step = t / FM, i = t % FM;
        __builtin_amdgcn_sched_barrier(0);
        i32x8_t a = af[t % 3];
        const int s = (int)sa[t % 3];
        constexpr int OP = DIRECT ? 0 : step;
        if constexpr (AF == A_E4M3) {
          const i32x8_t high = high_band(a);
          a ^= high;
#pragma unroll
          for (int j = 0; j < FN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[step][j], high, acc[i][j], 4, 0, OP, (int)(DIRECT && step ? sw1[j] : sw[j]), OP, s);
        }
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[step][j], a, acc[i][j], 4, AF != A_E2M1 ? 0 : 4, OP, (int)(DIRECT && step ? sw1[j] : sw[j]), OP, s);
        __builtin_amdgcn_sched_barrier(0);
      };
      for_each_int<0, N - 2>([&](auto t_) {
        constexpr int t = decltype(t_)::value, step = t / FM, i = t % FM;
        af[(t + 2) % 3] = load_a(ab, (t + 2) / FM, (t + 2) % FM);
        sa[(t + 2) % 3] = load_scale(sb, v & 3, (t + 2) / FM, wm * FM + (t + 2) % FM);
        if constexpr (step + 1 < T::STEPS) {
#pragma unroll
          for (int j = 0; j < FN; ++j)
            if (FM - FN + j == i || (FM < FN && i == 0)) {
              wf[1][j] = load_w(wb, 0, 1, j);
              if constexpr (DIRECT) sw1[j] = load_scale(sb, 0, 1, FM * WM + wn * FN + j);
            }
        }
        products(t_);
      });
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) asm volatile("" : "+v"(acc[i][j]));       // the products stay in front of the wait (no instruction)
      // All of the stage is in registers.
      wait_stage(stored);
      stored = false;
      last = v + T::STEPS >= steps;
      const int next_v = last ? v0 : v + T::STEPS;
      if (!DIRECT && f_period >= 0) turn_scales(f_period, sb ^ 1);
      WAIT_LDS();
      BARRIER();
      ab = after(ab, NS);
      if (AF == A_E2M1 || (next_v & 1) == 0 || last) wb = after(wb, NS);
      if (DIRECT) sb = ab;
      else if ((next_v & 3) == 0 || last) sb ^= 1;
      i32x8_t w_next[FN], a0, a1;
      uint32_t sw_next[FN], s0, s1;
      first_fragments(next_v & 3, w_next, a0, a1, sw_next, s0, s1);
      products(std::integral_constant<int, N - 2>{});
#pragma unroll
      for (int j = 0; j < FN; ++j) asm volatile("" : "+v"(acc[FM - 2][j]));    // (these stay in front of the asking)
      fetch();
      products(std::integral_constant<int, N - 1>{});
#pragma unroll
      for (int j = 0; j < FN; ++j) { wf[0][j] = w_next[j]; sw[j] = sw_next[j]; }
      af[0] = a0; af[1] = a1; sa[0] = s0; sa[1] = s1;
      v += T::STEPS;
    } while (!last);

    results();
    bias_buf = after(bias_buf, T::NB);
    idx += (int)gridDim.x;
    if (idx >= nwg) break;
    tile_at(idx, m0, n0);
  }
}

// ---- few rows -----------------------------------------------------------------------------------------------------------------------
// Few rows, or few columns: 16 columns n a workgroup, whose waves share K and add their sums up in LDS, in wave order.  Fragments come straight from
// memory -- each byte of W is read once, and there is nothing to wait for but that one read: a tile walk of the same product pays a
// memory latency a stage.  SRC: quantised rows (MX_E2M1 / MX_E4M3), or values of type T that the lanes quantise themselves, with the
// codes of clipenc_op_quant_mx; each workgroup does it again, so beyond MX_VALUE_COLS columns it has 64 of them (12 800 x 5120, one row in
// e4m3: 15 us instead of 26; 4096 x 1024, whose workgroups are then a quarter of the CUs: 5.9 instead of 3.9).
// One row of 8192 x 1664 takes 3.7 us from codes, whose 7 MB of weights are 1.4 us of HBM and whose launch and one trip to memory are the
// rest; 12 800 x 5120 (35 MB) 11 us, 3.2 TB/s.
struct MxFewParams {
  MxGemmParams g;
  const void* x; long ld_x; int k;                // values: [M] rows of k
};

// A lane's 32 values as they lie in a fragment -> its 4 or 8 words and its block's scale byte.  e2m1: block g, columns 32 g .. 32 g + 31.
// e4m3: 16 columns of block g / 2 and 16 of block 2 + g / 2, shared with lane ^ 16; the scale of block g comes from a lane that has it.
__device__ __forceinline__ i32x8_t quantise_fragment(const float (&v)[32], int fmt, uint32_t& scale) {
  uint32_t m[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 32; ++i) m[i >> 4] = max(m[i >> 4], __float_as_uint(v[i]) & 0x7fffffffu);
  i32x8_t q = {0, 0, 0, 0, 0, 0, 0, 0};
  if (fmt == MX_E2M1) {
    float inv;
    scale = mx_block_scale(max(m[0], m[1]), 2, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = mx_to_e2m1(v + 8 * i, inv);
      q[i] = scale == 0xffu ? 0 : (int)w;
    }
  } else {
    uint32_t x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float inv;
      x[h] = mx_block_scale(max(m[h], (uint32_t)__shfl_xor((int)m[h], 16)), 8, inv);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const mx_u32x2_t w = mx_to_e4m3(v + 16 * h + 8 * i, inv);
        q[4 * h + 2 * i] = x[h] == 0xffu ? 0 : (int)w[0];
        q[4 * h + 2 * i + 1] = x[h] == 0xffu ? 0 : (int)w[1];
      }
    }
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const uint32_t both = (uint32_t)__shfl((int)(x[0] | x[1] << 8), (lane & 15) + (g == 1 ? 32 : g == 2 ? 0 : 16 * g));
    scale = g < 2 ? both & 0xffu : both >> 8;
  }
  return q;
}
// the columns c .. c + 15 of a row of k as floats, zeros behind its end
template <typename T>
__device__ __forceinline__ void load16(const T* row, int c, int k, float* v) {
  constexpr int PACKS = sizeof(T) / 2 * 2, PER = 16 / PACKS;                       // 16-byte packs, values in each
  if (c + 16 <= k) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      u32x4_t r;
      if constexpr (sizeof(T) == 2) r = ((const Pack16*)(row + c + i * PER))->v;
      else r = ((const Pack32*)(row + c + i * PER))->v;
      if constexpr (std::is_same<T, __bf16>::value) {
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[8 * i + 2 * e] = __uint_as_float(r[e] << 16); v[8 * i + 2 * e + 1] = __uint_as_float(r[e] & 0xffff0000u); }
      } else if constexpr (std::is_same<T, _Float16>::value) {
        const f16x8_t h = __builtin_bit_cast(f16x8_t, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * i + e] = (float)h[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * i + e] = __uint_as_float(r[e]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = c + i < k ? (float)row[c + i] : 0.0f;
  }
}

constexpr int FEW_WAVES = 8, MX_VALUE_COLS = 8192;

// Scale words of U neighbouring K steps of a row, the lane's byte lowest
template <int U>
__device__ __forceinline__ void load_words(const uint8_t* scales, size_t step, int g, uint32_t (&s)[U]) {
  struct __attribute__((packed, aligned(4))) Words { uint32_t v[U]; };
  const Words w = *(const Words*)(scales + step * 4);
#pragma unroll
  for (int u = 0; u < U; ++u) s[u] = w.v[u] >> (8 * g);
}

// T = void: the rows are quantised;  AF: A_*;  MF, NF: 16-row and 16-column fragments;  U: K steps whose loads are under way together.  A wave has
// neighbouring steps, so that it reads whole lines of its rows and the scales of U steps at once.
template <typename T, int AF, int MF, int NF, int U>
__global__ __launch_bounds__(FEW_WAVES * 64) void mx_few_kernel(const MxFewParams fp) {
  const MxGemmParams& p = fp.g;
  constexpr bool VALUES = !std::is_same<T, void>::value;
  constexpr int FMT = AF == A_E2M1 ? MX_E2M1 : MX_E4M3;
  __shared__ __attribute__((aligned(16))) float sums[FEW_WAVES][MF * NF][256];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
  const int n0 = (blockIdx.z * gridDim.x + blockIdx.x) * (NF * 16), m0 = blockIdx.y * (MF * 16);
  if (n0 >= p.N) return;                                                           // (the whole workgroup)
  size_t w_row[NF], a_row[MF];                                                     // in K steps
#pragma unroll
  for (int j = 0; j < NF; ++j) w_row[j] = (size_t)min(n0 + j * 16 + r16, p.N - 1) * p.nk;
#pragma unroll
  for (int i = 0; i < MF; ++i) a_row[i] = (size_t)min(m0 + i * 16 + r16, p.M - 1) * (VALUES ? (size_t)fp.ld_x : (size_t)p.nk);
  f32x4_t acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4_t{0, 0, 0, 0};
  auto steps = [&](int ks, auto n_) {
    constexpr int C = decltype(n_)::value;
    i32x8_t wf[C][NF], af[C][MF];
    uint32_t sw[NF][C], sa[MF][C];
#pragma unroll
    for (int j = 0; j < NF; ++j) load_words<C>(p.w_scale, w_row[j] + ks, g, sw[j]);
#pragma unroll
    for (int i = 0; i < MF; ++i)
      if constexpr (!VALUES) load_words<C>(p.a_scale, a_row[i] + ks, g, sa[i]);
#pragma unroll
    for (int u = 0; u < C; ++u) {
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const i32x4_t v = *(const i32x4_t*)(p.w + (w_row[j] + ks + u) * 64 + g * 16);
        wf[u][j] = __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
      }
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        if constexpr (VALUES) {
          const T* x = (const T*)fp.x + a_row[i];
          const int c = (ks + u) * 128 + g * (FMT == MX_E2M1 ? 32 : 16);
          float f[32];
          load16(x, c, fp.k, f);
          load16(x, c + (FMT == MX_E2M1 ? 16 : 64), fp.k, f + 16);
          af[u][i] = quantise_fragment(f, FMT, sa[i][u]);
        } else if constexpr (AF == A_E2M1) {
          const i32x4_t q = *(const i32x4_t*)(p.a + (a_row[i] + ks + u) * 64 + g * 16);
          af[u][i] = __builtin_shufflevector(q, q, 0, 1, 2, 3, -1, -1, -1, -1);
        } else {
          const uint8_t* q = p.a + (a_row[i] + ks + u) * 128 + g * 16;
          const i32x4_t lo = *(const i32x4_t*)q, hi = *(const i32x4_t*)(q + 64);
          af[u][i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);                                             // the loads in front of the products
#pragma unroll
    for (int u = 0; u < C; ++u)
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        i32x8_t a = af[u][i];
        if constexpr (AF == A_E4M3) {
          const i32x8_t high = high_band(a);
          a ^= high;
#pragma unroll
          for (int j = 0; j < NF; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[u][j], high, acc[i][j], 4, 0, 0, (int)sw[j][u], 0, (int)sa[i][u]);
        }
#pragma unroll
        for (int j = 0; j < NF; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[u][j], a, acc[i][j], 4, AF != A_E2M1 ? 0 : 4, 0, (int)sw[j][u], 0, (int)sa[i][u]);
      }
  };
  const int per = (p.nk + waves - 1) / waves, end = min((w + 1) * per, p.nk);
  int ks = w * per;
  for (; ks + U <= end; ks += U) steps(ks, std::integral_constant<int, U>{});
  if constexpr (U > 1)
    for (; ks < end; ++ks) steps(ks, std::integral_constant<int, 1>{});
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) *(f32x4_t*)&sums[w][i * NF + j][r16 * 16 + g * 4] = acc[i][j];   // row r16, columns 4 g .. 4 g + 3
  __syncthreads();
  for (int t = tid; t < MF * NF * 256; t += blockDim.x) {
    const int m = m0 + t / (NF * 256) * 16 + (t & 255) / 16, n = n0 + t / 256 % NF * 16 + (t & 15);
    float v = 0.0f;
    for (int i = 0; i < waves; ++i) v += sums[i][t / 256][t & 255];
    if (m < p.M && n < p.N) {
      if (p.bias) v += p.bias[n];
      f32x4_t one[1] = {f32x4_t{v, v, v, v}};
      activate<true>(one, p.act);
      const size_t at = (size_t)m * p.N + n;
      store_elem(p.out, at, p.out_dtype, p.resid ? one[0][0] + load_elem(p.resid, at, p.out_dtype) : one[0][0]);
    }
  }
}

// A dimension of a launch holds fewer than 2^32 work items -- 2^23 workgroups of 512, 2^27 columns in 16s --, and more are cut off without an
// error: beyond FEW_COLUMNS workgroups the columns go on in the grid's third dimension (2^30 of them: 16 rows of it).
constexpr unsigned FEW_COLUMNS = 1u << 22;
template <typename T, int AF, int MF, int NF, int U>
hipError_t launch_few_u(const MxFewParams& p, hipStream_t stream) {
  const int waves = p.g.nk < FEW_WAVES ? p.g.nk : FEW_WAVES;
  const unsigned cols = (unsigned)((p.g.N + NF * 16 - 1) / (NF * 16)), x = cols < FEW_COLUMNS ? cols : FEW_COLUMNS;
  const dim3 grid(x, (unsigned)((p.g.M + MF * 16 - 1) / (MF * 16)), (cols + x - 1) / x);
  hipLaunchKernelGGL((mx_few_kernel<T, AF, MF, NF, U>), grid, dim3((unsigned)waves * 64), 0, stream, p);
  return hipGetLastError();
}
// as many steps under way as a wave has, and its registers hold
template <typename T, int AF, int MF, int NF = 1>
hipError_t launch_few(const MxFewParams& p, hipStream_t stream) {
  const int per = (p.g.nk + FEW_WAVES - 1) / FEW_WAVES;
  if constexpr (std::is_same<T, void>::value && MF <= 2)
    if (per >= 4) return launch_few_u<T, AF, MF, NF, 4>(p, stream);
  return per >= 2 ? launch_few_u<T, AF, MF, NF, 2>(p, stream) : launch_few_u<T, AF, MF, NF, 1>(p, stream);
}

template <int AF, int BM, int BN, int WM, int WN, int NS, bool DIRECT>
hipError_t launch(const MxGemmParams& p, hipStream_t stream) {
  using T = Tile<AF, BM, BN, WM, WN, NS, DIRECT>;
  static DeviceKernelSetup setup;
  int n_cu = 0;
  if (hipError_t e = setup.ensure((const void*)mx_gemm_kernel<AF, BM, BN, WM, WN, NS, DIRECT>, T::LDS, &n_cu); e != hipSuccess) return e;
  const long tiles = (long)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  if (tiles > 0x3fffffff) return hipErrorInvalidValue;
  const long resident = (long)n_cu * (163840 / T::LDS);             // workgroups that the CUs hold
  hipLaunchKernelGGL((mx_gemm_kernel<AF, BM, BN, WM, WN, NS, DIRECT>), dim3((unsigned)(tiles < resident ? tiles : resident)), dim3(T::THREADS), T::LDS, stream, p);
  return hipGetLastError();
}

constexpr int CUS = 256;                // (a device with fewer CUs only takes its turns earlier)
// Fewer than a 256 x 256 tile a CU.  64 x 64 tiles while the CUs hold them in one go, two a CU; a third one on some of them costs as much as
// one on each, and 128 x 128 tiles then take less time (e2m1 / e4m3, us in 64 x 64 and in 128 x 128:  448 tiles, 400 rows x 1024 -> 4096, 6.9 / 11.6
// and 7.7 / 13.3;  494, 1154 x 8192 -> 1664, 26 / 58 and 33 / 71;  528, 2056 x 1024 -> 1024, 8.7 / 15.7 and 7.7 / 13.1;  560, 400 x 1280 -> 5120,
// 9.9 / 18.5 and 8.5 / 15.5;  640, 577 x 1024 -> 4096, 9.1 / 16.0 and 10.4 / 15.6, the one that loses;  832, 770 x 1024 -> 4096, 10.7 / 19.4 and
// 8.1 / 13.8).  128 x 128: eight waves with four stages in LDS while they are at most one a CU, and latency is what a stage costs, else four waves, two
// workgroups a CU.  (e4m3: waves of 32 x 64, which part each row fragment for four products instead of two: 46 -> 40 us at 2885 x 4001 -> 1003.)
template <int AF>
hipError_t small_tiles(const MxGemmParams& p, hipStream_t stream) {
  const long tiles64 = (long)((p.M + 63) / 64) * ((p.N + 63) / 64), tiles128 = (long)((p.M + 127) / 128) * ((p.N + 127) / 128);
  if (tiles64 <= 2 * CUS) return launch<AF, 64, 64, 2, 2, 4, true>(p, stream);
  if (tiles128 > 256) return launch<AF, 128, 128, 2, 2, 2, false>(p, stream);
  if constexpr (AF == A_E4M3) return launch<AF, 128, 128, 4, 2, 4, true>(p, stream);
  else return launch<AF, 128, 128, 2, 4, 4, true>(p, stream);
}

// The few-row kernel: up to 16 rows; up to 48 while its workgroups are at most two a CU (e2m1 / e4m3, 48 rows: 8192 columns of 1664
// 5.4 / 10.8 us, in 64 x 64 tiles 7.8 / 13.0; 12 800 columns of 5120 28 / 47 against 15 / 32); more rows while its workgroups of 64 rows x
// 16 columns are at most one a CU -- a long K is then shared by eight waves instead of walked by four (256 x 4096 -> 1024 9.5 / 14.1 us
// against 10.5 / 24.3; 384 rows 16.0 / 25.9 against 10.6 / 24.2).
inline bool few(const MxGemmParams& p) { return p.M <= 16 || (long)((p.M + 63) / 64) * ((p.N + 15) / 16) <= (p.M <= 48 ? 2 * CUS : CUS); }
template <int AF>
hipError_t few_rows(const MxGemmParams& p, hipStream_t stream) {
  MxFewParams f{};
  f.g = p;
  return p.M <= 16 ? launch_few<void, AF, 1>(f, stream) : p.M <= 32 ? launch_few<void, AF, 2>(f, stream) : launch_few<void, AF, 4>(f, stream);
}

template <int AF>
hipError_t large_tiles(const MxGemmParams& p, hipStream_t stream) {
  return launch<AF, 256, 256, 2, 4, 2, false>(p, stream);
}

template <int AF>
hipError_t choose(MxGemmParams p, hipStream_t stream) {
  if (few(p)) return few_rows<AF>(p, stream);
  // 256 x 256 tiles once they give every CU one.  Where a last round of them would leave three quarters of the CUs idle, its rows go to a
  // second launch of its own kind: 65 792 x 4096 -> 1024 is 4 rounds and 4 tiles.
  const long tn = (p.N + 255) / 256, tiles = (long)((p.M + 255) / 256) * tn;
  if (tiles < CUS) return small_tiles<AF>(p, stream);
  const int rest = (int)(tiles % CUS);
  const long rows = tiles / CUS * CUS / tn * 256;
  if (rest == 0 || rest * 4 > CUS || rows == 0 || rows >= p.M) return large_tiles<AF>(p, stream);
  const int M = p.M;
  p.M = (int)rows;
  if (hipError_t e = large_tiles<AF>(p, stream); e != hipSuccess) return e;
  p.M = M - (int)rows;
  p.a += (size_t)rows * p.nk * (AF == A_E2M1 ? 64 : 128);
  p.a_scale += (size_t)rows * p.nk * 4;
  const size_t skip = (size_t)rows * p.N * (p.out_dtype == MX_DT_F32 ? 4 : 2);
  p.out = (char*)p.out + skip;
  if (p.resid) p.resid = (const char*)p.resid + skip;
  return few(p) ? few_rows<AF>(p, stream) : small_tiles<AF>(p, stream);
}

}  // namespace

hipError_t ce_mx_gemm(MxGemmParams p, int a_fmt, hipStream_t stream) {
  // Results that do not fit the L2s and are not the residual stream's next rows leave with the streaming cache policy: the operands'
  // panels stay (65 792 x 1024 -> 4096: 265 -> 253 us; onto a residual it costs 1 %).
  p.streamed = !p.resid && (size_t)p.M * p.N * 2 > (64u << 20);
  if (a_fmt == MX_E2M1) return choose<A_E2M1>(p, stream);
  return choose<A_E4M3>(p, stream);
}

template <typename T, int AF>
static hipError_t few_values_of(const MxFewParams& f, hipStream_t stream) {
  return f.g.N > MX_VALUE_COLS ? launch_few<T, AF, 1, 4>(f, stream) : launch_few<T, AF, 1>(f, stream);
}
template <typename T>
static hipError_t few_values(const MxFewParams& f, int fmt, hipStream_t stream) {
  return fmt == MX_E2M1 ? few_values_of<T, A_E2M1>(f, stream) : few_values_of<T, A_E4M3>(f, stream);
}
hipError_t ce_mx_gemm_values(const MxGemmParams& p, const void* x, int dtype, long ld_x, int k, int fmt, hipStream_t stream) {
  if (!mx_takes_values(p.M, p.N, k)) return hipErrorInvalidValue;
  MxFewParams f{};
  f.g = p; f.x = x; f.ld_x = ld_x; f.k = k;
  return dtype == MX_DT_BF16 ? few_values<__bf16>(f, fmt, stream) : dtype == MX_DT_F16 ? few_values<_Float16>(f, fmt, stream) : few_values<float>(f, fmt, stream);
}
