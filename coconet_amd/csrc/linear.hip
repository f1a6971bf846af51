// A dense layer with its epilogue fused into the product, and its gradients (gfx950).
//
//   forward    z = X.W + bias, Y = act(z) + resid, pre = z          X [M x K], W [K x N], row-major
//   backward   dz = dY * act'(pre), dX = dz.W^T, dW (+)= X^T.dz, db (+)= column sums of dz
//
// All three products are C[rows x cols] = sum over c of P(row, c) * Q(c, col) with operands that lie in memory either with
// the summed index contiguous ("along": X and dz in forward and dX, W in dX) or with the outer index contiguous
// ("across": W in forward, X and dz in dW).  Both kinds are fetched as they lie, in 16-byte pieces, and both become the
// same matrix-core fragments (8 consecutive c of one row or column per lane): an "along" tile is read from LDS by plain
// 16-byte reads, an "across" tile through the transposing ds_read_b64_tr_b16.
#include "ccn_common.hpp"

#include <atomic>
#include <cmath>
#include <new>
#include <type_traits>

namespace ccn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

template <bool F16> __device__ __forceinline__ float half_in(uint16_t h) { return F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h); }
template <bool F16> __device__ __forceinline__ uint16_t half_out(float f) {   // round to nearest even (gfx950 converts to bfloat16 itself)
  return F16 ? f32_to_f16_bits(f) : __builtin_bit_cast(uint16_t, (__bf16)f);
}

// ---- activations, in fp32 ----------------------------------------------------------------------------------------------
// A quarter-rate exp2 and reciprocal (1 ulp each) and a handful of multiply-adds per element: at one wavefront per SIMD the
// library's erff / tanhf / expf and the IEEE division cost more than the tile's stores.  Absolute errors stay below 3e-7
// of the argument, and on the left, where the gates are small themselves, relative ones below 3e-5 down to 1e-36 (GELU 9e-6 at
// z = -13, 3e-6 at -6, nearly all of it the roundings of the exponent): a fraction of the half step of a 16-bit output.
// Far out the limits hold exactly (0 on the left, z and slope 1 on the right, also at infinity); a NaN stays one.
constexpr float kLog2e = 1.44269504088896341f, kSqrtHalf = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kTanhC = 0.79788456080286536f, kTanhA = 0.044715f;   // sqrt(2/pi)
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * x));
}
// Phi(-|z|) = exp(-z^2/2) * t * P(t), t = 1/(1 + 0.45 x), x = |z|/sqrt 2: the form of formula 7.1.26 of Abramowitz and Stegun, with a P of
// degree 7 fitted to erfc(x) exp(x^2) / 2 for all x >= 0, so that the tail, which z multiplies, is right relative to itself: of all such
// P the one with the smallest largest error, where Phi/30 counts as much as 1 absolutely.  Largest errors: 7.2e-8 of 1, 1.8e-6 of
// Phi(-|z|).  (7.1.26's own coefficients bound the absolute error alone, 1.5e-7: 7 half steps of a bfloat16 at z = -10.)
// *bell: exp(-z^2/2).
__device__ __forceinline__ float normal_cdf(float z, float* bell) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.45f * kSqrtHalf, fabsf(z), 1.0f));
  *bell = __builtin_amdgcn_exp2f(-0.5f * kLog2e * z * z);
  float p = fmaf(0.032212199f, t, -0.116187377f);
  p = fmaf(p, t, 0.099890082f);
  p = fmaf(p, t, 0.021964574f);
  p = fmaf(p, t, 0.094696882f);
  p = fmaf(p, t, 0.113523449f);
  p = fmaf(p, t, 0.126957498f);
  p = fmaf(p, t, 0.126942743f);
  const float tail = p * t * *bell;   // Phi(-|z|)
  return z < 0.0f ? tail : 1.0f - tail;
}
__device__ __forceinline__ float gelu_tanh_gate(float z) {   // (1 + tanh u)/2 = sigmoid(2u)
  return sigmoid(2.0f * kTanhC * z * fmaf(kTanhA * z, z, 1.0f));
}
// v <- act(v) for eight values.  The gate times z; a z so far left that the gate is 0 is cut off, -inf * 0 would be NaN.
__device__ __forceinline__ void act_values(int act, float* v) {
  if (act == CCN_ACT_NONE) return;
  if (act == CCN_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = v[e] < 0.0f ? 0.0f : v[e];
  } else if (act == CCN_ACT_GELU) {
    float bell;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = fmaxf(v[e], -104.0f) * normal_cdf(v[e], &bell);
  } else if (act == CCN_ACT_GELU_TANH) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = fmaxf(v[e], -104.0f) * gelu_tanh_gate(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = fmaxf(v[e], -104.0f) * sigmoid(v[e]);
  }
}
// g <- g * act'(z) for eight values.  Beyond +-104 the slopes are 0 and 1; a NaN in z stays one.
template <class Slope> __device__ __forceinline__ void times_slope(const float* z, float* g, Slope slope) {
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const float s = slope(__builtin_amdgcn_fmed3f(z[e], -104.0f, 104.0f));
    g[e] *= z[e] != z[e] ? z[e] : s;
  }
}
__device__ __forceinline__ void act_slopes(int act, const float* z, float* g) {
  if (act == CCN_ACT_RELU) {
    times_slope(z, g, [](float x) { return x > 0.0f ? 1.0f : 0.0f; });
  } else if (act == CCN_ACT_GELU) {
    times_slope(z, g, [](float x) {
      float bell;
      const float p = normal_cdf(x, &bell);
      return fmaf(x * kInvSqrt2Pi, bell, p);
    });
  } else if (act == CCN_ACT_GELU_TANH) {
    times_slope(z, g, [](float x) {
      const float s = gelu_tanh_gate(x);
      return fmaf(x * s * (1.0f - s) * (2.0f * kTanhC), fmaf(3.0f * kTanhA * x, x, 1.0f), s);
    });
  } else if (act == CCN_ACT_SILU) {
    times_slope(z, g, [](float x) {
      const float s = sigmoid(x);
      return s * fmaf(x, 1.0f - s, 1.0f);
    });
  }
}

// ---- eight neighbouring elements of a row --------------------------------------------------------------------------------
// gfx950 loads and stores 16 bytes at any 2-byte aligned address; `n` is how many of the eight are there (behind a row's
// end they are neither read nor written).
// Loading is done in two steps, so that many loads can be in flight before the first is looked at: fetch_piece reads the piece at
// column `col` of a row of `len` elements, or the row's last 16 bytes where the piece would cross (or lie behind) the end;
// trim_piece then shifts the `n` = len - col elements down and puts zeros behind them (n <= 0: zeros).
__device__ __forceinline__ u32x4 fetch_piece(const uint16_t* row, int col, int len) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if (len >= 8) {   // uniform
    const int at = len - 8;
    __builtin_memcpy(&v, row + (col < at ? col : at), 16);
  } else {
#pragma unroll
    for (int e = 0; e < 7; e++)
      if (e < len) v[e >> 1] |= (uint32_t)row[e] << (16 * (e & 1));   // trimmed to what is there already
  }
  return v;
}
__device__ __forceinline__ u32x4 trim_piece(u32x4 v, int n, int len) {
  if (__ballot(n < 8) == 0) return v;
  const int s = n >= 8 || len < 8 ? 0 : 8 - n;   // (a row of fewer than 8 elements is one piece, loaded unshifted)
  if (s & 4) v = u32x4{v[2], v[3], 0u, 0u};
  if (s & 2) v = u32x4{v[1], v[2], v[3], 0u};
  if (s & 1) v = u32x4{(v[0] >> 16) | (v[1] << 16), (v[1] >> 16) | (v[2] << 16), (v[2] >> 16) | (v[3] << 16), v[3] >> 16};
  if (n <= 0) v = u32x4{0u, 0u, 0u, 0u};
  return v;
}
__device__ __forceinline__ void store_piece(uint16_t* p, const u32x4 v, int n) {
  if (n >= 8) {
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 7; e++)
      if (e < n) p[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
  }
}
template <bool F16> __device__ __forceinline__ void unpack(const u32x4 v, float* x) {
#pragma unroll
  for (int e = 0; e < 8; e++) x[e] = half_in<F16>((uint16_t)(v[e >> 1] >> (16 * (e & 1))));
}
template <bool F16> __device__ __forceinline__ u32x4 pack(const float* x) {
  u32x4 v;
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = (uint32_t)half_out<F16>(x[2 * e]) | ((uint32_t)half_out<F16>(x[2 * e + 1]) << 16);
  return v;
}

struct LinEpi {
  const float* bias;
  const uint16_t* resid;
  uint16_t* pre;
  void* out;
  size_t ldr, ldp, ldo;
  int act;
  int accumulate;   // fp32 output only
};

// Finishing elements (row, col .. col+7) of the output, n of them inside the row, in two steps, so that the loads of
// several pieces can be in flight together.  OUT32: an fp32 output, stored or added to; else the forward epilogue (of
// which a plain 16-bit product is the case with nothing to do).  The bias depends on the column alone.
struct Bias8 { float b[8]; };
__device__ __forceinline__ void load_bias(Bias8& x, const LinEpi& ep, size_t col, int n) {
#pragma unroll
  for (int e = 0; e < 8; e++) x.b[e] = 0.0f;
  if (!ep.bias) return;
  if (n >= 8) {
    __builtin_memcpy(x.b, ep.bias + col, 32);
  } else {
#pragma unroll
    for (int e = 0; e < 7; e++)
      if (e < n) x.b[e] = ep.bias[col + e];
  }
}
// Where the pieces of one lane lie: uniform bases and steps (scalar registers) and one 32-bit offset per lane and array.
struct Places {
  uint8_t *out, *pre;
  const uint8_t* res;
  size_t sout, spre, sres;     // bytes from a piece to the lane's next one
  uint32_t vout, vpre, vres;
};
// row0, col0: uniform corner; the lane's first piece is at (row0 + lr, col0 + lc), the next ones `step` rows further each.
template <bool OUT32>
__device__ __forceinline__ Places places(const LinEpi& ep, size_t row0, size_t col0, int lr, int lc, int step) {
  constexpr int kOut = OUT32 ? 4 : 2;
  Places w;
  w.out = static_cast<uint8_t*>(ep.out) + (row0 * ep.ldo + col0) * kOut;
  w.sout = (size_t)step * ep.ldo * kOut;
  w.vout = (uint32_t)(lr * (int)ep.ldo + lc) * kOut;
  w.res = reinterpret_cast<const uint8_t*>(ep.resid) + (row0 * ep.ldr + col0) * 2;
  w.sres = (size_t)step * ep.ldr * 2;
  w.vres = (uint32_t)(lr * (int)ep.ldr + lc) * 2;
  w.pre = reinterpret_cast<uint8_t*>(ep.pre) + (row0 * ep.ldp + col0) * 2;
  w.spre = (size_t)step * ep.ldp * 2;
  w.vpre = (uint32_t)(lr * (int)ep.ldp + lc) * 2;
  return w;
}
template <bool OUT32> struct Old8 { u32x4 r; };        // the residual
template <> struct Old8<true> { float d[8]; };         // what is added to
template <bool OUT32>
__device__ __forceinline__ void load_old(Old8<OUT32>& x, const LinEpi& ep, const Places& w, int i, int n, int back) {
  if constexpr (OUT32) {
    if (!ep.accumulate) return;
    const float* const o = reinterpret_cast<const float*>(w.out + i * w.sout + w.vout);
    if (n >= 8) {
      __builtin_memcpy(x.d, o, 32);
    } else {
#pragma unroll
      for (int e = 0; e < 7; e++)
        if (e < n) x.d[e] = o[e];
    }
  } else {
    if (ep.resid) x.r = trim_piece(fetch_piece(reinterpret_cast<const uint16_t*>(w.res + i * w.sres + w.vres) - back, back, back + n), n, back + n);
  }
}
template <bool F16, bool OUT32>
__device__ __forceinline__ void finish8(float* v, const Bias8& bias, const Old8<OUT32>& old, const LinEpi& ep, const Places& w, int i, int n) {
  if constexpr (OUT32) {
    float* const o = reinterpret_cast<float*>(w.out + i * w.sout + w.vout);
    if (ep.accumulate) {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = old.d[e] + v[e];
    }
    if (n >= 8) {
      __builtin_memcpy(o, v, 32);
    } else {
#pragma unroll
      for (int e = 0; e < 7; e++)
        if (e < n) o[e] = v[e];
    }
  } else {
    if (ep.bias) {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += bias.b[e];
    }
    if (ep.pre) store_piece(reinterpret_cast<uint16_t*>(w.pre + i * w.spre + w.vpre), pack<F16>(v), n);
    act_values(ep.act, v);
    if (ep.resid) {
      float x[8];
      unpack<F16>(old.r, x);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += x[e];
    }
    store_piece(reinterpret_cast<uint16_t*>(w.out + i * w.sout + w.vout), pack<F16>(v), n);
  }
}

// Which tile a workgroup takes.  Workgroup b runs on XCD b % 8: every XCD gets a contiguous range of tile numbers, and
// tiles are numbered down four tile rows before the next tile column, so the workgroups an XCD runs at a time form a block
// whose operand panels are shared in its L2.
__device__ __forceinline__ void tile_of(uint32_t b, int tiles_r, int tiles_c, int& tr, int& tc) {
  const uint32_t total = (uint32_t)tiles_r * (uint32_t)tiles_c, x = b & 7u, q = total >> 3, rest = total & 7u;
  const uint32_t id = x * q + (x < rest ? x : rest) + (b >> 3);
  const uint32_t band = 4u * (uint32_t)tiles_c, g = id / band, in = id - g * band;
  const uint32_t first = 4u * g, left = (uint32_t)tiles_r - first, h = left < 4u ? left : 4u;
  tr = (int)(first + in % h);
  tc = (int)(in / h);
}

enum { kOut16 = 0, kOut32 = 1, kOutPartial = 2 };   // what a tile leaves: a 16-bit or an fp32 output, or a split's fp32 sums

struct LinProd {
  const uint16_t* p;   // row operand
  const uint16_t* q;   // column operand
  size_t ldp, ldq;
  int rows, cols, sum;
  int read_r, read_c;  // rows or columns of the operands that may be read: rows, cols, or for an "across" operand that many rounded up to 8
  int tiles_r, tiles_c;
  int per_split;       // summed elements per split (a multiple of 64)
  int brief;           // the sum is short: no ring
  float* partial;      // [splits][rows][cols rounded up to 8] when splits > 1
};

template <bool F16> __device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// ---- 16-byte aligned operands: tiles on a ring of direct-to-LDS stages -------------------------------------------------------
// A 256-thread workgroup owns a tile of (64*FR) x (64*FC), its four wavefronts a quarter each, FR x FC blocks of 32 x 32.
// The operands travel from memory to LDS directly, into a ring of four stages of RK summed elements; requests of 1 KiB are
// spread between the matrix instructions, and one is waited for three steps after it was made.  An "along" stage holds rows
// of 2*RK bytes, the 16-byte pieces swizzled so that the 32 rows of a fragment meet no bank twice; an "across" stage RK rows as
// in memory, swizzled by 4*(k%4).  Tiles at the edge read the last row or the last 8 columns again (results not stored); a
// sum that is no multiple of RK ends with a step loaded through registers with zeros behind the end.  The ring's LDS makes it one
// workgroup per CU; a short sum takes one stage, through registers, and up to four share a CU.
//   4 x 4   256 x 256, RK 32: 256 accumulators per lane, in the accumulation half of the register file; per 16 summed elements a
//           wavefront reads eight fragments for sixteen matrix instructions
//   4 x 2   256 x 128, RK 32: six fragments for eight
//   2 x 2   128 x 128, RK 64: for outputs of few large tiles.  A step of 64 summed elements takes 0.40 us; its matrix instructions
//           fill 512 clocks of it and its LDS reads 300 (counted over 777 x 1537 x 2049): neither bounds it, one wavefront per SIMD
//           waits for the other's part of the stage.  An "along" request covers whole 128-byte lines (RK 32, two workgroups per
//           CU: half of every line fetched is wasted)
// 8192 x 8192 x 4096 with bias, gelu_tanh and the kept pre-activation: 416 to 457 us from card to card, 1.2-1.32 PFLOP/s; dX and dW of it
// 412-465 and 390-424.  The clock falls to 1.55-1.7 GHz under these products; of its cycles the matrix units are busy in 75 % (dX 69, dW
// 78), the LDS reads in 20 % (GRBM_GUI_ACTIVE, SQ_VALU_MFMA_BUSY_CYCLES, SQ_LDS_IDX_ACTIVE).
constexpr size_t kRMaxLd = (size_t)1 << 21;  // 256 rows of it stay inside the 2 GiB that a buffer descriptor spans
constexpr int kStages = 4;
template <int FR, int FC> struct Ring {
  static constexpr int RK = FR == 4 ? 32 : 64;
  static constexpr int kRounds = RK / 16;
  static constexpr int kRows = 64 * FR, kCols = 64 * FC;
  static constexpr int kSideP = kRows * RK * 2, kSideQ = kCols * RK * 2, kStage = kSideP + kSideQ;
  static constexpr int kCStride = 32 * FC + 4;   // floats per row of a wavefront's 32 x (32*FC) piece of the output
  static constexpr int kLds = kStages * kStage;
  static constexpr int kPieces = 4 * 32 * kCStride * 4, kBriefLds = kStage > kPieces ? kStage : kPieces;   // one stage, then the output's pieces
  static constexpr int kPerStep = (FR + FC) * RK / 32;   // requests of a wavefront per step
  static_assert(kLds >= kPieces, "output pieces");
};

__device__ __forceinline__ u32x4 descriptor(const void* base) {   // no stride; the offsets used below stay inside the matrix
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return u32x4{(uint32_t)a, (uint32_t)(a >> 32), 0x7ffffffcu, 0x00020000u};
}
// 1 KiB from memory to LDS, lane L's 16 bytes to position L.  In assembly, because the compiler puts a wait for ALL
// outstanding loads before every LDS read that follows a direct load which it can see; here the waits are placed by hand:
// a stage is read only behind the wait and the barrier of its step.
__device__ __forceinline__ void load_to_lds(u32x4 rs, uint32_t lds_addr, uint32_t voff, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds_addr), "v"(voff), "s"(rs), "s"(soff) : "memory");
}
constexpr int waitcnt(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8); }

// One operand of F 64-row (or 64-column) bands, RK summed elements at a time.
template <bool ALONG, int F, int RK> struct RSide {
  static constexpr int kOuter = 64 * F, kRequests = F * RK / 32;   // of a wavefront, per stage
  static constexpr int kRowBytes = ALONG ? 2 * RK : 2 * kOuter;    // a row of the stage: one outer index, or one summed element
  static constexpr int kLanes = kRowBytes / 16, kPer = 64 / kLanes;   // lanes per row, rows per request
  const uint16_t* base;   // along: the tile's first row;  across: its first column
  uint32_t voff[ALONG ? kRequests : 1], soff0, soffj;
  size_t ld;
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (!ALONG) return 4 * (row & 3);
    else return RK == 32 ? (row >> 2) & 3 : (row & 7) ^ ((row >> 3) & 7);
  }
  // wavefront w makes requests j of a stage: its rows kPer*(w + 4j) .. +kPer-1.  outer: rows, or columns that may be read (a
  // multiple of 8)
  __device__ __forceinline__ void init(const uint16_t* p, size_t ld_, int o0, int outer, int lane, int wave) {
    ld = ld_;
    const int in = lane / kLanes, slot = lane % kLanes;
    if constexpr (ALONG) {
      base = p + (size_t)o0 * ld;
      const int last = outer - 1 - o0;
#pragma unroll
      for (int j = 0; j < kRequests; j++) {
        const int r = kPer * (wave + 4 * j) + in;
        voff[j] = (uint32_t)(r < last ? r : last) * (uint32_t)(ld * 2) + 16u * (uint32_t)(slot ^ swizzle(r));
      }
      soff0 = soffj = 0;
    } else {
      base = p + o0;
      const int c = 8 * (slot ^ swizzle(kPer * wave + in)), last = outer - 8 - o0;   // (a multiple of 4 rows from j to j + 1)
      voff[0] = (uint32_t)in * (uint32_t)(ld * 2) + 2u * (uint32_t)(c < last ? c : last);
      soff0 = (uint32_t)(kPer * wave) * (uint32_t)(ld * 2);
      soffj = (uint32_t)(4 * kPer) * (uint32_t)(ld * 2);
    }
  }
  __device__ __forceinline__ void request(uint32_t lds_addr, int step, int j) const {
    if constexpr (ALONG) load_to_lds(descriptor(base), lds_addr + j * 4096, voff[j], (uint32_t)step * (RK * 2));
    else load_to_lds(descriptor(base + (size_t)step * RK * ld), lds_addr + j * 4096, voff[0], soff0 + j * soffj);
  }
  // the summed elements from `k` on, `left` of them (RK are used), through registers.  outer: as for init
  struct Held { u32x4 v[kRequests]; };
  __device__ __forceinline__ void hold(Held& h, int k, int left, int o0, int outer, int t) const {
#pragma unroll
    for (int i = 0; i < kRequests; i++) {
      const int id = t + 256 * i, row = id / kLanes, c = 8 * ((id % kLanes) ^ swizzle(row));
      if constexpr (ALONG) {
        const int last = outer - 1 - o0;
        h.v[i] = fetch_piece(base + (size_t)(row < last ? row : last) * ld, k + c, k + left);
      } else {
        h.v[i] = fetch_piece(base - o0 + (size_t)(k + (row < left ? row : left - 1)) * ld, o0 + c, outer);
      }
    }
  }
  __device__ __forceinline__ void put(uint8_t* lds, const Held& h, int k, int left, int o0, int outer, int t) const {
#pragma unroll
    for (int i = 0; i < kRequests; i++) {
      const int id = t + 256 * i, row = id / kLanes, c = 8 * ((id % kLanes) ^ swizzle(row));
      *reinterpret_cast<u32x4*>(lds + id * 16) = ALONG ? trim_piece(h.v[i], left - c, k + left) : trim_piece(h.v[i], row < left ? outer - o0 - c : 0, outer);
    }
  }
  // fragment f: 32 rows or columns from 32*f of this wavefront's half of the tile, 16 summed elements from 16*ks on
  static __device__ __forceinline__ int address(int half, int lane) {
    const int li = lane & 31, lh = lane >> 5;
    if constexpr (ALONG) return (32 * F * half + li) * kRowBytes;
    const int a16 = lane & 15, g2 = (lane >> 4) & 1;
    return (lh * 8 + (a16 >> 2)) * kRowBytes + (((4 * F * half + 2 * g2 + ((a16 >> 1) & 1)) ^ (4 * (a16 >> 2))) * 16) + 8 * (a16 & 1);
  }
  static __device__ __forceinline__ s16x8 frag(const uint8_t* lds, int at, int f, int ks, int lane) {
    if constexpr (ALONG) {
      const int li = lane & 31, lh = lane >> 5;   // a half of the tile is a multiple of 64 rows: it does not change the swizzle
      return *reinterpret_cast<const s16x8*>(lds + at + f * 32 * kRowBytes + (((2 * ks + lh) ^ swizzle(32 * f + li)) << 4));
    } else {
      const uint8_t* p = lds + (at ^ (f * 64)) + ks * (16 * kRowBytes);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p + 4 * kRowBytes));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// finish8 for pieces that are all inside the row, addressed as the ring's tiles want it: a descriptor per array, the piece in
// a scalar offset (it moves `step` rows from one to the next) and one 32-bit offset per lane.
template <bool OUT32> struct WholePieces {
  typedef __amdgpu_buffer_rsrc_t rsrc_t;
  rsrc_t out, res, pre;
  uint32_t vout, vres, vpre, sout, sres, spre;
  static constexpr int kOut = OUT32 ? 4 : 2;
  // All CUs write their tiles at about the same time: nontemporal stores do not push the operand panels out of L2 (8192 x
  // 1024 x 8192: 164 us with ordinary ones, 147 with these, 141 with none).
  static constexpr int kNt = 2;
  static __device__ __forceinline__ rsrc_t at(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0x7ffffffc, 0x00020000);
  }
  __device__ __forceinline__ WholePieces(const LinEpi& ep, size_t row0, size_t col0, int lr, int lc, int step) {
    out = at(static_cast<uint8_t*>(ep.out) + (row0 * ep.ldo + col0) * kOut);
    res = at(ep.resid + (row0 * ep.ldr + col0));
    pre = at(ep.pre + (row0 * ep.ldp + col0));
    vout = (uint32_t)(lr * (int)ep.ldo + lc) * kOut;
    vres = (uint32_t)(lr * (int)ep.ldr + lc) * 2;
    vpre = (uint32_t)(lr * (int)ep.ldp + lc) * 2;
    sout = (uint32_t)step * (uint32_t)ep.ldo * kOut;
    sres = (uint32_t)step * (uint32_t)ep.ldr * 2;
    spre = (uint32_t)step * (uint32_t)ep.ldp * 2;
  }
  __device__ __forceinline__ void load_old(Old8<OUT32>& x, const LinEpi& ep, int i) const {
    if constexpr (OUT32) {
      if (!ep.accumulate) return;
      const u32x4 lo = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(out, vout, i * sout, 0));
      const u32x4 hi = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(out, vout + 16, i * sout, 0));
      __builtin_memcpy(x.d, &lo, 16);
      __builtin_memcpy(x.d + 4, &hi, 16);
    } else {
      if (ep.resid) x.r = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(res, vres, i * sres, 0));
    }
  }
  template <bool F16> __device__ __forceinline__ void finish(float* v, const Bias8& bias, const Old8<OUT32>& old, const LinEpi& ep, int i) const {
    if constexpr (OUT32) {
      if (ep.accumulate) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = old.d[e] + v[e];
      }
      u32x4 lo, hi;
      __builtin_memcpy(&lo, v, 16);
      __builtin_memcpy(&hi, v + 4, 16);
      __builtin_amdgcn_raw_buffer_store_b128(lo, out, vout, i * sout, kNt);
      __builtin_amdgcn_raw_buffer_store_b128(hi, out, vout + 16, i * sout, kNt);
    } else {
      if (ep.bias) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += bias.b[e];
      }
      if (ep.pre) __builtin_amdgcn_raw_buffer_store_b128(pack<F16>(v), pre, vpre, i * spre, kNt);
      act_values(ep.act, v);
      if (ep.resid) {
        float x[8];
        unpack<F16>(old.r, x);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += x[e];
      }
      __builtin_amdgcn_raw_buffer_store_b128(pack<F16>(v), out, vout, i * sout, kNt);
    }
  }
};
// The same interface for rows that may start anywhere (pieces inside the row; what is behind the last one: edge_elements).
template <bool OUT32> struct AnyPieces {
  Places w;
  __device__ __forceinline__ AnyPieces(const LinEpi& ep, size_t row0, size_t col0, int lr, int lc, int step)
      : w(places<OUT32>(ep, row0, col0, lr, lc, step)) {}
  __device__ __forceinline__ void load_old(Old8<OUT32>& x, const LinEpi& ep, int i) const { ccn::load_old<OUT32>(x, ep, w, i, 8, 0); }
  template <bool F16> __device__ __forceinline__ void finish(float* v, const Bias8& bias, const Old8<OUT32>& old, const LinEpi& ep, int i) const {
    finish8<F16, OUT32>(v, bias, old, ep, w, i, 8);
  }
};
// The last `n` (1..7) columns of 32 rows of an output whose width is no multiple of 8, an element per lane and turn: at(row, e)
// gives the finished sum.  rows: how many of the 32 are inside the matrix.
template <bool F16, bool OUT32, class At>
__device__ __forceinline__ void edge_elements(const LinEpi& ep, size_t row0, size_t col, int n, int rows, int lane, At at) {
  constexpr int kTurns = 4;   // 7 * 32 elements at most
  const uint32_t magic = 65536u / (uint32_t)n + 1u;   // i / n for i < 224
  float v[kTurns], old[kTurns], bias[kTurns];
  size_t r[kTurns], c[kTurns];
  bool on[kTurns];
#pragma unroll
  for (int u = 0; u < kTurns; u++) {
    const uint32_t i = (uint32_t)(lane + kWave * u), q = (i * magic) >> 16, e = i - q * (uint32_t)n;
    on[u] = (int)q < rows;
    r[u] = row0 + q;
    c[u] = col + e;
    v[u] = old[u] = bias[u] = 0.0f;
    if (on[u]) {
      v[u] = at((int)q, (int)e);
      if constexpr (OUT32) {
        if (ep.accumulate) old[u] = static_cast<const float*>(ep.out)[r[u] * ep.ldo + c[u]];
      } else {
        if (ep.bias) bias[u] = ep.bias[c[u]];
        if (ep.resid) old[u] = half_in<F16>(ep.resid[r[u] * ep.ldr + c[u]]);
      }
    }
  }
  if constexpr (OUT32) {
#pragma unroll
    for (int u = 0; u < kTurns; u++)
      if (on[u]) static_cast<float*>(ep.out)[r[u] * ep.ldo + c[u]] = old[u] + v[u];
  } else {
    float x[8];   // as the pieces compute them
#pragma unroll
    for (int u = 0; u < 8; u++) x[u] = u < kTurns ? v[u & 3] + bias[u & 3] : 0.0f;
#pragma unroll
    for (int u = 0; u < kTurns; u++)
      if (on[u] && ep.pre) ep.pre[r[u] * ep.ldp + c[u]] = half_out<F16>(x[u]);
    act_values(ep.act, x);
#pragma unroll
    for (int u = 0; u < kTurns; u++)
      if (on[u]) static_cast<uint16_t*>(ep.out)[r[u] * ep.ldo + c[u]] = half_out<F16>(ep.resid ? x[u] + old[u] : x[u]);
  }
}

// One tile.  OUT: kOut16, kOut32 or kOutPartial.  WHOLE: every piece of an output row is inside it and 16-byte aligned.
template <bool F16, bool PA, bool QA, int FR, int FC, int OUT, bool WHOLE>
__device__ __forceinline__ void ring_tile(const LinProd& pr, const LinEpi& ep, const uint32_t tile, const int split, uint8_t* const lds_ring) {
  typedef Ring<FR, FC> R;
  constexpr int RK = R::RK;
  int tr, tc;
  tile_of(tile, pr.tiles_r, pr.tiles_c, tr, tc);
  const int r0 = tr * R::kRows, c0 = tc * R::kCols;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);   // a scalar: it goes into descriptors
  const int wr = wave >> 1, wc = wave & 1, li = lane & 31, lh = lane >> 5;
  // this split's whole steps, and the elements behind them
  const int k_begin = OUT == kOutPartial ? split * pr.per_split : 0, first = k_begin / RK;
  const int k_end = OUT == kOutPartial && pr.sum - k_begin > pr.per_split ? k_begin + pr.per_split : pr.sum;
  // (a short sum goes through registers altogether: it needs a quarter of the LDS, and four workgroups share a CU)
  const int nk = pr.brief ? 0 : (k_end - k_begin) / RK;

  RSide<PA, FR, RK> sp;
  RSide<QA, FC, RK> sq;
  sp.init(pr.p, pr.ldp, r0, pr.read_r, lane, wave);
  sq.init(pr.q, pr.ldq, c0, pr.read_c, lane, wave);
  typedef __attribute__((address_space(3))) void* lds_void_ptr;
  const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((lds_void_ptr)lds_ring) + (uint32_t)wave * 1024u;
  // request j of step `kt` (past the end: the last step's again, unused), into stage `stage`
  auto request_p = [&](int stage, int kt, int j) { sp.request(lds0 + stage * R::kStage, first + (kt < nk ? kt : nk - 1), j); };
  auto request_q = [&](int stage, int kt, int j) { sq.request(lds0 + stage * R::kStage + R::kSideP, first + (kt < nk ? kt : nk - 1), j); };
  const int pat = sp.address(wr, lane), qat = sq.address(wc, lane);
  auto read_p = [&](int stage, int f, int ks) { return sp.frag(lds_ring + stage * R::kStage, pat, f, ks, lane); };
  auto read_q = [&](int stage, int f, int ks) { return sq.frag(lds_ring + stage * R::kStage + R::kSideP, qat, f, ks, lane); };

  f32x16 acc[FC][FR];   // [column block][row block]: register 4*i+e is row 32*rb + li, column 32*cb + 8*i + 4*lh + e
#pragma unroll
  for (int a = 0; a < FC; a++)
#pragma unroll
    for (int b = 0; b < FR; b++)
#pragma unroll
      for (int i = 0; i < 16; i++) acc[a][b][i] = 0.0f;

  // A round of 16 summed elements multiplies from fragment set `set` while the fragments of the next round are read into the
  // other set from (stage rbuf, sixteen rks), in the order in which that round needs them; between the matrix instructions part
  // `part` (of kRounds) of the requests for step `lkt` goes out.  Every piece is pinned in place: the order is the schedule.
  s16x8 fq[2][FC], fp[2][FR];
  auto pin = [] { __builtin_amdgcn_sched_barrier(0); };
  auto round = [&](int set, int rbuf, int rks, int lstage, int lkt, int part) {
    const int o = set ^ 1;
    auto m = [&](int rb, int cb) { acc[cb][rb] = mfma32<F16>(fq[set][cb], fp[set][rb], acc[cb][rb]); };
    if constexpr (FR == 4 && FC == 4) {
      // Odd steps make their two parts in the other order: a request of an "along" operand touches half of every 128-byte line,
      // and the other half then follows one round later, while the line is still in L1 (dX of 8192 x 8192 x 4096: 430 -> 412 us).
      const int half = part ^ (lstage & 1);
      fq[o][0] = read_q(rbuf, 0, rks); m(0, 0); pin();
      fp[o][0] = read_p(rbuf, 0, rks); m(0, 1); pin();
      fq[o][1] = read_q(rbuf, 1, rks); m(0, 2); pin();
      m(0, 3); pin();
      request_p(lstage, lkt, 2 * half); pin();
      fq[o][2] = read_q(rbuf, 2, rks); m(1, 0); pin();
      fq[o][3] = read_q(rbuf, 3, rks); m(1, 1); pin();
      fp[o][1] = read_p(rbuf, 1, rks); m(1, 2); pin();
      m(1, 3); pin();
      request_p(lstage, lkt, 2 * half + 1); pin();
      fp[o][2] = read_p(rbuf, 2, rks); m(2, 0); pin();
      m(2, 1); pin();
      m(2, 2); pin();
      m(2, 3); pin();
      request_q(lstage, lkt, 2 * half); pin();
      fp[o][3] = read_p(rbuf, 3, rks); m(3, 0); pin();
      m(3, 1); pin();
      m(3, 2); pin();
      m(3, 3); pin();
      request_q(lstage, lkt, 2 * half + 1); pin();
    } else if constexpr (FR == 4) {
      const int half = part ^ (lstage & 1);   // as above
      fq[o][0] = read_q(rbuf, 0, rks); m(0, 0); pin();
      fp[o][0] = read_p(rbuf, 0, rks); m(0, 1); pin();
      request_p(lstage, lkt, 2 * half); pin();
      fq[o][1] = read_q(rbuf, 1, rks); m(1, 0); pin();
      fp[o][1] = read_p(rbuf, 1, rks); m(1, 1); pin();
      request_p(lstage, lkt, 2 * half + 1); pin();
      fp[o][2] = read_p(rbuf, 2, rks); m(2, 0); pin();
      m(2, 1); pin();
      request_q(lstage, lkt, half); pin();
      fp[o][3] = read_p(rbuf, 3, rks); m(3, 0); pin();
      m(3, 1); pin();
    } else {
      static_assert(FR == 2 && FC == 2, "a schedule is written out for 4 x 4, 4 x 2 and 2 x 2 blocks");
      fq[o][0] = read_q(rbuf, 0, rks); m(0, 0); pin();
      fp[o][0] = read_p(rbuf, 0, rks); m(0, 1); pin();
      request_p(lstage, lkt, part); pin();
      fq[o][1] = read_q(rbuf, 1, rks); m(1, 0); pin();
      fp[o][1] = read_p(rbuf, 1, rks); m(1, 1); pin();
      request_q(lstage, lkt, part); pin();
    }
  };
  // Step kt multiplies from stage kt%4:
  //   all rounds but the last   read the next sixteen of this step; parts 1.. of the requests for step kt+3
  //   barrier      every wavefront waits for its own requests for step kt+1 (those of two newer steps stay in flight) and for
  //                its LDS reads, then for the others: stage (kt+1)%4 is complete, nobody reads stage kt%4 any more
  //   last round   reads the first sixteen of step kt+1; part 0 of the requests for step kt+4, into stage kt%4
  auto step = [&](int st, int kt) {
#pragma unroll
    for (int i = 0; i + 1 < R::kRounds; i++) round(i & 1, st, i + 1, (st + 3) & 3, kt + 3, i + 1);
    __builtin_amdgcn_s_waitcnt(waitcnt(2 * R::kPerStep, 0));
    __builtin_amdgcn_s_barrier();
    pin();
    round(1, (st + 1) & 3, 0, st, kt + 4, 0);
  };
  if (nk > 0) {
#pragma unroll
    for (int st = 0; st < 4; st++) {
      // of stage 3 part 0 only (with two rounds that is the second half of the rows: the stage is odd)
      constexpr int kp = decltype(sp)::kRequests, kq = decltype(sq)::kRequests;
#pragma unroll
      for (int j = 0; j < kp; j++)
        if (st < 3 || (R::kRounds == 2 ? j >= kp / 2 : j < kp / R::kRounds)) request_p(st, st, j);
#pragma unroll
      for (int j = 0; j < kq; j++)
        if (st < 3 || (R::kRounds == 2 ? j >= kq / 2 : j < kq / R::kRounds)) request_q(st, st, j);
    }
    __builtin_amdgcn_s_waitcnt(waitcnt(2 * R::kPerStep + R::kPerStep / R::kRounds, 0));   // the requests for step 0 have landed
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int f = 0; f < FC; f++) fq[0][f] = read_q(0, f, 0);
#pragma unroll
    for (int f = 0; f < FR; f++) fp[0][f] = read_p(0, f, 0);
    int kt = 0;
    for (; kt + 4 <= nk; kt += 4) {
      step(0, kt);
      step(1, kt + 1);
      step(2, kt + 2);
      step(3, kt + 3);
    }
    if (kt < nk) step(0, kt);
    if (kt + 1 < nk) step(1, kt + 1);
    if (kt + 2 < nk) step(2, kt + 2);
    __builtin_amdgcn_s_waitcnt(waitcnt(0, 0));   // the last reads of LDS and the last (unused) loads into it are done
    __builtin_amdgcn_s_barrier();                // ... everywhere, before the stages are written to
  }
  for (int k = k_begin + nk * RK; k < k_end; k += RK) {
    typename decltype(sp)::Held hp;
    typename decltype(sq)::Held hq;
    sp.hold(hp, k, k_end - k, r0, pr.read_r, t);
    sq.hold(hq, k, k_end - k, c0, pr.read_c, t);
    sp.put(lds_ring, hp, k, k_end - k, r0, pr.read_r, t);
    sq.put(lds_ring + R::kSideP, hq, k, k_end - k, c0, pr.read_c, t);
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < R::kRounds; ks++) {
      if (k + 16 * ks >= k_end) break;
#pragma unroll
      for (int f = 0; f < FC; f++) fq[0][f] = read_q(0, f, ks);
#pragma unroll
      for (int f = 0; f < FR; f++) fp[0][f] = read_p(0, f, ks);
#pragma unroll
      for (int rb = 0; rb < FR; rb++)
#pragma unroll
        for (int cb = 0; cb < FC; cb++) acc[cb][rb] = mfma32<F16>(fq[0][cb], fp[0][rb], acc[cb][rb]);
    }
    __syncthreads();
  }
  // The accumulators leave through wavefront-private pieces of LDS, 32 rows of 32*FC columns at a time, as whole rows.  In a
  // row of a piece the first and the second halves of all 8-column groups lie together (conflict-free 16-byte reads).
  constexpr int kLanesPerRow = 4 * FC, kStep = kWave / kLanesPerRow, kBlockPieces = 32 / kStep, kPieces = FR * kBlockPieces;
  constexpr int kAhead = 4;
  constexpr bool kO32 = OUT == kOut32;
  float* const cw = reinterpret_cast<float*>(lds_ring) + wave * (32 * R::kCStride);
  const int lr = lane / kLanesPerRow, lc = lane % kLanesPerRow;
  const int row_first = r0 + 32 * FR * wr, col_first = c0 + 32 * FC * wc;
  const int n = pr.cols - (col_first + 8 * lc);
  // piece i is row row_first + lr + kStep*i; those inside the matrix (a split's sums lie in rows of whole pieces)
  const int pieces = n >= (OUT == kOutPartial ? 1 : 8) ? (pr.rows - (row_first + lr) + kStep - 1) / kStep : 0;
  const int edge = WHOLE || OUT == kOutPartial ? 0 : pr.cols & 7, edge_at = pr.cols - edge - col_first;
  typedef std::conditional_t<WHOLE, WholePieces<kO32>, AnyPieces<kO32>> Where;
  const Where where(ep, (size_t)row_first, (size_t)col_first, lr, 8 * lc, kStep);
  Bias8 bias;
  if constexpr (OUT == kOut16) load_bias(bias, ep, (size_t)(col_first + 8 * lc), n >= 8 ? 8 : 0);
  Old8<kO32> old[kAhead];
  auto fetch_old = [&](int u, int i) {
    if constexpr (OUT != kOutPartial) {
      if (i < pieces && i < kPieces) where.load_old(old[u], ep, i);
    }
  };
#pragma unroll
  for (int u = 0; u < kAhead; u++) fetch_old(u, u);
#pragma unroll
  for (int b = 0; b < FR; b++) {
#pragma unroll
    for (int a = 0; a < FC; a++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const f32x4 v = {acc[a][b][4 * i], acc[a][b][4 * i + 1], acc[a][b][4 * i + 2], acc[a][b][4 * i + 3]};
        *reinterpret_cast<f32x4*>(cw + li * R::kCStride + 4 * (4 * a + i) + 16 * FC * lh) = v;
      }
    __builtin_amdgcn_wave_barrier();   // a wavefront's LDS operations complete in order
#pragma unroll 1
    for (int s = 0; s < kBlockPieces; s += kAhead) {
      float v[kAhead][8];
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const float* const src = cw + (kStep * (s + u) + lr) * R::kCStride + 4 * lc;
        __builtin_memcpy(v[u], src, 16);
        __builtin_memcpy(v[u] + 4, src + 16 * FC, 16);
      }
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const int i = kBlockPieces * b + s + u;
        if constexpr (OUT == kOutPartial) {
          if (i < pieces) {
            const size_t ld = ((size_t)pr.cols + 7) & ~(size_t)7;
            f32x4* const o = reinterpret_cast<f32x4*>(pr.partial + ((size_t)split * pr.rows + (row_first + lr + kStep * i)) * ld + col_first + 8 * lc);
            o[0] = f32x4{v[u][0], v[u][1], v[u][2], v[u][3]};
            o[1] = f32x4{v[u][4], v[u][5], v[u][6], v[u][7]};
          }
        } else {
          if (i < pieces) where.template finish<F16>(v[u], bias, old[u], ep, i);
          fetch_old(u, i + kAhead);
        }
      }
    }
    if constexpr (!WHOLE && OUT != kOutPartial) {
      if (edge && edge_at >= 0 && edge_at < 32 * FC)
        edge_elements<F16, kO32>(ep, (size_t)(row_first + 32 * b), (size_t)(col_first + edge_at), edge, pr.rows - (row_first + 32 * b) < 32 ? pr.rows - (row_first + 32 * b) : 32, lane,
                                 [&](int r, int e) { return cw[r * R::kCStride + (edge_at >> 1) + (e & 3) + (e >> 2) * 16 * FC]; });
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <bool F16, bool PA, bool QA, int FR, int FC, int OUT, bool WHOLE>
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(FR == 4 ? 1 : 2, FR == 4 ? 1 : 4)))
void linear_ring_kernel(const LinProd pr, const LinEpi ep) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_ring[];
  ring_tile<F16, PA, QA, FR, FC, OUT, WHOLE>(pr, ep, blockIdx.x, (int)blockIdx.y, lds_ring);
}

// Adds the splits of a product up and finishes the output.  2^shift lanes share a piece of eight columns: lane l adds the
// splits l, l + 2^shift, ... in ascending order, then the lanes' sums are added pairwise (a fixed order for given sizes).
template <bool F16, bool OUT32>
__global__ __launch_bounds__(kBlock) void linear_join_kernel(const float* __restrict__ partial, const int splits, const int rows,
                                                             const int cols, const int shift, const LinEpi ep) {
  const size_t ld = ((size_t)cols + 7) & ~(size_t)7, pieces = ld / 8;
  const size_t id = (size_t)blockIdx.x * kBlock + threadIdx.x, i = id >> shift;
  const int lane = (int)(id & ((1u << shift) - 1u));
  const bool live = i < pieces * (size_t)rows;
  const size_t row = live ? i / pieces : 0, col = live ? (i - row * pieces) * 8 : 0;
  const float* p = partial + ((size_t)lane * rows + row) * ld + col;
  const size_t step = ((size_t)rows * ld) << shift;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = 0.0f;
  if (live) {
#pragma unroll 4
    for (int s = lane; s < splits; s += 1 << shift) {
      float x[8];
      __builtin_memcpy(x, p, 32);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += x[e];
      p += step;
    }
  }
  for (int k = 0; k < shift; k++)
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] += __shfl_xor(v[e], 1 << k, kWave);
  if (!live || lane) return;
  const int n = cols - (int)col;
  Bias8 bias;
  Old8<OUT32> old;
  const Places where = places<OUT32>(ep, row, col, 0, 0, 0);
  load_bias(bias, ep, col, n);
  load_old<OUT32>(old, ep, where, 0, n, (int)col);
  finish8<F16, OUT32>(v, bias, old, ep, where, 0, n);
}

// ---- operands whose rows are not made of aligned 16-byte pieces --------------------------------------------------------------
// A copy with aligned rows, zeros behind each row's end up to the next row: the ring then runs on it.  It costs a launch and two
// passes over the operand at the memory's rate, less than matrix instructions fed from unaligned loads through registers lose over
// a long sum (777 x 1537 x 2049: 24 instead of 57 us, 2049 x 2049 x 2049: 54 instead of 90).  A short sum is not worth it: brief_product.
struct PackJob {
  const uint16_t* src;
  uint16_t* dst;
  size_t ld, ldd;   // ldd: a multiple of 8
  int rows, cols, rows_out;   // rows_out: rows written, those from `rows` on zeros
};
constexpr int kPackRows = 16;
__global__ __launch_bounds__(kBlock) void linear_pack_kernel(const PackJob a, const PackJob b) {
  const PackJob& job = blockIdx.z ? b : a;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = ((int)blockIdx.x * kWave + lane) * 8;
  if ((size_t)col >= job.ldd) return;
  for (int r0 = (int)blockIdx.y * kPackRows; r0 < job.rows_out; r0 += (int)gridDim.y * kPackRows) {
    u32x4 v[kPackRows / 4];
#pragma unroll
    for (int u = 0; u < kPackRows / 4; u++) {
      const int r = r0 + 4 * u + wave;
      v[u] = u32x4{0u, 0u, 0u, 0u};
      if (r < job.rows) v[u] = fetch_piece(job.src + (size_t)r * job.ld, col, job.cols);
    }
#pragma unroll
    for (int u = 0; u < kPackRows / 4; u++) {
      const int r = r0 + 4 * u + wave;
      if (r < job.rows_out) *reinterpret_cast<u32x4*>(job.dst + (size_t)r * job.ldd + col) = trim_piece(v[u], job.cols - col, job.cols);
    }
  }
}

// ---- few rows: the weights are read once, at the memory's rate ---------------------------------------------------------------
// Up to 64 rows (16*MT): what counts is reading W, and every wavefront keeps 8 KiB of it in flight beside the 8 KiB it works on.
// W goes from memory to registers and from there into v_mfma_f32_16x16x32, whose row operand it is; X (16 rows of it per
// instruction) comes from the caches.  A wavefront's step:
//   across (forward)   32 summed elements x 128 columns: lane (q, c) = (lane/16, lane%16) loads rows 8q .. 8q+7 of columns
//                      8c .. 8c+7 and turns that 8 x 8 block over in registers: eight fragments of column 8c + j
//   along (dX)         64 rows of W x 64 summed elements, fragments as they lie; row tiles are dealt so that a lane ends up
//                      with eight neighbouring outputs
// The four wavefronts of a workgroup take steps in turn and add up through LDS.  A strip whose sum is split over workgroups:
// up to 16 rows, the one that arrives last finishes (each wavefront for the rows that it has held in every split): partial sums
// go out and come back with the agent-scope bit (sc1: written through to, and read from, where the XCDs are coherent), complete
// (vmcnt 0) before the wavefront counts itself in; splits are added in ascending order whoever does it, and the counter is back
// at zero when the call ends.  With more rows a wavefront has too much to add, and the join kernel does it (64 x 1024 x 1024:
// 10.1 us, 13.3 without; 32 x 4096 x 4096: 13.5, 14.5).  16 x 8192 x 4096 (67 MB of weights): 14.9 us, 4.5 TB/s, where the weights
// are still in the Infinity Cache from the call before, of which reading W alone takes this grid 10.5, X 0.8, the split sums' way
// through memory 2.5; 18.7 where other layers' weights have been read since.
constexpr int kFewRows = 64, kFewWaves = 4, kFewMaxSplits = 16, kFewCounter = 32;
typedef u32x4 u32x4_u __attribute__((aligned(2)));
template <bool ALONG> struct Few {
  static constexpr int kWidth = ALONG ? 64 : 128;   // outputs of a strip
  static constexpr int kStep = ALONG ? 64 : 32;     // summed elements of a wavefront's step
  static constexpr int kAcc = ALONG ? 4 : 8;
};
struct FewArgs {
  const uint16_t* x;
  const uint16_t* w;
  size_t ldx, ldw;
  int rows, cols, sum;
  int per_split;        // a multiple of kStep
  float* partial;       // [splits][rows][cols rounded up to 8]
  uint32_t* counters;   // [strips][kFewWaves], zero, each on a cache line of its own (16 x 4096 x 4096: 11.2 us; 12.7 side by side)
};
constexpr size_t kFewStream = (size_t)48 << 20;   // elements of W: 96 MiB
constexpr int kAuxSc1 = 16;   // agent scope, in a gfx950 buffer instruction's cache policy
struct Through {
  __amdgpu_buffer_rsrc_t rs;
  __device__ __forceinline__ explicit Through(float* base) : rs(__builtin_amdgcn_make_buffer_rsrc(base, 0, 0x7ffffffc, 0x00020000)) {}
  __device__ __forceinline__ void store(uint32_t at, const float* v) const {
    u32x4 lo, hi;
    __builtin_memcpy(&lo, v, 16);
    __builtin_memcpy(&hi, v + 4, 16);
    __builtin_amdgcn_raw_buffer_store_b128(lo, rs, at, 0, kAuxSc1);
    __builtin_amdgcn_raw_buffer_store_b128(hi, rs, at + 16, 0, kAuxSc1);
  }
  __device__ __forceinline__ void load(float* v, uint32_t at) const {
    const u32x4 lo = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, kAuxSc1));
    const u32x4 hi = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at + 16, 0, kAuxSc1));
    __builtin_memcpy(v, &lo, 16);
    __builtin_memcpy(v + 4, &hi, 16);
  }
};
template <bool F16> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// STREAM: W is read past the caches.  That is faster where it is no longer there, and slower where it still is, from the last call of
// the same layer (us, cached / past the caches, 256 MB of Infinity Cache):
//   rows x sum x cols                   the same weights again    other weights in between
//   16 x 8192 x 8192, 134 MB            24.2 / 26.1               28.2 / 26.8
//   16 x 8192 x 6144, 101 MB            24.4 / 27.1               30.4 / 27.9
//   16 x 8192 x 4096, 67 MB (64 rows)   15.5 / 15.8 (21.5 / 23.3) 18.7 / 16.6 (24.6 / 23.4)
//   16 x 4096 x 4096, 34 MB (64 rows)    8.8 /  9.8 (15.7 / 18.1) 11.5 / 11.0 (17.0 / 18.4)
// A call cannot know which it is.  kFewStream supposes that less than 96 MiB may still be there and that more is not.  A model that reads
// more than the cache between two calls of a layer of 67 MB would gain 5 to 12 % from a lower bound; one that does not would lose 1 to 8.
template <bool F16, int MT, bool ALONG, bool STREAM>
__global__ __launch_bounds__(kFewWaves * kWave) void linear_few_kernel(const FewArgs a, const LinEpi ep) {
  typedef Few<ALONG> D;
  constexpr int kStride = D::kWidth + 4;
  __shared__ __attribute__((aligned(16))) float red[kFewWaves][16 * kStride];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), q = lane >> 4, c = lane & 15;
  const int strip = blockIdx.x, split = blockIdx.y, splits = gridDim.y;
  const int n0 = strip * D::kWidth;
  const int k_begin = split * a.per_split, k_end = a.sum - k_begin < a.per_split ? a.sum : k_begin + a.per_split;

  // W pieces i = 0..7 of a step.  across: row 8q + i, columns 8c..;  along: row tile i/2, half i%2 of the summed elements
  const uint16_t* wp[ALONG ? 4 : 1];
  if constexpr (ALONG) {
#pragma unroll
    for (int T = 0; T < 4; T++) {
      const int r = n0 + 32 * (T >> 1) + 8 * (c >> 2) + 4 * (T & 1) + (c & 3);
      wp[T] = a.w + (size_t)(r < a.cols ? r : a.cols - 1) * a.ldw + 8 * q;
    }
  } else {
    wp[0] = a.w + (size_t)(8 * q) * a.ldw + n0 + 8 * c;
  }
  const bool inside = ALONG || n0 + D::kWidth <= a.cols;
  const uint16_t* xp[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    const int r = 16 * m + c;
    xp[m] = a.x + (size_t)(r < a.rows ? r : a.rows - 1) * a.ldx + 8 * q;
  }
  struct Step {
    u32x4 w[8], x[MT][ALONG ? 2 : 1];
  };
  auto fetch = [&](Step& s, int k) {
    if (inside && k + D::kStep <= k_end) {
      auto piece = [&](int i) { return ALONG ? wp[i >> 1] + k + 32 * (i & 1) : wp[0] + (size_t)(k + i) * a.ldw; };
      if constexpr (STREAM) {
#pragma unroll
        for (int i = 0; i < 8; i++) s.w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_u*>(piece(i)));
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) __builtin_memcpy(&s.w[i], piece(i), 16);
      }
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int h = 0; h < (ALONG ? 2 : 1); h++) __builtin_memcpy(&s.x[m][h], xp[m] + k + 32 * h, 16);
      return;
    }
    // a step at an edge: the last rows and pieces again, trimmed to zeros behind the end of the sum
    auto row_of = [&](int i) { return k + 8 * q + i < k_end ? k + 8 * q + i : k_end - 1; };   // across
#pragma unroll
    for (int i = 0; i < 8; i++)
      s.w[i] = ALONG ? fetch_piece(wp[i >> 1] - 8 * q, k + 32 * (i & 1) + 8 * q, k_end) : fetch_piece(a.w + (size_t)row_of(i) * a.ldw, n0 + 8 * c, a.cols);
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int h = 0; h < (ALONG ? 2 : 1); h++) s.x[m][h] = fetch_piece(xp[m] - 8 * q, k + 32 * h + 8 * q, k_end);
#pragma unroll
    for (int i = 0; i < 8; i++)
      s.w[i] = ALONG ? trim_piece(s.w[i], k_end - (k + 32 * (i & 1) + 8 * q), k_end)
                     : trim_piece(s.w[i], k + 8 * q + i < k_end ? a.cols - (n0 + 8 * c) : 0, a.cols);
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int h = 0; h < (ALONG ? 2 : 1); h++) s.x[m][h] = trim_piece(s.x[m][h], k_end - (k + 32 * h + 8 * q), k_end);
  };
  f32x4 acc[MT][D::kAcc];
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int j = 0; j < D::kAcc; j++) acc[m][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto multiply = [&](const Step& s) {
    if constexpr (ALONG) {
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int m = 0; m < MT; m++) acc[m][i >> 1] = mfma16<F16>(s.w[i], s.x[m][i & 1], acc[m][i >> 1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        u32x4 f;   // column 8c + j, summed elements 8q .. 8q+7
#pragma unroll
        for (int e = 0; e < 4; e++)
          f[e] = __builtin_amdgcn_perm(s.w[2 * e + 1][j >> 1], s.w[2 * e][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int m = 0; m < MT; m++) acc[m][j] = mfma16<F16>(f, s.x[m][0], acc[m][j]);
      }
    }
  };
  {
    constexpr int kStride2 = kFewWaves * D::kStep;
    Step s0, s1;
    int k = k_begin + wave * D::kStep;
    if (k < k_end) fetch(s0, k);
    for (; k < k_end; k += 2 * kStride2) {
      if (k + kStride2 < k_end) fetch(s1, k + kStride2);
      multiply(s0);
      if (k + 2 * kStride2 < k_end) fetch(s0, k + 2 * kStride2);
      if (k + kStride2 < k_end) multiply(s1);
    }
  }
  // element (m, col) of the strip: across: lane (q, c = m) holds columns 8*(4q + i) + j in acc[..][j][i];
  // along: 32*(T/2) + 8q + 4*(T%2) + i in acc[..][T][i]
  constexpr int kPieces = D::kWidth / 8;
  const int row = t / kPieces, piece = t % kPieces, col = n0 + 8 * piece, n = a.cols - col;
  const size_t ldp = ((size_t)a.cols + 7) & ~(size_t)7;
  // what is read beside the product, on its way while the wavefronts' sums are added up
  Bias8 bias;
  Old8<false> old[MT];
  auto where = [&](int m) { return places<false>(ep, (size_t)(16 * m + row), (size_t)col, 0, 0, 0); };
  if ((MT == 1 || splits == 1) && row < 16 && n > 0) {
    load_bias(bias, ep, (size_t)col, n);
#pragma unroll
    for (int m = 0; m < MT; m++)
      if (16 * m + row < a.rows) load_old<false>(old[m], ep, where(m), 0, n, col);
  }
#pragma unroll
  for (int m = 0; m < MT; m++) {
    if (m) __syncthreads();
    if constexpr (ALONG) {
#pragma unroll
      for (int T = 0; T < 4; T++) *reinterpret_cast<f32x4*>(&red[wave][c * kStride + 32 * (T >> 1) + 8 * q + 4 * (T & 1)]) = acc[m][T];
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          *reinterpret_cast<f32x4*>(&red[wave][c * kStride + 8 * (4 * q + i) + 4 * h]) =
              f32x4{acc[m][4 * h][i], acc[m][4 * h + 1][i], acc[m][4 * h + 2][i], acc[m][4 * h + 3][i]};
    }
    __syncthreads();
    if (row < 16 && 16 * m + row < a.rows) {
      float v[8];
      __builtin_memcpy(v, &red[0][row * kStride + 8 * piece], 32);
#pragma unroll
      for (int w = 1; w < kFewWaves; w++) {
        float x[8];
        __builtin_memcpy(x, &red[w][row * kStride + 8 * piece], 32);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += x[e];
      }
      if (n <= 0) {
      } else if (splits == 1) {
        finish8<F16, false>(v, bias, old[m], ep, where(m), 0, n);
      } else {
        float* const at = a.partial + ((size_t)split * a.rows + 16 * m + row) * ldp + col;
        if constexpr (MT == 1) Through(a.partial).store((uint32_t)((at - a.partial) * 4), v);
        else __builtin_memcpy(at, v, 32);
      }
    }
  }
  if (MT > 1 || splits == 1) return;
  // a wavefront joins the rows that it holds here, with the same wavefront of the other splits
  const int first = wave * (kWave / kPieces);
  if (first >= 16 || first >= a.rows) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // its partial sums have arrived
  uint32_t* const counter = a.counters + ((size_t)strip * kFewWaves + wave) * kFewCounter;
  uint32_t arrived = 0;
  if (lane == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if ((uint32_t)__builtin_amdgcn_readfirstlane((int)arrived) != (uint32_t)splits - 1u) return;
  asm volatile("" ::: "memory");                     // nothing below is read before
  if (lane == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (row < a.rows && n > 0) {
    const Through through(a.partial);
    const uint32_t at = (uint32_t)((row * ldp + col) * 4), step = (uint32_t)(a.rows * ldp * 4);
    float x[kFewMaxSplits][8], v[8];
#pragma unroll
    for (int s = 0; s < kFewMaxSplits; s++)
      if (s < splits) through.load(x[s], at + s * step);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = x[0][e];
#pragma unroll
    for (int s = 1; s < kFewMaxSplits; s++)
      if (s < splits) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += x[s][e];
      }
    finish8<F16, false>(v, bias, old[0], ep, where(0), 0, n);
  }
}

// Up to 4 rows, forward: strips of 32 columns and no split of the sum over workgroups, whose joining costs as long as the reading of
// a small W (1 x 1024 x 8192: 8.5 us).  A wavefront's step is 128 summed elements x 32 columns: lane (kr, c2) = (lane/4, lane%4)
// loads rows 8kr .. 8kr+7 of columns 8*c2 .. and turns the 8 x 8 block over as above.  One v_mfma_f32_16x16x32 then has the four
// column groups of four different eights of summed elements (h = kr%4) as its rows, and four rows of X with the same four eights
// as its columns: of its 16 x 16 results the 4 x 4 blocks with equal h are sums, the others are dropped.  The wavefronts of a
// workgroup take steps in turn; two neighbouring strips, which share every cache line of W, are dealt to one XCD.
constexpr int kOneRows = 4, kOneWidth = 32, kOneStep = 128, kOneSum = 2048;
template <bool F16, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void linear_one_kernel(const FewArgs a, const LinEpi ep) {
  __shared__ __attribute__((aligned(16))) float red[WAVES * 4][kOneRows * kOneWidth + 4];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), kr = lane >> 2, c2 = lane & 3;
  const int b = (int)blockIdx.x, full = (int)gridDim.x & ~15;
  const int strip = b < full ? (b & ~15) + 2 * (b & 7) + ((b >> 3) & 1) : b;
  const int n0 = strip * kOneWidth;
  const uint16_t* const xrow = a.x + (size_t)(c2 < a.rows ? c2 : a.rows - 1) * a.ldx;
  const bool inside = n0 + kOneWidth <= a.cols;
  struct Step { u32x4 w[8], x; };
  auto fetch = [&](Step& s, int k) {
    const int k8 = k + 8 * kr;
    if (inside && k + kOneStep <= a.sum) {
#pragma unroll
      for (int i = 0; i < 8; i++) __builtin_memcpy(&s.w[i], a.w + (size_t)(k8 + i) * a.ldw + n0 + 8 * c2, 16);
      __builtin_memcpy(&s.x, xrow + k8, 16);
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) s.w[i] = fetch_piece(a.w + (size_t)(k8 + i < a.sum ? k8 + i : a.sum - 1) * a.ldw, n0 + 8 * c2, a.cols);
    s.x = fetch_piece(xrow, k8, a.sum);
#pragma unroll
    for (int i = 0; i < 8; i++) s.w[i] = trim_piece(s.w[i], k8 + i < a.sum ? a.cols - (n0 + 8 * c2) : 0, a.cols);
    s.x = trim_piece(s.x, a.sum - k8, a.sum);
  };
  f32x4 acc[8];
#pragma unroll
  for (int j = 0; j < 8; j++) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto multiply = [&](const Step& s) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      u32x4 f;
#pragma unroll
      for (int e = 0; e < 4; e++) f[e] = __builtin_amdgcn_perm(s.w[2 * e + 1][j >> 1], s.w[2 * e][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
      acc[j] = mfma16<F16>(f, s.x, acc[j]);
    }
  };
  {
    constexpr int kTurn = WAVES * kOneStep;
    Step s0, s1;
    int k = wave * kOneStep;
    if (k < a.sum) fetch(s0, k);
    for (; k < a.sum; k += 2 * kTurn) {
      if (k + kTurn < a.sum) fetch(s1, k + kTurn);
      multiply(s0);
      if (k + 2 * kTurn < a.sum) fetch(s0, k + 2 * kTurn);
      if (k + kTurn < a.sum) multiply(s1);
    }
  }
  // lane (h, h', m) = (lane/16, lane/4%4, lane%4) with h == h' holds row m, columns 8i + j, in acc[j][i]
  const int h = lane >> 4, m = lane & 3;
  if (h == ((lane >> 2) & 3)) {
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int u = 0; u < 2; u++)
        *reinterpret_cast<f32x4*>(&red[wave * 4 + h][m * kOneWidth + 8 * i + 4 * u]) =
            f32x4{acc[4 * u][i], acc[4 * u + 1][i], acc[4 * u + 2][i], acc[4 * u + 3][i]};
  }
  __syncthreads();
  // 128 sums of 4*WAVES: four threads each, then one
  const int at = t & 127, part = t >> 7;
  constexpr int kParts = WAVES / 2;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4 * WAVES / kParts; i++) s += red[part * (4 * WAVES / kParts) + i][at];
  __syncthreads();
  red[part][at] = s;
  __syncthreads();
  const int row = t >> 2, col = n0 + 8 * (t & 3), n = a.cols - col;
  if (t < 16 && row < a.rows && n > 0) {
    float v[8];
    __builtin_memcpy(v, &red[0][8 * t], 32);
#pragma unroll
    for (int p = 1; p < kParts; p++) {
      float x[8];
      __builtin_memcpy(x, &red[p][8 * t], 32);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += x[e];
    }
    const Places where = places<false>(ep, (size_t)row, (size_t)col, 0, 0, 0);
    Bias8 bias;
    Old8<false> old;
    load_bias(bias, ep, (size_t)col, n);
    load_old<false>(old, ep, where, 0, n, col);
    finish8<F16, false>(v, bias, old, ep, where, 0, n);
  }
}

// ---- dz and the column sums ------------------------------------------------------------------------------------------------
// dz = dY * act'(pre), rounded to the operands' type into the workspace (aligned rows, zeros up to a multiple of 8 columns), and
// fp32 sums over a chunk of rows of the unrounded dz.  The rounding is the matrix instructions': both their operands have the type of W
// and X, and to carry dz in two parts would double both products.  It is the only rounding beside the output's own, and as large: dX
// and dW of a bf16 layer are off by 2.35e-3 of their norm, 1.66e-3 with an unrounded dz.  LANES lanes share a row's strip of 8*LANES columns, a workgroup of WAVES
// wavefronts works on WAVES * 64/LANES rows at a time, ROWS times that in flight.
//   64, 4, 2     many rows (8192 x 4096, gelu_tanh: 45 us; 48 with four in flight): a strip of 512 columns, chunks of rows over the chip, linear_db_kernel adds the chunks up
//   16, 16, 1    up to 64 rows, all at once: one chunk, its sums are db itself (`add`: added to it)
template <bool F16, int LANES, int WAVES, int ROWS>
__global__ __launch_bounds__(WAVES * kWave) void linear_dz_kernel(const uint16_t* __restrict__ dY, const size_t lddy,
                                                                  const uint16_t* __restrict__ pre, const size_t ldp,
                                                                  uint16_t* __restrict__ dz, const size_t lddz, float* __restrict__ sums,
                                                                  const int M, const int N, const int act, const int rows_per_chunk,
                                                                  const int add) {
  constexpr int kPass = WAVES * (kWave / LANES), kWidth = 8 * LANES;
  __shared__ float part[WAVES][kWidth + 8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, piece = lane % LANES;
  const int col = (int)blockIdx.x * kWidth + piece * 8, n = N - col;
  const int m0 = (int)blockIdx.y * rows_per_chunk;
  const int m1 = M - m0 < rows_per_chunk ? M : m0 + rows_per_chunk;
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; e++) s[e] = 0.0f;
  if (n > 0) {
    for (int m = m0 + wave * (kWave / LANES) + lane / LANES; m < m1; m += ROWS * kPass) {
      u32x4 gv[ROWS], zv[ROWS];
#pragma unroll
      for (int u = 0; u < ROWS; u++) {
        const int r = m + u * kPass;
        if (r < m1) {
          gv[u] = fetch_piece(dY + (size_t)r * lddy, col, N);
          if (act != CCN_ACT_NONE) zv[u] = fetch_piece(pre + (size_t)r * ldp, col, N);
        }
      }
#pragma unroll
      for (int u = 0; u < ROWS; u++) {
        const int r = m + u * kPass;
        if (r < m1) {
          float g[8];
          unpack<F16>(trim_piece(gv[u], n, N), g);
          if (act != CCN_ACT_NONE) {   // (behind the row's end dY and pre are zeros, and so is the product)
            float z[8];
            unpack<F16>(trim_piece(zv[u], n, N), z);
            act_slopes(act, z, g);
          }
          if (dz) *reinterpret_cast<u32x4*>(dz + (size_t)r * lddz + col) = pack<F16>(g);
#pragma unroll
          for (int e = 0; e < 8; e++) s[e] += g[e];
        }
      }
    }
  }
  if (!sums) return;
#pragma unroll
  for (int off = LANES; off < kWave; off <<= 1)
#pragma unroll
    for (int e = 0; e < 8; e++) s[e] += __shfl_xor(s[e], off, kWave);
  if (lane < LANES) {
#pragma unroll
    for (int e = 0; e < 8; e++) part[wave][piece * 8 + e] = s[e];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < kWidth; c += WAVES * kWave) {
    const int at = (int)blockIdx.x * kWidth + c;
    if (at < N) {
      float x = part[0][c];
#pragma unroll
      for (int w = 1; w < WAVES; w++) x += part[w][c];
      float* const o = sums + (size_t)blockIdx.y * N + at;
      *o = add ? *o + x : x;
    }
  }
}
// db[n] = (db[n] +) the sum of the chunks' sums: 64 columns per workgroup of WAVES wavefronts, each every WAVES-th chunk.
struct DbArgs {
  const float* sums;
  float* db;
  int cols, chunks, accumulate;
};
template <int WAVES> __device__ __forceinline__ void add_chunks(const DbArgs& a, const int block, float* const part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = block * kWave + lane;
  float s = 0.0f;
  if (c < a.cols) {
#pragma unroll 8
    for (int k = wave; k < a.chunks; k += WAVES) s += a.sums[(size_t)k * a.cols + c];
  }
  part[wave * kWave + lane] = s;
  __syncthreads();
  if (wave == 0 && c < a.cols) {
    float x = part[lane];
#pragma unroll
    for (int w = 1; w < WAVES; w++) x += part[w * kWave + lane];
    a.db[c] = a.accumulate ? a.db[c] + x : x;
  }
}
constexpr int kDbWaves = 16;
__global__ __launch_bounds__(kDbWaves * kWave) void linear_db_kernel(const DbArgs a) {
  __shared__ float part[kDbWaves * kWave];
  add_chunks<kDbWaves>(a, (int)blockIdx.x, part);
}

// Both products of a backward pass, and db, in one launch: the tiles of small ones run side by side on CUs that one product alone
// would leave idle, and two launches are saved.  SPLIT: 1 the sum of dX, or 2 that of dW, is split over workgroups (the join kernel
// adds the splits up).  The product whose workgroups take longer is dealt out first.
struct PairArgs {
  LinProd x, w;    // dX, dW
  LinEpi ex, ew;
  DbArgs db;
  int nx, nw, w_first;   // workgroups of each; those behind them are db's
};
template <bool F16, bool OUT32, bool WHOLE, int SPLIT>
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(2, 4))) void linear_pair_kernel(const PairArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_ring[];
  const int b = (int)blockIdx.x;
  if (b >= a.nx + a.nw) {
    add_chunks<kBlock / kWave>(a.db, b - a.nx - a.nw, reinterpret_cast<float*>(lds_ring));
    return;
  }
  if (a.w_first ? b >= a.nw : b < a.nx) {
    const int at = a.w_first ? b - a.nw : b, tiles = a.x.tiles_r * a.x.tiles_c, split = SPLIT == 1 ? at / tiles : 0;
    ring_tile<F16, true, true, 2, 2, SPLIT == 1 ? kOutPartial : kOut16, WHOLE || SPLIT == 1>(a.x, a.ex, (uint32_t)(at - split * tiles), split, lds_ring);
  } else {
    const int at = a.w_first ? b : b - a.nx, tiles = a.w.tiles_r * a.w.tiles_c, split = SPLIT == 2 ? at / tiles : 0;
    ring_tile<F16, false, false, 2, 2, SPLIT == 2 ? kOutPartial : OUT32 ? kOut32 : kOut16, WHOLE || SPLIT == 2>(a.w, a.ew, (uint32_t)(at - split * tiles), split,
                                                                                                          lds_ring);
  }
}

constexpr size_t kMaxLd = (size_t)1 << 22;
constexpr int kMaxChunks = 256;      // row chunks of the column sums
constexpr int kMaxSplits = 16;

#define CCN_TRY(expr)                  \
  do {                                 \
    const int _rc = (expr);            \
    if (_rc != CCN_OK) return _rc;     \
  } while (0)

inline size_t round8(size_t n) { return (n + 7) & ~(size_t)7; }
// Rows of the plan's own matrices start on cache lines: requests of 128 bytes that straddle two of them cost a fifth of a product's
// time (777 x 1536 x 2048 15.0 us, 777 x 1544 x 2048 18.7).
inline size_t pitch(size_t n) { return (n + 63) & ~(size_t)63; }
inline bool aligned2(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace ccn

using namespace ccn;

struct ccn_linear_plan {
  int device = -1;
  int max_m = 0, max_n = 0, max_k = 0;
  uint16_t* dz = nullptr;
  uint16_t* px = nullptr;    // aligned copies of X and W
  uint16_t* pw = nullptr;    // (nullptr: up to kFewRows rows)
  float* sums = nullptr;
  float* partial = nullptr;
  size_t partial_floats = 0;
  uint32_t* counters = nullptr;   // arrivals per strip of the few-row kernels; zero between calls
};

namespace {

// A 16-bit matrix as the products take it.  extent: columns that may be read (its width, or that rounded up to 8).
struct Operand {
  const uint16_t* p;
  size_t ld;
  int rows, extent;
};
// Whether the ring can fetch it: aligned 16-byte pieces, and as a sum's rows ("across") only whole ones.
bool ring_fetches(const Operand& o, bool along) {
  return aligned16(o.p) && o.ld % 8 == 0 && o.ld <= kRMaxLd && (along || o.extent % 8 == 0);
}

// More than 64 KiB of dynamic LDS have to be asked for, once for every kernel and device.
int allow_lds(const void* kernel, int bytes, std::atomic<uint32_t>& devices) {
  int dev = -1;
  CCN_HIP(hipGetDevice(&dev));
  if (dev < 0 || dev > 31) return CCN_ENODEV;
  if (devices.load(std::memory_order_relaxed) >> dev & 1u) return CCN_OK;
  CCN_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  devices.fetch_or(1u << dev, std::memory_order_relaxed);
  return CCN_OK;
}
template <bool F16, bool PA, bool QA, int FR, int FC, int OUT, bool WHOLE>
int launch_ring(const LinProd& pr, const LinEpi& ep, int splits, hipStream_t s) {
  constexpr int kLds = Ring<FR, FC>::kLds;
  static std::atomic<uint32_t> devices{0};
  CCN_TRY(allow_lds((const void*)linear_ring_kernel<F16, PA, QA, FR, FC, OUT, WHOLE>, kLds, devices));
  const int lds = pr.brief ? Ring<FR, FC>::kBriefLds : kLds;
  hipLaunchKernelGGL((linear_ring_kernel<F16, PA, QA, FR, FC, OUT, WHOLE>), dim3((unsigned)(pr.tiles_r * pr.tiles_c), (unsigned)splits),
                     dim3(kBlock), lds, s, pr, ep);
  CCN_HIP(hipGetLastError());
  return CCN_OK;
}
template <bool F16, bool OUT32>
int launch_join(const float* partial, int rows, int cols, int splits, const LinEpi& ep, hipStream_t s) {
  const size_t pieces = (size_t)rows * (((size_t)cols + 7) / 8);
  int shift = 0;   // lanes per piece: until there are 2^16 threads
  while (shift < 4 && (2 << shift) <= splits && (pieces << shift) < 65536) shift++;
  const size_t blocks = ((pieces << shift) + kBlock - 1) / kBlock;
  if (blocks > 0x7fffffffull) return CCN_ERANGE;
  hipLaunchKernelGGL((linear_join_kernel<F16, OUT32>), dim3((unsigned)blocks), dim3(kBlock), 0, s, partial, splits, rows, cols, shift, ep);
  CCN_HIP(hipGetLastError());
  return CCN_OK;
}
template <bool F16, bool PA, bool QA, int FR, int FC>
int product_ring(LinProd& pr, const LinEpi& ep, bool out32, bool whole, int splits, hipStream_t s) {
  pr.tiles_r = (pr.rows + 64 * FR - 1) / (64 * FR);
  pr.tiles_c = (pr.cols + 64 * FC - 1) / (64 * FC);
  if constexpr (FR == 2) {
    if (splits > 1) {
      CCN_TRY((launch_ring<F16, PA, QA, FR, FC, kOutPartial, true>(pr, ep, splits, s)));
      return out32 ? launch_join<F16, true>(pr.partial, pr.rows, pr.cols, splits, ep, s) : launch_join<F16, false>(pr.partial, pr.rows, pr.cols, splits, ep, s);
    }
  }
  if (out32) {
    if constexpr (!PA && !QA) {
      if (whole) return launch_ring<F16, PA, QA, FR, FC, kOut32, true>(pr, ep, 1, s);
      return launch_ring<F16, PA, QA, FR, FC, kOut32, false>(pr, ep, 1, s);
    } else {
      return CCN_EINVAL;
    }
  }
  if (whole) return launch_ring<F16, PA, QA, FR, FC, kOut16, true>(pr, ep, 1, s);
  return launch_ring<F16, PA, QA, FR, FC, kOut16, false>(pr, ep, 1, s);
}

template <bool F16, bool ALONG, bool STREAM> void launch_few(dim3 grid, dim3 block, const FewArgs& a, const LinEpi& ep, hipStream_t s) {
  switch ((a.rows + 15) / 16) {
    case 1: hipLaunchKernelGGL((linear_few_kernel<F16, 1, ALONG, STREAM && !ALONG>), grid, block, 0, s, a, ep); break;
    case 2: hipLaunchKernelGGL((linear_few_kernel<F16, 2, ALONG, STREAM && !ALONG>), grid, block, 0, s, a, ep); break;
    case 3: hipLaunchKernelGGL((linear_few_kernel<F16, 3, ALONG, STREAM && !ALONG>), grid, block, 0, s, a, ep); break;
    default: hipLaunchKernelGGL((linear_few_kernel<F16, 4, ALONG, STREAM && !ALONG>), grid, block, 0, s, a, ep); break;
  }
}
// Up to kFewRows rows.
template <bool F16, bool ALONG>
int product_few(ccn_linear_plan* plan, const uint16_t* x, size_t ldx, const uint16_t* w, size_t ldw, int rows, int cols, int sum,
                const LinEpi& ep, int cus, hipStream_t s) {
  typedef Few<ALONG> D;
  FewArgs a;
  a.x = x;
  a.w = w;
  a.ldx = ldx;
  a.ldw = ldw;
  a.rows = rows;
  a.cols = cols;
  a.sum = sum;
  a.counters = plan->counters;
  if constexpr (!ALONG) {
    // (one row, us with this kernel / with the other: 1024 x 1024 4.8 / 5.9, 2048 x 1024 6.6 / 7.0, 1024 x 8192 6.5 / 8.5, but
    // 4096 x 1024 8.8 / 7.5 and 4096 x 4096 13.8 / 10.8: a CU alone reads a long strip too slowly)
    const int narrow = (cols + kOneWidth - 1) / kOneWidth;
    if (rows <= kOneRows && sum <= kOneSum) {
      if (narrow >= cus) hipLaunchKernelGGL((linear_one_kernel<F16, 8>), dim3((unsigned)narrow), dim3(8 * kWave), 0, s, a, ep);
      else hipLaunchKernelGGL((linear_one_kernel<F16, 16>), dim3((unsigned)narrow), dim3(16 * kWave), 0, s, a, ep);
      CCN_HIP(hipGetLastError());
      return CCN_OK;
    }
  }
  const int strips = (cols + D::kWidth - 1) / D::kWidth, steps = (sum + D::kStep - 1) / D::kStep;
  // a workgroup for every CU, each wavefront with a step at least
  int splits = (cus + strips - 1) / strips;
  if (splits > steps / kFewWaves) splits = steps / kFewWaves;
  if (splits > kFewMaxSplits) splits = kFewMaxSplits;
  if ((size_t)(splits > 1 ? splits : 0) * (size_t)rows * round8((size_t)cols) > plan->partial_floats) splits = 1;
  if (splits < 1) splits = 1;
  a.per_split = ((steps + splits - 1) / splits) * D::kStep;
  splits = (sum + a.per_split - 1) / a.per_split;   // no empty split
  a.partial = plan->partial;
  const dim3 grid((unsigned)strips, (unsigned)splits), block(kFewWaves * kWave);
  if (!ALONG && (size_t)cols * (size_t)sum > kFewStream) launch_few<F16, ALONG, true>(grid, block, a, ep, s);
  else launch_few<F16, ALONG, false>(grid, block, a, ep, s);
  CCN_HIP(hipGetLastError());
  if (rows > 16 && splits > 1) return launch_join<F16, false>(a.partial, rows, cols, splits, ep, s);
  return CCN_OK;
}

// How a product runs on the ring, by estimated time.  Measured in us: a step of 64 summed elements takes a CU 0.40 with one
// 128 x 128 tile on it, 1.0 with two, 0.9 with a 256 x 128 tile and 1.6 with a 256 x 256 one; 5, 6 or 8 go into the first loads and
// the output; a split adds 1.8 for the join kernel and 0.4 per MB of partial sums, written and read.
//   rows x sum x cols        256 x 256    256 x 128    128 x 128, splits 1 / 2 / 4 / 8
//   256 x 4096 x 4096        75           -            28 / 22 / 22 / 31
//   1024 x 8192 x 1024       133          -            46.7 / 32.3 / 32.6 / 37.4
//   1024 x 1024 x 1024       30.2         -            11.9 / 13.4 / 15.6 / 22.9
//   2048 x 4096 x 4096       79           62.9         65.7
//   4096 x 4096 x 4096       107.6        122.6        129
enum RingTile { kTile256, kTile256x128, kTile128 };
struct RingPlan {
  RingTile tile;
  int splits;
  double us;
};
RingPlan choose_ring(int rows, int cols, int sum, size_t partial_floats, int cus) {
  const auto tiles = [&](int r, int c) { return (double)((rows + r - 1) / r) * (double)((cols + c - 1) / c); };
  const double steps = (double)((sum + 63) / 64), t128 = tiles(128, 128);
  const size_t each = (size_t)rows * round8((size_t)cols);
  RingPlan best{kTile256, 1, 8.0 + 1.6 * steps * std::ceil(tiles(256, 256) / cus)};
  const double half = 6.0 + 0.9 * steps * std::ceil(tiles(256, 128) / cus);
  if (half < best.us) best = RingPlan{kTile256x128, 1, half};
  for (int s = 1; s <= kMaxSplits; s++) {
    if (s > 1 && (s * 2.0 > steps || (double)s * t128 > 2.0 * cus || (size_t)s * each > partial_floats)) break;
    const double deep = std::ceil(s * t128 / cus);
    double t = 5.0 + std::ceil(steps / s) * (deep < 2.0 ? 0.40 : 0.5 * deep);
    if (s > 1) t += 1.8 + 0.4e-6 * 4.0 * (double)s * (double)each;
    if (t < best.us) best = RingPlan{kTile128, s, t};
  }
  return best;
}

// Whether a product does without the ring: short sums (`brief`), where there are more tiles than CUs (four workgroups then share a
// CU: 65 x 4096 x 4096, dW: 33 instead of 48 us for a whole backward pass), or where an operand would have to be copied first (us,
// M x N x K, rows of odd length, through registers / with the copy: forward 129 x 129 x 129 9.8 / 10.3, 200 x 131 x 135 9.8 / 12.2, 777 x 2049 x
// 190 10.9 / 12.3, 2000 x 1001 x 190 12.8 / 12.6; backward 129 x 129 x 129 12.4 / 14.2, 100 x 515 x 2049 17.5 / 18.2, 190 x 2001 x 2001 33.9 / 32.5.
// Rows of fewer than 8 elements are fetched one by one: 100 x 5 x 190 13.0 / 9.8).
constexpr int kBriefSum = 192;
bool brief_product(const Operand& p, bool p_along, const Operand& q, bool q_along, int rows, int cols, int sum, int cus) {
  if (sum > kBriefSum) return false;
  return (size_t)((rows + 127) / 128) * (size_t)((cols + 127) / 128) > (size_t)cus || !ring_fetches(p, p_along) || !ring_fetches(q, q_along);
}
// A product whose operands the ring can fetch (or a brief one): C [rows x cols].
LinProd make_product(const ccn_linear_plan* plan, const Operand& p, bool p_along, const Operand& q, bool q_along, int rows, int cols, int sum, int cus) {
  LinProd pr;
  pr.p = p.p;
  pr.q = q.p;
  pr.ldp = p.ld;
  pr.ldq = q.ld;
  pr.rows = rows;
  pr.cols = cols;
  pr.sum = sum;
  pr.read_r = p_along ? rows : p.extent;
  pr.read_c = q_along ? cols : q.extent;
  pr.tiles_r = (rows + 127) / 128;
  pr.tiles_c = (cols + 127) / 128;
  pr.per_split = 0;
  pr.brief = brief_product(p, p_along, q, q_along, rows, cols, sum, cus) ? 1 : 0;
  pr.partial = plan->partial;
  return pr;
}
// Whether every piece of the output's rows (and of what is read or written beside it) is inside its row and 16-byte aligned.
bool whole_pieces(const LinEpi& ep, int cols, bool out32) {
  const auto ok = [](const void* x, size_t ld, int size) {
    return aligned16(x) && ld % (size_t)(16 / size) == 0 && ld * (size_t)size <= 2 * kRMaxLd;
  };
  return cols % 8 == 0 && ok(ep.out, ep.ldo, out32 ? 4 : 2) && (!ep.resid || ok(ep.resid, ep.ldr, 2)) && (!ep.pre || ok(ep.pre, ep.ldp, 2));
}
template <bool F16, bool PA, bool QA>
int run_product(LinProd& pr, const LinEpi& ep, bool out32, RingPlan how, hipStream_t s) {
  if ((size_t)pr.tiles_r * (size_t)pr.tiles_c > 0x7fffffffull) return CCN_ERANGE;
  const bool whole = whole_pieces(ep, pr.cols, out32);
  const int steps = (pr.sum + 63) / 64;
  pr.per_split = 64 * ((steps + how.splits - 1) / how.splits);
  if (how.splits > 1) how.splits = (pr.sum + pr.per_split - 1) / pr.per_split;   // no empty split
  if (how.tile == kTile256) return product_ring<F16, PA, QA, 4, 4>(pr, ep, out32, whole, 1, s);
  if (how.tile == kTile256x128) return product_ring<F16, PA, QA, 4, 2>(pr, ep, out32, whole, 1, s);
  return product_ring<F16, PA, QA, 2, 2>(pr, ep, out32, whole, how.splits, s);
}
template <bool F16, bool OUT32, bool WHOLE, int SPLIT> int launch_pair(const PairArgs& a, hipStream_t s) {
  constexpr int kLds = Ring<2, 2>::kLds;
  static std::atomic<uint32_t> devices{0};
  CCN_TRY(allow_lds((const void*)linear_pair_kernel<F16, OUT32, WHOLE, SPLIT>, kLds, devices));
  const int lds = a.x.brief && a.w.brief ? Ring<2, 2>::kBriefLds : kLds;
  const int blocks = a.nx + a.nw + (a.db.db ? (a.db.cols + kWave - 1) / kWave : 0);
  hipLaunchKernelGGL((linear_pair_kernel<F16, OUT32, WHOLE, SPLIT>), dim3((unsigned)blocks), dim3(kBlock), lds, s, a);
  CCN_HIP(hipGetLastError());
  return CCN_OK;
}
template <bool F16, bool OUT32> int product_pair(const PairArgs& a, int split, int splits, hipStream_t s) {
  const bool wx = whole_pieces(a.ex, a.x.cols, false), ww = whole_pieces(a.ew, a.w.cols, OUT32);   // (of a split product: the join's)
  if (split == 1) {
    CCN_TRY((ww ? launch_pair<F16, OUT32, true, 1>(a, s) : launch_pair<F16, OUT32, false, 1>(a, s)));
    return launch_join<F16, false>(a.x.partial, a.x.rows, a.x.cols, splits, a.ex, s);
  }
  if (split == 2) {
    CCN_TRY((wx ? launch_pair<F16, OUT32, true, 2>(a, s) : launch_pair<F16, OUT32, false, 2>(a, s)));
    return launch_join<F16, OUT32>(a.w.partial, a.w.rows, a.w.cols, splits, a.ew, s);
  }
  return wx && ww ? launch_pair<F16, OUT32, true, 0>(a, s) : launch_pair<F16, OUT32, false, 0>(a, s);
}

// How the two run side by side, by estimated time: as long as a workgroup's longest sum, and as all the work dealt over the CUs, in
// steps of 64 summed elements (0.45 us), what a workgroup does before and after its sum being worth 8 of them.  Splitting one of
// the sums pays where it is much the longer one; it costs a join kernel (5.5 us with its launch, and 0.4 per MB of partial sums), and
// is left alone beside a product of many tiles with a short sum, which want the CUs themselves.  (Sizes alone decide: how an
// operand is aligned does not change a result's bits.)  Whole backward passes in us, unsplit / split:
//   M x N x K  128 x 1024 x 1024 12.9 / 14.9    1001 x 2049 x 515 30.9 / 28.2    8192 x 256 x 256 25.9 / 17.7    700 x 8000 x 128 31.1 / 21.1
// split: 0 none, 1 the first one's, 2 the second one's.
struct PairPlan {
  int split, splits;
  double us;
};
PairPlan choose_pair(const LinProd& x, const LinProd& w, size_t partial_floats, int cus) {
  const double sx = (x.sum + 63) / 64, sw = (w.sum + 63) / 64, tx = (double)x.tiles_r * x.tiles_c, tw = (double)w.tiles_r * w.tiles_c;
  const auto time = [&](double nx, double nw) {   // splits of each
    const double lx = std::ceil(sx / nx) + 8.0, lw = std::ceil(sw / nw) + 8.0;
    return 1.0 + 0.45 * std::fmax(std::fmax(lx, lw), (tx * nx * lx + tw * nw * lw) / cus);
  };
  PairPlan best{0, 1, time(1, 1)};
  if ((x.sum <= kBriefSum && tx > cus) || (w.sum <= kBriefSum && tw > cus)) return best;
  for (int which = 1; which <= 2; which++) {
    const LinProd& p = which == 1 ? x : w;
    const size_t each = (size_t)p.rows * round8((size_t)p.cols);
    for (int n = 2; n <= kMaxSplits && n * 128 <= p.sum && (size_t)n * each <= partial_floats; n++) {
      const double t = (which == 1 ? time(n, 1) : time(1, n)) + 5.5 + 0.4e-6 * 4.0 * (double)n * (double)each;
      if (t < best.us) best = PairPlan{which, n, t};
    }
  }
  return best;
}

// Aligned copies of up to two operands into the plan (nullptr: none).
int pack(const Operand* a, int a_cols, uint16_t* a_to, const Operand* b, int b_cols, uint16_t* b_to, int b_rows_out, hipStream_t s) {
  const auto job = [](const Operand* o, int cols, uint16_t* to, int rows_out) {
    return o ? PackJob{o->p, to, o->ld, pitch((size_t)cols), o->rows, cols, rows_out} : PackJob{};
  };
  PackJob x = job(a, a_cols, a_to, a ? a->rows : 0), y = job(b, b_cols, b_to, b_rows_out);
  if (!a) {
    x = y;
    y = PackJob{};
  }
  const size_t width = x.ldd > y.ldd ? x.ldd : y.ldd;
  const int rows = x.rows_out > y.rows_out ? x.rows_out : y.rows_out, gy = (rows + kPackRows - 1) / kPackRows;
  const dim3 grid((unsigned)((width + 511) / 512), (unsigned)(gy < 65535 ? gy : 65535), a && b ? 2u : 1u);
  hipLaunchKernelGGL(linear_pack_kernel, grid, dim3(kBlock), 0, s, x, y);
  CCN_HIP(hipGetLastError());
  return CCN_OK;
}

int check_plan(const ccn_linear_plan* plan, int M, int N, int K, int act, const DeviceInfo** di) {
  if (!plan || M < 0 || N < 1 || K < 1 || act < CCN_ACT_NONE || act > CCN_ACT_SILU) return CCN_EINVAL;
  if (M > plan->max_m || N > plan->max_n || K > plan->max_k) return CCN_ERANGE;
  const int rc = current_device_info(di);
  if (rc != CCN_OK) return rc;
  return (*di)->device == plan->device ? CCN_OK : CCN_EINVAL;
}
// A 16-bit matrix argument: 0, or why it is refused.
int check16(const void* p, size_t ld, int cols) {
  if (!p || !aligned2(p) || ld < (size_t)cols) return CCN_EINVAL;
  return ld > kMaxLd ? CCN_ERANGE : CCN_OK;
}

template <bool F16>
int linear_forward(ccn_linear_plan* plan, const uint16_t* X, size_t ldx, const uint16_t* W, size_t ldw, const float* bias,
                   const uint16_t* resid, size_t ldr, uint16_t* Y, size_t ldy, uint16_t* pre, size_t ldp, int M, int N, int K,
                   int act, void* stream) {
  const DeviceInfo* di = nullptr;
  CCN_TRY(check_plan(plan, M, N, K, act, &di));
  if (M == 0) return CCN_OK;
  CCN_TRY(check16(X, ldx, K));
  CCN_TRY(check16(W, ldw, N));
  CCN_TRY(check16(Y, ldy, N));
  if (resid) CCN_TRY(check16(resid, ldr, N));
  if (pre) CCN_TRY(check16(pre, ldp, N));
  if (!aligned4(bias)) return CCN_EINVAL;
  const LinEpi ep{bias, resid, pre, Y, ldr, ldp, ldy, act, 0};
  hipStream_t s = as_stream(stream);
  if (M <= kFewRows) return product_few<F16, false>(plan, X, ldx, W, ldw, M, N, K, ep, di->cu_count, s);
  Operand x{X, ldx, M, K}, w{W, ldw, K, N};
  const bool cx = !ring_fetches(x, true), cw = !ring_fetches(w, false);
  int sum = K;
  if ((cx || cw) && !brief_product(x, true, w, false, M, N, K, di->cu_count)) {
    // both copied: the sum goes on over zeros to whole steps, and has no last step through registers (K = 1537: 2 us less)
    if (cx && cw) sum = (int)pitch((size_t)K);
    CCN_TRY(pack(cx ? &x : nullptr, K, plan->px, cw ? &w : nullptr, N, plan->pw, sum, s));
    if (cx) x = Operand{plan->px, pitch((size_t)K), M, (int)round8((size_t)K)};
    if (cw) w = Operand{plan->pw, pitch((size_t)N), sum, (int)round8((size_t)N)};
  }
  LinProd pr = make_product(plan, x, true, w, false, M, N, sum, di->cu_count);
  return run_product<F16, true, false>(pr, ep, false, choose_ring(M, N, K, plan->partial_floats, di->cu_count), s);
}

template <bool F16>
int linear_backward(ccn_linear_plan* plan, const uint16_t* dY, size_t lddy, const uint16_t* pre, size_t ldp, const uint16_t* X,
                    size_t ldx, const uint16_t* W, size_t ldw, uint16_t* dX, size_t lddx, void* dW, size_t lddw, int dw_type,
                    float* db, int accumulate, int M, int N, int K, int act, void* stream) {
  const DeviceInfo* di = nullptr;
  CCN_TRY(check_plan(plan, M, N, K, act, &di));
  const bool dw32 = dw_type == CCN_TYPE_F32;
  if (!dw32 && dw_type != (F16 ? CCN_TYPE_F16 : CCN_TYPE_BF16)) return CCN_EINVAL;
  if (accumulate && dW && !dw32) return CCN_EINVAL;
  if (dW && (lddw < (size_t)N || !(dw32 ? aligned4(dW) : aligned2(dW)))) return CCN_EINVAL;
  if (dW && lddw > kMaxLd) return CCN_ERANGE;
  if (!aligned4(db)) return CCN_EINVAL;
  if (M > 0) {
    CCN_TRY(check16(dY, lddy, N));
    if (act != CCN_ACT_NONE) CCN_TRY(check16(pre, ldp, N));
    if (dX) {
      CCN_TRY(check16(dX, lddx, K));
      CCN_TRY(check16(W, ldw, N));
    }
    if (dW) CCN_TRY(check16(X, ldx, K));
  }
  hipStream_t s = as_stream(stream);
  // dz goes to the workspace when there is an activation, and when dY is not laid out as the ring wants it
  Operand g{dY, lddy, M, N};
  const bool few = M <= kFewRows;   // dX by the kernel for few rows, which takes anything
  Operand x{X, ldx, M, K}, w{W, ldw, K, N};
  const bool brief_dx = dX && !few && brief_product(g, true, w, true, M, K, N, di->cu_count);
  const bool brief_dw = dW && brief_product(x, false, g, false, K, N, M, di->cu_count);
  const bool want_dz = M > 0 && (act != CCN_ACT_NONE ? dX || dW
                                                     : (dW && !brief_dw && !ring_fetches(g, false)) || (dX && !few && !brief_dx && !ring_fetches(g, true)));
  if (want_dz) g = Operand{plan->dz, pitch((size_t)N), M, (int)round8((size_t)N)};
  int chunks = 0;
  bool db_left = db != nullptr;
  if (M > 0 && (want_dz || db)) {
    uint16_t* const to = want_dz ? plan->dz : nullptr;
    if (few) {
      hipLaunchKernelGGL((linear_dz_kernel<F16, 16, 16, 1>), dim3((unsigned)((N + 127) / 128)), dim3(16 * kWave), 0, s, dY, lddy, pre, ldp, to, g.ld,
                         db, M, N, act, M, accumulate);
      db_left = false;
    } else {
      // rows per chunk: four workgroups for every CU, at least one row for each wavefront
      const int strips = (N + 511) / 512;
      int per = (int)(((size_t)M * strips + 4 * (size_t)di->cu_count - 1) / (4 * (size_t)di->cu_count));
      if (per < 4) per = 4;
      if ((M + per - 1) / per > kMaxChunks) per = (M + kMaxChunks - 1) / kMaxChunks;
      chunks = (M + per - 1) / per;
      hipLaunchKernelGGL((linear_dz_kernel<F16, 64, 4, 2>), dim3((unsigned)strips, (unsigned)chunks), dim3(kBlock), 0, s, dY, lddy, pre, ldp, to, g.ld,
                         db ? plan->sums : nullptr, M, N, act, per, 0);
    }
    CCN_HIP(hipGetLastError());
  }
  const DbArgs dba{plan->sums, db_left ? db : nullptr, N, chunks, accumulate};
  // operands that the ring cannot fetch: W along its rows for dX, X and dz across them for dW
  const bool cw = dX && M > 0 && !few && !brief_dx && !ring_fetches(w, true), cx = dW && M > 0 && !brief_dw && !ring_fetches(x, false);
  const LinEpi dx_ep{nullptr, nullptr, nullptr, dX, 0, 0, lddx, CCN_ACT_NONE, 0};
  const LinEpi dw_ep{nullptr, nullptr, nullptr, dW, 0, 0, lddw, CCN_ACT_NONE, accumulate ? 1 : 0};
  if (cw || cx) {
    CCN_TRY(pack(cx ? &x : nullptr, K, plan->px, cw ? &w : nullptr, N, plan->pw, K, s));
    if (cx) x = Operand{plan->px, pitch((size_t)K), M, (int)round8((size_t)K)};
    if (cw) w = Operand{plan->pw, pitch((size_t)N), K, (int)round8((size_t)N)};
  }
  RingPlan hx{}, hw{};
  LinProd px{}, pw{};
  const bool ring_dx = dX && M > 0 && !few;
  if (ring_dx) {
    px = make_product(plan, g, true, w, true, M, K, N, di->cu_count);
    hx = choose_ring(M, K, N, plan->partial_floats, di->cu_count);
  }
  if (dW) {
    pw = make_product(plan, x, false, g, false, K, N, M, di->cu_count);
    hw = choose_ring(K, N, M, plan->partial_floats, di->cu_count);
  }
  if (ring_dx && dW) {
    // side by side, if that is estimated to be faster than one after the other (3 us for what is between two launches)
    PairPlan both = choose_pair(px, pw, plan->partial_floats, di->cu_count);
    const double tx = (double)px.tiles_r * px.tiles_c, tw = (double)pw.tiles_r * pw.tiles_c;
    if (both.us < hx.us + hw.us + (db_left ? 6.0 : 3.0) && tx + tw < 1e6) {
      LinProd& p = both.split == 2 ? pw : px;
      const int steps = (p.sum + 63) / 64;
      p.per_split = 64 * ((steps + both.splits - 1) / both.splits);
      both.splits = (p.sum + p.per_split - 1) / p.per_split;   // no empty split
      const double lx = (N + 63) / 64 / (both.split == 1 ? (double)both.splits : 1.0), lw = (M + 63) / 64 / (both.split == 2 ? (double)both.splits : 1.0);
      const int nx = (int)tx * (both.split == 1 ? both.splits : 1), nw = (int)tw * (both.split == 2 ? both.splits : 1);
      const PairArgs a{px, pw, dx_ep, dw_ep, dba, nx, nw, lw > lx ? 1 : 0};
      return dw32 ? product_pair<F16, true>(a, both.split, both.splits, s) : product_pair<F16, false>(a, both.split, both.splits, s);
    }
  }
  if (db_left) {
    hipLaunchKernelGGL(linear_db_kernel, dim3((unsigned)((N + kWave - 1) / kWave)), dim3(kDbWaves * kWave), 0, s, dba);
    CCN_HIP(hipGetLastError());
  }
  if (ring_dx) CCN_TRY((run_product<F16, true, true>(px, dx_ep, false, hx, s)));
  else if (dX && M > 0) CCN_TRY((product_few<F16, true>(plan, g.p, g.ld, W, ldw, M, K, N, dx_ep, di->cu_count, s)));
  if (dW) CCN_TRY((run_product<F16, false, false>(pw, dw_ep, dw32, hw, s)));
  return CCN_OK;
}

}  // namespace

extern "C" {

int ccn_linear_plan_destroy(ccn_linear_plan* plan) {
  if (!plan) return CCN_OK;
  int rc = CCN_OK;
  if (plan->dz && hipFree(plan->dz) != hipSuccess) rc = CCN_EHIP;
  if (plan->px && hipFree(plan->px) != hipSuccess) rc = CCN_EHIP;
  if (plan->pw && hipFree(plan->pw) != hipSuccess) rc = CCN_EHIP;
  if (plan->sums && hipFree(plan->sums) != hipSuccess) rc = CCN_EHIP;
  if (plan->partial && hipFree(plan->partial) != hipSuccess) rc = CCN_EHIP;
  if (plan->counters && hipFree(plan->counters) != hipSuccess) rc = CCN_EHIP;
  delete plan;
  return rc;
}

int ccn_linear_plan_create(int max_M, int max_N, int max_K, ccn_linear_plan** out) {
  if (!out) return CCN_EINVAL;
  *out = nullptr;
  if (max_M < 1 || max_N < 1 || max_K < 1) return CCN_EINVAL;
  if ((size_t)max_N > kRMaxLd || (size_t)max_K > kRMaxLd || max_M > (1 << 30)) return CCN_ERANGE;
  const DeviceInfo* di = nullptr;
  CCN_TRY(current_device_info(&di));
  ccn_linear_plan* const p = new (std::nothrow) ccn_linear_plan();
  if (!p) return CCN_ENOMEM;
  p->device = di->device;
  p->max_m = max_M;
  p->max_n = max_N;
  p->max_k = max_K;
  // A split product has at most two 128 x 128 tiles on every CU, over all its splits, and two steps of 64 in each split (a sum of up
  // to three steps is not split).
  auto floats = [&](int rows, int cols, int sum) -> size_t {
    if (sum <= 3 * 64) return 0;
    const size_t tiles = (size_t)((rows + 127) / 128) * (size_t)((cols + 127) / 128);
    const size_t most = tiles * (size_t)(sum / 128 + 1), cap = 2 * (size_t)di->cu_count;
    return (most < cap ? most : cap) * (size_t)(128 * 128);
  };
  // (with few rows the ring works on dW alone, and W is read as it lies: a plan for them has neither copy nor partial sums of more)
  const bool few_only = max_M <= kFewRows;
  const size_t need[3] = {few_only ? 0 : floats(max_M, max_N, max_K), few_only ? 0 : floats(max_M, max_K, max_N), floats(max_K, max_N, max_M)};
  for (const size_t f : need) p->partial_floats = f > p->partial_floats ? f : p->partial_floats;
  const size_t few_cols = ((size_t)(max_N > max_K ? max_N : max_K) + 127) & ~(size_t)127;
  // A split sum of few rows has fewer than two workgroups for every CU, over all its splits, of up to 128 outputs each.
  const size_t few_most = (size_t)kFewMaxSplits * few_cols, few_cap = 2 * (size_t)di->cu_count * 128;
  const size_t few = (few_most < few_cap ? few_most : few_cap) * (size_t)(max_M < kFewRows ? (max_M + 15) & ~15 : kFewRows);
  p->partial_floats = few > p->partial_floats ? few : p->partial_floats;
  const size_t counters = few_cols / 64 * kFewWaves * kFewCounter;
  hipError_t e = hipMalloc((void**)&p->dz, (size_t)max_M * pitch((size_t)max_N) * sizeof(uint16_t));
  if (e == hipSuccess) e = hipMalloc((void**)&p->px, (size_t)max_M * pitch((size_t)max_K) * sizeof(uint16_t));
  if (e == hipSuccess && !few_only) e = hipMalloc((void**)&p->pw, pitch((size_t)max_K) * pitch((size_t)max_N) * sizeof(uint16_t));
  if (e == hipSuccess) e = hipMalloc((void**)&p->sums, (size_t)kMaxChunks * (size_t)max_N * sizeof(float));
  if (e == hipSuccess) e = hipMalloc((void**)&p->partial, p->partial_floats * sizeof(float));
  if (e == hipSuccess) e = hipMalloc((void**)&p->counters, counters * sizeof(uint32_t));
  if (e == hipSuccess) e = hipMemset(p->counters, 0, counters * sizeof(uint32_t));
  if (e == hipSuccess) e = hipDeviceSynchronize();   // the zeros are there for calls on any stream
  if (e != hipSuccess) {
    ccn_linear_plan_destroy(p);
    return hip_fail(e);
  }
  *out = p;
  return CCN_OK;
}

int ccn_linear_bf16(ccn_linear_plan* plan, const uint16_t* X, size_t ldx, const uint16_t* W, size_t ldw, const float* bias,
                    const uint16_t* resid, size_t ldr, uint16_t* Y, size_t ldy, uint16_t* pre, size_t ldp, int M, int N, int K,
                    int act, void* stream) {
  return linear_forward<false>(plan, X, ldx, W, ldw, bias, resid, ldr, Y, ldy, pre, ldp, M, N, K, act, stream);
}

int ccn_linear_f16(ccn_linear_plan* plan, const uint16_t* X, size_t ldx, const uint16_t* W, size_t ldw, const float* bias,
                   const uint16_t* resid, size_t ldr, uint16_t* Y, size_t ldy, uint16_t* pre, size_t ldp, int M, int N, int K,
                   int act, void* stream) {
  return linear_forward<true>(plan, X, ldx, W, ldw, bias, resid, ldr, Y, ldy, pre, ldp, M, N, K, act, stream);
}

int ccn_linear_backward_bf16(ccn_linear_plan* plan, const uint16_t* dY, size_t lddy, const uint16_t* pre, size_t ldp,
                             const uint16_t* X, size_t ldx, const uint16_t* W, size_t ldw, uint16_t* dX, size_t lddx, void* dW,
                             size_t lddw, int dw_type, float* db, int accumulate, int M, int N, int K, int act, void* stream) {
  return linear_backward<false>(plan, dY, lddy, pre, ldp, X, ldx, W, ldw, dX, lddx, dW, lddw, dw_type, db, accumulate, M, N, K, act, stream);
}

int ccn_linear_backward_f16(ccn_linear_plan* plan, const uint16_t* dY, size_t lddy, const uint16_t* pre, size_t ldp,
                            const uint16_t* X, size_t ldx, const uint16_t* W, size_t ldw, uint16_t* dX, size_t lddx, void* dW,
                            size_t lddw, int dw_type, float* db, int accumulate, int M, int N, int K, int act, void* stream) {
  return linear_backward<true>(plan, dY, lddy, pre, ldp, X, ldx, W, ldw, dX, lddx, dW, lddw, dw_type, db, accumulate, M, N, K, act, stream);
}

}  // extern "C"
