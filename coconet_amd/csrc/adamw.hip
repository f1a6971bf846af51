// AdamW over many tensors at once, moments in fp32 or in 8 bits (gfx950).
//
//   g = sum_p g[p] * inv_scale * *grad_scale          m <- b1*m + (1-b1)*g          v <- b2*v + ((1-b2)*g)*g
//   w <- w*(1 - lr*wd*decay_b) - lr * (m/(1-b1^t)) / (sqrt(v/(1-b2^t)) + eps)
//
// 8-bit moments: the moments of a tensor are cut into blocks of 256 elements.  A block holds m/sm and sqrt(v)/sr as OCP
// e4m3 values (round to nearest even), sm = max|m|/448 and sr = max sqrt(v)/448 in fp32.  sqrt(v) and not v: the update
// divides by sqrt(v), and e4m3's 2^18 between its smallest and largest value then span 2^36 of v.  A sqrt(v) that is
// not zero is held as at least the smallest e4m3 value: rounded to zero it would leave eps alone under the next step's
// first moment.  Everything between the load and the store of a moment is fp32.
//
// HBM-bound: a step cannot do without P*G + 8 bytes of gradients and weights per parameter plus 16 (fp32 moments) or
// 4 + 16/256 (8-bit ones), plus 2 for a 16-bit copy of the weights.  One wavefront works on one block, four neighbouring
// elements per lane, so that every access of a wavefront is one contiguous piece of 256 bytes to 1 KiB (eight elements per
// lane, whose fp32 pieces leave every other 16 bytes to the next instruction: 5.2 TB/s instead of 6.5 with fp32 moments),
// and the block's largest values are found by lane exchanges alone.  Two or four blocks per wavefront are slower (2^27
// elements, bf16 gradients and copy: 8-bit moments 346 / 354 / 365 us, fp32 ones 580 / 599 / 624).  With 8-bit moments the
// arithmetic is worth the memory's time: with IEEE divisions and square roots the same kernel took 428 us.
#include "ccn_common.hpp"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

namespace ccn {

constexpr int kAwBlock = 256;          // elements of one scale
constexpr int kAwLane = kAwBlock / kWave;   // 4 elements of a block per lane: every access of a wavefront is one contiguous piece
constexpr int kAwGroupShift = 5;       // blocks per entry of the coarse table: 32
constexpr uint32_t kAwGridX = 1u << 25;   // workgroups in a row of the grid: 2^31 of the 2^32 - 1 threads that a launch may have there
// A step of few blocks sets the overflow flag in its one launch: the wavefronts count themselves in, 32 of them on a counter and
// then the counters' last ones on one more, in steps of 1 or, with a gradient that is not finite, of 2^16 + 1; the very last one
// writes the flag and leaves the counters at zero.  A launch that clears the flag first costs more than this up to 2^22
// elements (us with it / without, fp32 moments: 500,000 8.8 / 6.1, 2 million 12.6 / 12.3, 4 million 21.7 / 21.7, 16 million
// 72.6 / 75.1; 8-bit ones: 8.9 / 6.3, 9.5 / 8.7, 14.0 / 13.9, 41.1 / 45.8)
constexpr uint32_t kAwFewBlocks = 8192, kAwCounter = 32;   // words from one counter to the next: a cache line each
constexpr float kE4m3Max = 448.0f, kE4m3Tiny = 0.001953125f;
constexpr float kAwFlush = 7.888609052210118e-31f;   // 2^-100: a block whose largest |m| is below it is held as zeros

struct AdamwBuf {
  uint64_t count;         // elements of the tensor
  uint32_t first_block;   // its first block
  float decay;            // factor on the weight decay
};
struct AdamwPrm {
  float b1, omb1, b2, omb2, eps, lr_wd, inv_scale;
  float rate, root_bc2;   // lr / (1-b1^t), 1 / sqrt(1-b2^t)
};
struct AdamwArgs {
  const uint32_t* coarse;        // tensor of the first block of every group of 32 blocks
  const uint32_t* first_block;   // [nbuff + kWave] first block of every tensor, then 0xffffffff
  const AdamwBuf* bufs;
  const void* const* table;      // [nbuff][CCN_MAX_RANKS + 2]: gradients, weights, 16-bit copy
  void* m;
  void* v;
  float* scales;                 // [2][blocks]
  const float* grad_scale;
  uint32_t* flag;
  uint32_t* arrivals;            // or nullptr: *flag was cleared before
  uint32_t blocks;
  int P, w16_type;
};
constexpr int kAwSlots = CCN_MAX_RANKS + 2;

enum { kGF32 = 0, kGBf16 = 1, kGF16 = 2 };
template <int G> struct GradType { typedef uint16_t T; };
template <> struct GradType<kGF32> { typedef float T; };
template <int G> __device__ __forceinline__ float widen(typename GradType<G>::T x) {
  if constexpr (G == kGF32) return x;
  else return G == kGF16 ? f16_bits_to_f32(x) : bf16_bits_to_f32(x);
}

// Four elements from `e` on: one wide load where they are all there and aligned, single ones elsewhere (zeros behind the
// end).
template <typename T> __device__ __forceinline__ Pack<T, kAwLane> load4(const T* p, uint64_t e, uint64_t n, bool wide) {
  if (wide) return load_stream<T, kAwLane>(p + e);
  Pack<T, kAwLane> r;
#pragma unroll
  for (int j = 0; j < kAwLane; j++) r.d[j] = e + j < n ? p[e + j] : T(0);
  return r;
}
template <typename T> __device__ __forceinline__ void store4(T* p, uint64_t e, uint64_t n, bool wide, const Pack<T, kAwLane>& x) {
  if (wide) {
    store_stream<T, kAwLane>(p + e, x);
    return;
  }
#pragma unroll
  for (int j = 0; j < kAwLane; j++)
    if (e + j < n) p[e + j] = x.d[j];
}

// The largest of a wavefront's values, none of which is negative: their bit patterns compare as integers.
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  const uint32_t y = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true);
  return x > y ? x : y;
}
__device__ __forceinline__ float wave_max(float f) {
  uint32_t x = __float_as_uint(f);
  x = dpp_max<0xB1>(x);    // quad_perm: neighbours
  x = dpp_max<0x4E>(x);    // quad_perm: pairs
  x = dpp_max<0x141>(x);   // row_half_mirror: quads
  x = dpp_max<0x140>(x);   // row_mirror: halves of 16 lanes
  const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)x, 0), b = (uint32_t)__builtin_amdgcn_readlane((int)x, 16);
  const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)x, 32), d = (uint32_t)__builtin_amdgcn_readlane((int)x, 48);
  const uint32_t ab = a > b ? a : b, cd = c > d ? c : d;
  return __uint_as_float(ab > cd ? ab : cd);
}
// The square root from the 1-ulp one by a Newton step on the residual: before its last rounding the result is within 2^-46 of the
// root, so that it is the correctly rounded one but for roots that close to the middle of two floats.  Below 2^-96 the argument is scaled: the instruction flushes denormals.
__device__ __forceinline__ float square_root(float x) {
  const bool small = x < 1.262177448353619e-29f;
  const float z = x * (small ? 18446744073709551616.0f : 1.0f);
  const float s = __builtin_amdgcn_sqrtf(z), h = 0.5f * __builtin_amdgcn_rcpf(s);
  const float r = fmaf(fmaf(-s, s, z), h, s) * (small ? 2.3283064365386963e-10f : 1.0f);
  return x > 0.0f ? r : 0.0f;
}

// 1/s, and x / s (inv: 1/s), by a Newton step each: correctly rounded but for quotients within 2^-46 of the middle of two floats.  A
// code then depends on the values and hardly ever on how a quotient next to a rounding border came about; the IEEE division
// sequence is three times as long.
__device__ __forceinline__ float inverse(float s) {
  const float r = __builtin_amdgcn_rcpf(s);
  return fmaf(fmaf(-s, r, 1.0f), r, r);
}
__device__ __forceinline__ float quotient(float x, float s, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-q, s, x), inv, q);
}
// Four values in units of the block's scale as e4m3.
__device__ __forceinline__ uint32_t to_e4m3(const float* x) {
  const int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], c, true);
}
__device__ __forceinline__ void from_e4m3(uint32_t c, float scale, float* x) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  x[0] = lo[0] * scale;
  x[1] = lo[1] * scale;
  x[2] = hi[0] * scale;
  x[3] = hi[1] * scale;
}

// One wavefront, one block.  CAP: gradient buffers loaded, all up front (those from P on are skipped under a uniform
// condition).
template <int G, int CAP, int BITS>
__global__ __launch_bounds__(kWave) void adamw_kernel(const AdamwArgs a, const AdamwPrm k) {
  typedef typename GradType<G>::T T;
  const uint32_t blk = blockIdx.x + blockIdx.y * gridDim.x;
  if (blk >= a.blocks) return;
  const int lane = threadIdx.x;
  // the tensor of this block: at most 32 tensors start inside a group of blocks, one per lane
  const uint32_t b0 = a.coarse[blk >> kAwGroupShift];
  const uint64_t before = __ballot(a.first_block[b0 + lane] <= blk);
  const uint32_t b = b0 + (uint32_t)__popcll(before) - 1u;
  const AdamwBuf buf = a.bufs[b];
  const void* const* const row = a.table + (size_t)b * kAwSlots;
  const uint64_t n = buf.count;
  float* const w = static_cast<float*>(const_cast<void*>(row[CCN_MAX_RANKS]));
  uint16_t* const w16 = static_cast<uint16_t*>(const_cast<void*>(row[CCN_MAX_RANKS + 1]));
  uintptr_t low = reinterpret_cast<uintptr_t>(w) | (a.w16_type ? reinterpret_cast<uintptr_t>(w16) : 0);
#pragma unroll
  for (int p = 0; p < CAP; p++)
    if (p < a.P) low |= reinterpret_cast<uintptr_t>(row[p]);
  const uint64_t e = (uint64_t)(blk - buf.first_block) * kAwBlock + lane * kAwLane;   // first element inside the tensor
  const uint64_t se = (uint64_t)blk * kAwBlock + lane * kAwLane;                      // and inside the moment arrays
  const bool wide = (low & 15u) == 0 && e + kAwLane <= n;

  Pack<T, kAwLane> gp[CAP];
  Pack<float, kAwLane> wp, mp, vp;
  uint32_t mc = 0, vc = 0;
  float sm = 0.0f, sr = 0.0f;
#pragma unroll
  for (int p = 0; p < CAP; p++)
    if (p < a.P) gp[p] = load4(static_cast<const T*>(row[p]), e, n, wide);
  wp = load4(w, e, n, wide);
  if constexpr (BITS == 32) {
    mp = load_stream<float, kAwLane>(static_cast<const float*>(a.m) + se);
    vp = load_stream<float, kAwLane>(static_cast<const float*>(a.v) + se);
  } else {
    mc = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.m) + se));
    vc = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + se));
    sm = a.scales[blk];
    sr = a.scales[a.blocks + blk];
  }
  const float gs = a.grad_scale ? k.inv_scale * *a.grad_scale : k.inv_scale;
  const float shrink = k.lr_wd * buf.decay;
  bool any_bad = false;
  if constexpr (BITS == 8) {
    from_e4m3(mc, sm, mp.d);
    from_e4m3(vc, sr, vp.d);
  }
  float root[kAwLane];
#pragma unroll
  for (int j = 0; j < kAwLane; j++) {
    float g = widen<G>(gp[0].d[j]);
#pragma unroll
    for (int p = 1; p < CAP; p++)
      if (p < a.P) g = g + widen<G>(gp[p].d[j]);
    g = g * gs;
    const float m0 = mp.d[j], v0 = BITS == 8 ? vp.d[j] * vp.d[j] : vp.d[j];
    const float m1 = k.b1 * m0 + k.omb1 * g;
    const float v1 = k.b2 * v0 + k.omb2 * g * g;
    // A gradient that is not finite, or whose square is not: the element keeps its weight and moments.  Asked of the gradient alone:
    // in v1 its square is weighted by 1-b2, and v0 is added.  A v1 that is not finite all the same (a restored v0 that is not) is
    // held too, without the flag.
    const bool bad = !(g * g < __builtin_inff()), hold = bad || !(v1 < __builtin_inff());
    any_bad = any_bad || (bad && (wide || e + j < n));   // behind the tensor's end the moments may hold anything
    const float r1 = square_root(v1);
    // The decay is a term of the update: 1 - shrink in fp32 is a multiple of 2^-24, a decay of 1e-7 would act as 1.2e-7 and one below
    // 3e-8 not at all, on every weight and step alike.
    const float w1 = wp.d[j] - fmaf(shrink, wp.d[j], (k.rate * m1) * __builtin_amdgcn_rcpf(r1 * k.root_bc2 + k.eps));
    wp.d[j] = hold ? wp.d[j] : w1;
    mp.d[j] = hold ? m0 : m1;
    if constexpr (BITS == 8) root[j] = hold ? vp.d[j] : r1;
    else vp.d[j] = hold ? v0 : v1;
  }
  store4(w, e, n, wide, wp);
  if (a.w16_type) {
    Pack<uint16_t, kAwLane> h;
#pragma unroll
    for (int j = 0; j < kAwLane; j++)
      h.d[j] = a.w16_type == CCN_TYPE_F16 ? f32_to_f16_bits(wp.d[j]) : __builtin_bit_cast(uint16_t, (__bf16)wp.d[j]);
    store4(w16, e, n, wide, h);
  }
  if constexpr (BITS == 32) {
    store_stream<float, kAwLane>(static_cast<float*>(a.m) + se, mp);
    store_stream<float, kAwLane>(static_cast<float*>(a.v) + se, vp);
  } else {
    if (!wide) {   // what lies behind a tensor's end must not weigh on its last block's scale
#pragma unroll
      for (int j = 0; j < kAwLane; j++)
        if (e + j >= n) mp.d[j] = root[j] = 0.0f;
    }
    const float mm = wave_max(fmaxf(fmaxf(fabsf(mp.d[0]), fabsf(mp.d[1])), fmaxf(fabsf(mp.d[2]), fabsf(mp.d[3]))));
    const float rm = wave_max(fmaxf(fmaxf(root[0], root[1]), fmaxf(root[2], root[3])));
    const float sm1 = mm < kAwFlush ? 0.0f : mm * (1.0f / kE4m3Max), sr1 = rm * (1.0f / kE4m3Max);
    const float im = sm1 > 0.0f ? inverse(sm1) : 0.0f, ir = sr1 > 0.0f ? inverse(sr1) : 0.0f;
    float y[kAwLane];
#pragma unroll
    for (int j = 0; j < kAwLane; j++) y[j] = __builtin_amdgcn_fmed3f(quotient(mp.d[j], sm1, im), -kE4m3Max, kE4m3Max);
    const uint32_t c = to_e4m3(y);
#pragma unroll
    for (int j = 0; j < kAwLane; j++)
      y[j] = root[j] > 0.0f ? __builtin_amdgcn_fmed3f(quotient(root[j], sr1, ir), kE4m3Tiny, kE4m3Max) : 0.0f;
    const uint32_t d = to_e4m3(y);
    __builtin_nontemporal_store(c, reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + se));
    __builtin_nontemporal_store(d, reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + se));
    if (lane == 0) {
      a.scales[blk] = sm1;
      a.scales[a.blocks + blk] = sr1;
    }
  }
  if (!a.flag) return;
  const bool wave_bad = __ballot(any_bad) != 0;
  if (lane != 0) return;
  if (!a.arrivals) {
    if (wave_bad) __hip_atomic_store(a.flag, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return;
  }
  const uint32_t group = blk >> kAwGroupShift, groups = (a.blocks + (1u << kAwGroupShift) - 1) >> kAwGroupShift;
  const uint32_t left = a.blocks - (group << kAwGroupShift), in_group = left < (1u << kAwGroupShift) ? left : 1u << kAwGroupShift;
  uint32_t* const mine = a.arrivals + (size_t)(1u + group) * kAwCounter;
  const uint32_t step = wave_bad ? 0x10001u : 1u, now = __hip_atomic_fetch_add(mine, step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + step;
  if ((now & 0xffffu) != in_group) return;
  __hip_atomic_store(mine, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint32_t step2 = now >> 16 ? 0x10001u : 1u, all = __hip_atomic_fetch_add(a.arrivals, step2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + step2;
  if ((all & 0xffffu) != groups) return;
  __hip_atomic_store(a.arrivals, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  *a.flag = all >> 16 ? 1u : 0u;
}

__global__ void adamw_clear_flag(uint32_t* flag) { *flag = 0u; }

}  // namespace ccn

using namespace ccn;

struct ccn_adamw_plan {
  int device = -1;
  int nbuff = 0, bits = 32;
  std::vector<int> live;               // the tensors that have elements
  uint32_t blocks = 0;
  uint32_t* coarse = nullptr;
  uint32_t* first_block = nullptr;
  AdamwBuf* bufs = nullptr;
  uint32_t* arrivals = nullptr;        // few blocks: counters, zero between calls
  const void** table_dev = nullptr;    // [live][kAwSlots]
  const void** table_pinned = nullptr;
  bool recorded = false;               // a step on this plan has been recorded
  hipEvent_t copied = nullptr;         // the last copy out of table_pinned
  std::vector<const void*> shadow;     // what the device table holds
};

namespace {

// Brings the device pointer table in line with the caller's pointers.  The copy is queued on the caller's stream; the
// host waits only for an earlier copy that is still reading the staging buffer.
int adamw_sync_table(ccn_adamw_plan* p, const void* const* g, int P, float* const* w, uint16_t* const* w16, hipStream_t s) {
  const size_t nl = p->live.size();
  bool same = true;
  for (size_t i = 0; i < nl; i++) {
    const size_t b = (size_t)p->live[i];
    const void** const row = p->shadow.data() + i * kAwSlots;
    for (int r = 0; r < P; r++) same = same && row[r] == g[(size_t)r * p->nbuff + b];
    same = same && row[CCN_MAX_RANKS] == w[b] && (!w16 || row[CCN_MAX_RANKS + 1] == w16[b]);
  }
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  CCN_HIP(hipStreamIsCapturing(s, &st));
  const bool recording = st != hipStreamCaptureStatusNone;
  if (same) {
    p->recorded = p->recorded || recording;
    return CCN_OK;
  }
  // a recorded copy would read the staging buffer at replay; and a recorded step reads the table at replay, so that the
  // pointers of a plan with one are not changed any more
  if (recording || p->recorded) return CCN_EINVAL;
  CCN_HIP(hipEventSynchronize(p->copied));
  // the device table is in an unknown state until the copy below is queued: forget what it held
  std::vector<const void*> next(p->shadow);
  std::fill(p->shadow.begin(), p->shadow.end(), nullptr);
  for (size_t i = 0; i < nl; i++) {
    const size_t b = (size_t)p->live[i];
    const void** const row = next.data() + i * kAwSlots;
    for (int r = 0; r < P; r++) row[r] = g[(size_t)r * p->nbuff + b];
    row[CCN_MAX_RANKS] = w[b];
    if (w16) row[CCN_MAX_RANKS + 1] = w16[b];
  }
  std::memcpy(p->table_pinned, next.data(), next.size() * sizeof(void*));
  CCN_HIP(hipMemcpyAsync(p->table_dev, p->table_pinned, next.size() * sizeof(void*), hipMemcpyHostToDevice, s));
  CCN_HIP(hipEventRecord(p->copied, s));
  p->shadow.swap(next);
  return CCN_OK;
}

template <int G, int CAP>
int adamw_launch(const ccn_adamw_plan* p, const AdamwArgs& a, const AdamwPrm& k, hipStream_t s) {
  const uint32_t gx = a.blocks < kAwGridX ? a.blocks : kAwGridX;
  const dim3 grid(gx, (a.blocks + gx - 1) / gx);
  // Wavefronts kept resident per CU, by a request for LDS that the kernel never touches (0: as many as fit, 32).  GB/s at
  // 2^26 elements with no cap / 24 / 20 / 16 / 13 wavefronts: fp32 moments and fp32 gradients 6095 / 6199 / 6391 / 6465 /
  // 6273 at 1 rank, 6145 / 6311 / 6468 / 6535 / 6001 at 8; fp32 moments and bf16 gradients 6214 / 6348 / 6416 / 6292 /
  // 5615 at 1 rank, 6331 / 6170 / 5393 / 5028 / 4110 at 8; 8-bit moments 6060 / 5616 / 4725 (bf16 gradients, 1 rank),
  // 6127 / 6344 / 6254 (fp32, 8 ranks): narrow accesses want every wavefront there is.
  const unsigned lds = p->bits == 8 ? 0u : G == kGF32 ? 10240u : a.P == 1 ? 8192u : 0u;
  if (p->bits == 8) hipLaunchKernelGGL((adamw_kernel<G, CAP, 8>), grid, dim3(kWave), lds, s, a, k);
  else hipLaunchKernelGGL((adamw_kernel<G, CAP, 32>), grid, dim3(kWave), lds, s, a, k);
  CCN_HIP(hipGetLastError());
  return CCN_OK;
}
template <int G>
int adamw_launch_p(const ccn_adamw_plan* p, const AdamwArgs& a, const AdamwPrm& k, hipStream_t s) {
  if (a.P == 1) return adamw_launch<G, 1>(p, a, k, s);
  if (a.P == 2) return adamw_launch<G, 2>(p, a, k, s);
  if (a.P <= 4) return adamw_launch<G, 4>(p, a, k, s);
  if (a.P <= 8) return adamw_launch<G, 8>(p, a, k, s);
  return adamw_launch<G, CCN_MAX_RANKS>(p, a, k, s);
}

int adamw_step(ccn_adamw_plan* p, const void* const* g, int P, int g_type, float* const* w, uint16_t* const* w16, int w16_type,
               void* m, void* v, float* scales, double lr, double beta1, double beta2, double eps, double wd, int step,
               double inv_scale, const float* grad_scale, uint32_t* flag, void* stream) {
  if (!p || !g || !w || P < 1 || P > CCN_MAX_RANKS || step < 1) return CCN_EINVAL;
  if (g_type != CCN_TYPE_F32 && g_type != CCN_TYPE_BF16 && g_type != CCN_TYPE_F16) return CCN_EINVAL;
  if (w16 && w16_type != CCN_TYPE_BF16 && w16_type != CCN_TYPE_F16) return CCN_EINVAL;
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0)) return CCN_EINVAL;
  if ((reinterpret_cast<uintptr_t>(grad_scale) | reinterpret_cast<uintptr_t>(flag)) & 3u) return CCN_EINVAL;
  const uintptr_t gmask = g_type == CCN_TYPE_F32 ? 3u : 1u;
  for (const int b : p->live) {
    for (int r = 0; r < P; r++) {
      const void* const x = g[(size_t)r * p->nbuff + b];
      if (!x || (reinterpret_cast<uintptr_t>(x) & gmask)) return CCN_EINVAL;
    }
    if (!w[b] || (reinterpret_cast<uintptr_t>(w[b]) & 3u)) return CCN_EINVAL;
    if (w16 && (!w16[b] || (reinterpret_cast<uintptr_t>(w16[b]) & 1u))) return CCN_EINVAL;
  }
  if (p->blocks) {
    if (!m || !v || !aligned16(m) || !aligned16(v)) return CCN_EINVAL;
    if (p->bits == 8 ? (!scales || (reinterpret_cast<uintptr_t>(scales) & 3u)) : scales != nullptr) return CCN_EINVAL;
  }
  const DeviceInfo* di = nullptr;
  int rc = current_device_info(&di);
  if (rc != CCN_OK) return rc;
  if (di->device != p->device) return CCN_EINVAL;
  hipStream_t s = as_stream(stream);
  if (p->blocks) {
    rc = adamw_sync_table(p, g, P, w, w16, s);
    if (rc != CCN_OK) return rc;
  }
  if (flag && !p->arrivals) {
    hipLaunchKernelGGL(adamw_clear_flag, dim3(1), dim3(1), 0, s, flag);
    CCN_HIP(hipGetLastError());
  }
  if (!p->blocks) return CCN_OK;
  AdamwPrm k;
  k.b1 = (float)beta1;
  k.omb1 = (float)(1.0 - beta1);
  k.b2 = (float)beta2;
  k.omb2 = (float)(1.0 - beta2);
  k.eps = (float)eps;
  k.lr_wd = (float)(lr * wd);
  k.rate = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
  k.root_bc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
  k.inv_scale = (float)inv_scale;
  AdamwArgs a;
  a.coarse = p->coarse;
  a.first_block = p->first_block;
  a.bufs = p->bufs;
  a.table = p->table_dev;
  a.m = m;
  a.v = v;
  a.scales = scales;
  a.grad_scale = grad_scale;
  a.flag = flag;
  a.arrivals = p->arrivals;
  a.blocks = p->blocks;
  a.P = P;
  a.w16_type = w16 ? w16_type : 0;
  switch (g_type) {
    case CCN_TYPE_F32: return adamw_launch_p<kGF32>(p, a, k, s);
    case CCN_TYPE_BF16: return adamw_launch_p<kGBf16>(p, a, k, s);
    default: return adamw_launch_p<kGF16>(p, a, k, s);
  }
}

int adamw_plan_create(const size_t* counts, const float* decay, int nbuff, int bits, ccn_adamw_plan** out);

}  // namespace

extern "C" {

int ccn_adamw_plan_destroy(ccn_adamw_plan* p) {
  if (!p) return CCN_OK;
  int rc = CCN_OK;
  if (p->copied && hipEventSynchronize(p->copied) != hipSuccess) rc = CCN_EHIP;
  if (p->copied && hipEventDestroy(p->copied) != hipSuccess) rc = CCN_EHIP;
  if (p->coarse && hipFree(p->coarse) != hipSuccess) rc = CCN_EHIP;
  if (p->first_block && hipFree(p->first_block) != hipSuccess) rc = CCN_EHIP;
  if (p->bufs && hipFree(p->bufs) != hipSuccess) rc = CCN_EHIP;
  if (p->arrivals && hipFree(p->arrivals) != hipSuccess) rc = CCN_EHIP;
  if (p->table_dev && hipFree(p->table_dev) != hipSuccess) rc = CCN_EHIP;
  if (p->table_pinned && hipHostFree(p->table_pinned) != hipSuccess) rc = CCN_EHIP;
  delete p;
  return rc;
}

int ccn_adamw_plan_create(const size_t* counts, const float* decay, int nbuff, int bits, ccn_adamw_plan** out) {
  if (!out) return CCN_EINVAL;
  *out = nullptr;
  if (!counts || nbuff < 1 || (bits != 8 && bits != 32)) return CCN_EINVAL;
  return guarded([&] { return adamw_plan_create(counts, decay, nbuff, bits, out); });
}

int ccn_adamw_plan_sizes(const ccn_adamw_plan* plan, size_t* elems, size_t* blocks) {
  if (!plan) return CCN_EINVAL;
  if (elems) *elems = (size_t)plan->blocks * kAwBlock;
  if (blocks) *blocks = (size_t)plan->blocks;
  return CCN_OK;
}

int ccn_adamw_scattered(ccn_adamw_plan* plan, const void* const* g, int P, int g_type, float* const* w, uint16_t* const* w16,
                        int w16_type, void* m, void* v, float* scales, double lr, double beta1, double beta2, double eps,
                        double wd, int step, double inv_scale, const float* grad_scale, uint32_t* overflow_flag, void* stream) {
  return guarded([&] {
    return adamw_step(plan, g, P, g_type, w, w16, w16_type, m, v, scales, lr, beta1, beta2, eps, wd, step, inv_scale, grad_scale,
                      overflow_flag, stream);
  });
}

}  // extern "C"

namespace {

int adamw_plan_create(const size_t* counts, const float* decay, int nbuff, int bits, ccn_adamw_plan** out) {
  std::vector<AdamwBuf> bufs;
  std::vector<uint32_t> first, coarse;
  std::vector<int> live;
  uint64_t blocks = 0;
  for (int b = 0; b < nbuff; b++) {
    if (counts[b] == 0) continue;
    if (counts[b] > ((size_t)1 << 48)) return CCN_ERANGE;
    const uint64_t nb = ((uint64_t)counts[b] + kAwBlock - 1) / kAwBlock;
    if (blocks + nb > 0x80000000ull) return CCN_ERANGE;   // block numbers are 32-bit, also those of a grid's last row
    const uint32_t i = (uint32_t)bufs.size();
    bufs.push_back(AdamwBuf{(uint64_t)counts[b], (uint32_t)blocks, decay ? decay[b] : 1.0f});
    first.push_back((uint32_t)blocks);
    live.push_back(b);
    for (uint64_t grp = (blocks + (1u << kAwGroupShift) - 1) >> kAwGroupShift; (grp << kAwGroupShift) < blocks + nb; grp++) coarse.push_back(i);
    blocks += nb;
  }
  const DeviceInfo* di = nullptr;
  const int rc = current_device_info(&di);
  if (rc != CCN_OK) return rc;
  ccn_adamw_plan* const p = new ccn_adamw_plan();
  p->device = di->device;
  p->nbuff = nbuff;
  p->bits = bits;
  p->blocks = (uint32_t)blocks;
  hipError_t e = hipSuccess;
  try {
    p->live.swap(live);
    first.insert(first.end(), kWave, 0xffffffffu);   // a wavefront looks at 64 tensors from its group's first one on
    const size_t words = p->live.size() * (size_t)kAwSlots;
    p->shadow.assign(words, nullptr);
    if (blocks) {
      e = hipMalloc((void**)&p->coarse, coarse.size() * sizeof(uint32_t));
      if (e == hipSuccess) e = hipMalloc((void**)&p->first_block, first.size() * sizeof(uint32_t));
      if (e == hipSuccess) e = hipMalloc((void**)&p->bufs, bufs.size() * sizeof(AdamwBuf));
      if (e == hipSuccess) e = hipMalloc((void**)&p->table_dev, words * sizeof(void*));
      if (e == hipSuccess) e = hipHostMalloc((void**)&p->table_pinned, words * sizeof(void*), hipHostMallocDefault);
      if (e == hipSuccess) e = hipEventCreateWithFlags(&p->copied, hipEventDisableTiming);
      if (e == hipSuccess) e = hipMemcpy(p->coarse, coarse.data(), coarse.size() * sizeof(uint32_t), hipMemcpyHostToDevice);
      if (e == hipSuccess) e = hipMemcpy(p->first_block, first.data(), first.size() * sizeof(uint32_t), hipMemcpyHostToDevice);
      if (e == hipSuccess) e = hipMemcpy(p->bufs, bufs.data(), bufs.size() * sizeof(AdamwBuf), hipMemcpyHostToDevice);
      if (blocks <= kAwFewBlocks) {
        const size_t bytes = (coarse.size() + 1) * kAwCounter * sizeof(uint32_t);   // a counter per entry of the coarse table, and one
        if (e == hipSuccess) e = hipMalloc((void**)&p->arrivals, bytes);
        if (e == hipSuccess) e = hipMemset(p->arrivals, 0, bytes);
        if (e == hipSuccess) e = hipDeviceSynchronize();   // the zeros are there for calls on any stream
      }
    }
  } catch (...) {
    ccn_adamw_plan_destroy(p);
    throw;
  }
  if (e != hipSuccess) {
    ccn_adamw_plan_destroy(p);
    return hip_fail(e);
  }
  *out = p;
  return CCN_OK;
}

}  // namespace
