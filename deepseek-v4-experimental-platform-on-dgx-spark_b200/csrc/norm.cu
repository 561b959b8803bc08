// RMS norm with the residual's addition, written in the input's type or as
// e4m3 codes with one scale per 1 x 128 block (what fp8_gemm / fp4_gemm take),
// which saves the norm's round trip through memory in front of a product:
//
//   h = x + residual           fp32, rounded to the input's type (the residual
//                              stream keeps that type, and the norm reads what
//                              the next layer will read)
//   y = h * w / sqrt(mean(h^2) + eps)                                     fp32
//   out = y                    rounded once, or
//   s = max(amax(block), 1e-4) / 448, as act_quant (kernel_sm121.py:55-87);
//   code = e4m3_rn(y / s)      2^ceil(log2 s) for s in the power-of-two form
//
// The codes come from the fp32 y: act_quant(rms_norm(x)) would round y to 16
// bits first.  Eight squares at a time are added in fp32 and their sums in fp64,
// in every form of the kernel, so that a row's result does not depend on how
// many rows the call has.  (Every square in fp64, or eight with what their sums
// round away, costs 12 % of 16384 x 7168 bf16 and 21 % of 1999 x 5120 f16; it
// would move y, by its last fp32 bit, in about one value of a hundred.)  The
// root is kept as a sum of two fp32; y, s and y / s are rounded to nearest, so
// values next to the border of two codes (with 16-bit inputs y / s often lies
// on one) fall as the formula in fp32 steps says, but for that last bit of y.
//
// HBM-bound: every value is read and written once.  A block of 128 values is
// half a warp x 8 values, so its amax is four shuffles.  Two forms:
//   rows      one row per CTA, loads straight into registers: few rows
//   ring      for many rows: the resident CTAs walk over the rows, rows arrive by
//             bulk copies in a ring of shared-memory buffers, so that loads go
//             on through the reduction and the stores of the row at hand; the
//             weight stays in registers.  16384 x 7168 bf16 with residual and
//             codes: 146 to 155 us (0.82 to 0.87 of the copy bandwidth; 142 in a
//             graph) against 192.
#include "common.cuh"

namespace rmsn {

constexpr int kMaxH = 16384;
constexpr int kMaxThreads = 512;
enum { kOut = 0, kCodes = 1 };

template <typename T> BS_DEVINL void load8(const T* p, float* f);
template <> BS_DEVINL void load8<float>(const float* p, float* f) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
template <> BS_DEVINL void load8<__nv_bfloat16>(const __nv_bfloat16* p, float* f) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  unpack<__nv_bfloat16>(v, f);
}
template <> BS_DEVINL void load8<__half>(const __half* p, float* f) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  unpack<__half>(v, f);
}
template <typename T> BS_DEVINL void store8(T* p, const float* f) { *reinterpret_cast<uint4*>(p) = pack<T>(f); }
template <> BS_DEVINL void store8<float>(float* p, const float* f) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

struct Args {
  const void* x;
  const void* res;   // or null
  const void* w;
  void* h;           // x + res (only with res)
  void* y;           // T [rows, H] or codes
  void* s;           // scales (kCodes)
  int64_t rows;
  int H;
  float eps;
  double inv_h;      // 1 / H
  int s_e8m0, pow2;
};

// max that propagates NaN, as torch.amax
BS_DEVINL float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Sum of eight squares: in fp32, and where that leaves its range (values above 2^60, tiny ones, infinities, NaN) in fp64.
BS_DEVINL double squares(const float* f) {
  const float a = fmaf(f[1], f[1], f[0] * f[0]), b = fmaf(f[3], f[3], f[2] * f[2]);
  const float c = fmaf(f[5], f[5], f[4] * f[4]), d = fmaf(f[7], f[7], f[6] * f[6]);
  const float s = (a + b) + (c + d);
  if (s > 0x1p-90f && s < 0x1p120f) return (double)s;
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) t = fma((double)f[i], (double)f[i], t);
  return t;
}
BS_DEVINL double row_sum(double sum, double* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
  sum = (lane & 15) < nw ? part[lane & 15] : 0.0;       // 16 warps at most; both halves of the warp add them up
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
// 1 / sqrt(v) as a sum of two fp32: a Newton step (with its second-order term) on the fp32 root, in fp64; the fp64
// root itself where v leaves fp32's range.
BS_DEVINL float2 inv_sqrt(double v) {
  const float r = rsqrtf((float)v);
  double x;
  if (r > 0.0f && r < __uint_as_float(0x7F800000u)) {
    const double d = (double)r;
    const double e = fma(-v * d, d, 1.0);
    x = fma(d, e * fma(e, 0.375, 0.5), d);
  } else {
    x = 1.0 / sqrt(v);
  }
  const float hi = (float)x;
  return make_float2(hi, fabsf(hi) < __uint_as_float(0x7F800000u) ? (float)(x - (double)hi) : 0.0f);
}

// y of one vector, in place; returns what put_codes takes as its largest.
template <typename T>
BS_DEVINL float scale_row(float* f, const float* g, float2 r) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float p = f[i] * g[i];                                   // exact for 16-bit values
    float e = p * r.y;
    if (sizeof(T) == 4) e = fmaf(fmaf(f[i], g[i], -p), r.x, e);
    f[i] = fmaf(p, r.x, e);
    m = max_nan(m, fabsf(sizeof(T) == 4 ? f[i] : p));
  }
  return m;
}

// Codes and scales of a thread's V vectors of y (vector v is number v blockDim + threadIdx of the row; H is a multiple
// of 128, so the 16 lanes of a block are all in the row or all out).  The V maxima over 16 lanes go through one
// butterfly, which leaves each group of lanes with one vector's: 5 shuffles for four vectors instead of 16, and one
// scale to compute per lane instead of four.
//
// `pmax`: the V vectors' largest |h w|, exact for 16-bit types, whose product with the row's factor r gives the block's
// amax unrounded; for fp32 the rounded y's largest magnitude, r = 1.
template <int V>
BS_DEVINL void put_codes(const Args& a, int64_t row, int nvec, const float (*f)[8], const float* pmax, float2 r) {
  const int lane = threadIdx.x & 31;
  const float* m = pmax;
  int own = 0;                       // the vector whose maximum this lane ends up with
  float amax;
  if constexpr (V == 4) {
    const bool b = lane & 8, c = lane & 4;
    const float p = max_nan(b ? m[1] : m[0], __shfl_xor_sync(0xffffffffu, b ? m[0] : m[1], 8));
    const float q = max_nan(b ? m[3] : m[2], __shfl_xor_sync(0xffffffffu, b ? m[2] : m[3], 8));
    amax = max_nan(c ? q : p, __shfl_xor_sync(0xffffffffu, c ? p : q, 4));
    own = (b ? 1 : 0) + (c ? 2 : 0);
  } else if constexpr (V == 2) {
    const bool b = lane & 8;
    amax = max_nan(b ? m[1] : m[0], __shfl_xor_sync(0xffffffffu, b ? m[0] : m[1], 8));
    amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 4));
    own = b ? 1 : 0;
  } else {
    amax = max_nan(m[0], __shfl_xor_sync(0xffffffffu, m[0], 8));
    amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 4));
  }
  amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  // amax / 448: the exact products' tail corrects the rounded quotient (an infinite or NaN amax is its own quotient)
  const float top = max_nan(amax * r.x, 1e-4f);
  float s = top;
  if (top < __uint_as_float(0x7F800000u)) {
    const float tail = top == 1e-4f ? 0.0f : fmaf(amax, r.y, fmaf(amax, r.x, -top));
    const float q = div_markstein(top, 448.0f, 1.0f / 448.0f);
    s = fmaf(fmaf(-448.0f, q, top) + tail, 1.0f / 448.0f, q);
  }
  if (a.pow2) s = bs_round_pow2(s);
  const float z = a.pow2 && s < __uint_as_float(0x7F800000u) ? bs_inv_pow2(s) : __frcp_rn(s);
  const int c_own = own * blockDim.x + threadIdx.x;
  if ((lane & (V == 4 ? 3 : V == 2 ? 7 : 15)) == 0 && c_own < nvec) {
    const int64_t at = row * (a.H >> 7) + (c_own >> 4);
    if (a.s_e8m0) reinterpret_cast<uint8_t*>(a.s)[at] = bs_f32_to_e8m0(s);
    else reinterpret_cast<float*>(a.s)[at] = s;
  }
  uint8_t* y = reinterpret_cast<uint8_t*>(a.y) + row * a.H + threadIdx.x * 8;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int from = (lane & 16) + (v & 1) * 8 + (v >> 1) * 4;
    const float k = V == 1 ? z : __shfl_sync(0xffffffffu, z, from);
    float g[8];
    if (a.pow2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = f[v][i] * k;
    } else {
      // one correction of y * RN(1/s): the remainder is exact, so the sum rounds to the nearest of y / s
      const float d = V == 1 ? s : __shfl_sync(0xffffffffu, s, from);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        g[i] = f[v][i] * k;
        g[i] = fmaf(fmaf(-d, g[i], f[v][i]), k, g[i]);
      }
    }
    uint2 q;
    q.x = bs_cvt_e4m3x2(g[0], g[1]) | ((uint32_t)bs_cvt_e4m3x2(g[2], g[3]) << 16);
    q.y = bs_cvt_e4m3x2(g[4], g[5]) | ((uint32_t)bs_cvt_e4m3x2(g[6], g[7]) << 16);
    if ((int)(v * blockDim.x + threadIdx.x) < nvec) *reinterpret_cast<uint2*>(y + v * blockDim.x * 8) = q;
  }
}

// One row per CTA; thread t holds the 8-value vectors t, t + blockDim, ... of it.
template <typename T, int MODE, bool RES, int V>
__global__ void __launch_bounds__(kMaxThreads) rms_rows_kernel(const Args a) {
  __shared__ double part[32];
  const int nvec = a.H >> 3;
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.H;
  const T* res = reinterpret_cast<const T*>(a.res) + row * a.H;
  float f[V][8];
  pdl_wait();
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = v * blockDim.x + threadIdx.x;
    if (c < nvec) {
      load8<T>(x + c * 8, f[v]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[v][i] = 0.0f;
    }
  }
  if (RES) {
    float r[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = v * blockDim.x + threadIdx.x;
      if (c < nvec) load8<T>(res + c * 8, r[v]);
    }
    T* h = reinterpret_cast<T*>(a.h) + row * a.H;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = v * blockDim.x + threadIdx.x;
      if (c < nvec) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[v][i] = bs_to_f32<T>(bs_from_f32<T>(f[v][i] + r[v][i]));
        store8<T>(h + c * 8, f[v]);
      }
    }
  }
  pdl_launch_dependents();
  double sum = 0.0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sum += squares(f[v]);
  }
  const float2 r = inv_sqrt(fma(row_sum(sum, part), a.inv_h, (double)a.eps));
  const T* w = reinterpret_cast<const T*>(a.w);
  float m[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = v * blockDim.x + threadIdx.x;
    m[v] = 0.0f;
    if (c < nvec) {
      float g[8];
      load8<T>(w + c * 8, g);
      m[v] = scale_row<T>(f[v], g, r);
      if (MODE == kOut) store8<T>(reinterpret_cast<T*>(a.y) + row * a.H + c * 8, f[v]);
    }
  }
  if (MODE == kCodes) put_codes<V>(a, row, nvec, f, m, sizeof(T) == 4 ? make_float2(1.0f, 0.0f) : r);
}

constexpr int kMaxStages = 8;
// Rows per CTA from which the ring is used, and rows up to which a thread takes one or two vectors of a row instead of
// four: few rows are latency (1 row of 4096: 2.1 us with one vector, 2.5 with two), many rows with codes are instructions
// (60000 x 1024 f16: 56 us with four vectors, 61 with two); without codes two are as fast and take fewer registers.
constexpr int kRingRows = 4;
constexpr int kFewRows = 296, kSomeRows = 1200;
struct RingTail {
  double part[2][32];
  uint64_t full[kMaxStages];
  int abort;
};

template <typename T, int MODE, bool RES, int V>
__global__ void __maxnreg__(RES ? 128 : 96) rms_ring_kernel(const Args a, int stages) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int nvec = a.H >> 3;
  const uint32_t row_bytes = (uint32_t)a.H * sizeof(T);
  const uint32_t stage_bytes = RES ? 2 * row_bytes : row_bytes;
  RingTail& t = *reinterpret_cast<RingTail*>(smem + (size_t)stages * stage_bytes);
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&t.full[s], 1);
    t.abort = 0;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  const int64_t first = blockIdx.x, step = gridDim.x;
  auto issue = [&](int64_t row, int s) {
    mbar_arrive_expect_tx(&t.full[s], stage_bytes);
    bulk_load(smem + (size_t)s * stage_bytes, reinterpret_cast<const T*>(a.x) + row * a.H, row_bytes, &t.full[s]);
    if (RES)
      bulk_load(smem + (size_t)s * stage_bytes + row_bytes, reinterpret_cast<const T*>(a.res) + row * a.H, row_bytes,
                &t.full[s]);
  };
  if (threadIdx.x == 0)
    for (int s = 0; s < stages; ++s)
      if (first + s * step < a.rows) issue(first + s * step, s);
  uint4 w[V][sizeof(T) / 2];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = v * blockDim.x + threadIdx.x;
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k)
      w[v][k] = c < nvec ? reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.w) + c * 8)[k] : make_uint4(0, 0, 0, 0);
  }
  int s = 0, n = 0;
  uint32_t phase = 0;
  for (int64_t row = first; row < a.rows; row += step, ++n) {
    if (!mbar_test_wait(&t.full[s], phase)) mbar_wait(&t.full[s], phase, &t.abort);
    const T* x = reinterpret_cast<const T*>(smem + (size_t)s * stage_bytes);
    const T* res = reinterpret_cast<const T*>(smem + (size_t)s * stage_bytes + row_bytes);
    T* h = reinterpret_cast<T*>(a.h) + row * a.H;
    float f[V][8];
    double sum = 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = v * blockDim.x + threadIdx.x;
      if (c < nvec) {
        load8<T>(x + c * 8, f[v]);
        if (RES) {
          float r[8];
          load8<T>(res + c * 8, r);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[v][i] = bs_to_f32<T>(bs_from_f32<T>(f[v][i] + r[i]));
          store8<T>(h + c * 8, f[v]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[v][i] = 0.0f;
      }
      sum += squares(f[v]);
    }
    // the barrier in row_sum: every thread has read this stage
    const float2 r = inv_sqrt(fma(row_sum(sum, t.part[n & 1]), a.inv_h, (double)a.eps));
    if (t.abort) break;                  // uniform: set before the barrier or seen by the next one's wait
    if (threadIdx.x == 0 && row + stages * step < a.rows) issue(row + stages * step, s);
    float m[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = v * blockDim.x + threadIdx.x;
      float g[8];
      load8<T>(reinterpret_cast<const T*>(w[v]), g);
      m[v] = scale_row<T>(f[v], g, r);
      if (MODE == kOut && c < nvec) store8<T>(reinterpret_cast<T*>(a.y) + row * a.H + c * 8, f[v]);
    }
    if (MODE == kCodes) put_codes<V>(a, row, nvec, f, m, sizeof(T) == 4 ? make_float2(1.0f, 0.0f) : r);
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
  // after a wait that ran out: what is still in flight writes this CTA's shared memory
  if (t.abort && threadIdx.x == 0)
    for (int k = 0; k < stages; ++k)
      for (uint32_t j = 0; j < (1u << 16); ++j)
        if (mbar_try_wait(&t.full[k], k < s ? phase ^ 1 : phase)) break;
  pdl_launch_dependents();
}

int sm_count() {
  static int slots[hostcache::kMaxDevices];
  const int n = hostcache::device_attr(slots, cudaDevAttrMultiProcessorCount);
  return n > 0 ? n : 148;
}

template <typename T, int MODE, bool RES, int V>
cudaError_t launch_v(const Args& a, int threads, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // The ring where three rows fit each CTA's buffers and each CTA gets kRingRows rows at least (its start is a serial
  // load).
  if constexpr (V > 1) {             // one vector a thread is for few rows
    auto kern = rms_ring_kernel<T, MODE, RES, V>;
    static int regs_of[hostcache::kMaxDevices];
    const int regs = hostcache::get(regs_of, [&] {
      cudaFuncAttributes at;
      return cudaFuncGetAttributes(&at, kern) == cudaSuccess ? (at.numRegs + 7) / 8 * 8 : 128;
    });
    const int fit = 65536 / regs / threads;
    const int stage = a.H * (int)sizeof(T) * (RES ? 2 : 1), room = 224 * 1024;
    int ctas = fit < 16 ? fit : 16;
    while (ctas > 1 && ctas * (3 * stage + (int)sizeof(RingTail) + 1024) > room) --ctas;
    const int mine = room / ctas - (int)sizeof(RingTail) - 1024;
    if (a.rows >= (int64_t)kRingRows * ctas * sm_count() && ctas >= 2 && 3 * stage <= mine) {
      const int stages = mine / stage < kMaxStages ? mine / stage : kMaxStages;
      static int done[hostcache::kMaxDevices];
      const cudaError_t e = (cudaError_t)hostcache::get(
          done, [&] { return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, room); });
      if (e != cudaSuccess) return e;
      cfg.gridDim = dim3((unsigned)(ctas * sm_count()));
      cfg.dynamicSmemBytes = (size_t)stages * stage + sizeof(RingTail);
      return cudaLaunchKernelEx(&cfg, kern, a, stages);
    }
  }
  cfg.gridDim = dim3((unsigned)a.rows);
  return cudaLaunchKernelEx(&cfg, rms_rows_kernel<T, MODE, RES, V>, a);
}

template <typename T, int MODE, bool RES>
cudaError_t launch(const Args& a, cudaStream_t st) {
  const int nvec = a.H >> 3;
  // threads for V vectors each, a whole number of warps (and so of 128-blocks)
  auto threads = [&](int V) { return ((nvec + V - 1) / V + 31) / 32 * 32; };
  if (a.rows < kFewRows && threads(1) <= kMaxThreads) return launch_v<T, MODE, RES, 1>(a, threads(1), st);
  if ((MODE == kOut || a.rows < kSomeRows) && threads(2) <= kMaxThreads) return launch_v<T, MODE, RES, 2>(a, threads(2), st);
  return launch_v<T, MODE, RES, 4>(a, threads(4), st);
}

}  // namespace rmsn

cudaError_t bs_launch_rms_norm(const rmsn::Args& a, int dtype, int codes, cudaStream_t st) {
  if (a.rows == 0) return cudaSuccess;
  auto go = [&](auto t) {
    using T = decltype(t);
    if (codes) return a.res ? rmsn::launch<T, rmsn::kCodes, true>(a, st) : rmsn::launch<T, rmsn::kCodes, false>(a, st);
    return a.res ? rmsn::launch<T, rmsn::kOut, true>(a, st) : rmsn::launch<T, rmsn::kOut, false>(a, st);
  };
  if (dtype == BS_DT_BF16) return go(__nv_bfloat16());
  if (dtype == BS_DT_F16) return go(__half());
  return go(float());
}
