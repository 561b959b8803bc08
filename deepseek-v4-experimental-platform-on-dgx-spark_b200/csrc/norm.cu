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
// bits first.  y / s is y * RN(1/s), within an ulp and a half of the quotient;
// only values that close to a border between two codes can differ by a step.
//
// HBM-bound: a row is read once into registers (16-byte loads, all issued
// before the first use), its sum of squares reduced across the CTA, and every
// value written once.  A block of 128 values is half a warp x 8 values, so its
// amax is four shuffles.
#include "common.cuh"

namespace rmsn {

constexpr int kMaxH = 16384;
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
  int s_e8m0, pow2;
};

// One row per CTA; thread t holds the 8-value vectors t, t + blockDim, ... of it.
template <typename T, int MODE, bool RES, int V>
__global__ void __launch_bounds__(1024) rms_kernel(Args a) {
  __shared__ float part[32];
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
  float sum = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(f[v][i], f[v][i], sum);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = (threadIdx.x & 31) < (blockDim.x >> 5) ? part[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float rstd = 1.0f / sqrtf(sum / (float)a.H + a.eps);
  const T* w = reinterpret_cast<const T*>(a.w);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = v * blockDim.x + threadIdx.x;
    const bool in = c < nvec;
    if (in) {
      float g[8];
      load8<T>(w + c * 8, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[v][i] *= rstd * g[i];
      if (MODE == kOut) store8<T>(reinterpret_cast<T*>(a.y) + row * a.H + c * 8, f[v]);
    }
    if (MODE == kCodes) {
      // H is a multiple of 128 here: the 16 lanes of a block are all in or all out
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = nan_max(amax, fabsf(f[v][i]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) amax = nan_max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      amax = amax < 1e-4f ? 1e-4f : amax;   // NaN passes through
      float s = __fdiv_rn(amax, 448.0f);
      if (a.pow2) s = bs_round_pow2(s);
      const float r = __frcp_rn(s);
      uint2 q;
      q.x = bs_cvt_e4m3x2(f[v][0] * r, f[v][1] * r) | ((uint32_t)bs_cvt_e4m3x2(f[v][2] * r, f[v][3] * r) << 16);
      q.y = bs_cvt_e4m3x2(f[v][4] * r, f[v][5] * r) | ((uint32_t)bs_cvt_e4m3x2(f[v][6] * r, f[v][7] * r) << 16);
      if (in) {
        *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(a.y) + row * a.H + c * 8) = q;
        if ((threadIdx.x & 15) == 0) {
          const int64_t at = row * (a.H >> 7) + (c >> 4);
          if (a.s_e8m0) reinterpret_cast<uint8_t*>(a.s)[at] = bs_f32_to_e8m0(s);
          else reinterpret_cast<float*>(a.s)[at] = s;
        }
      }
    }
  }
}

template <typename T, int MODE, bool RES, int V>
cudaError_t launch_v(const Args& a, int threads, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, rms_kernel<T, MODE, RES, V>, a);
}

template <typename T, int MODE, bool RES>
cudaError_t launch(const Args& a, cudaStream_t st) {
  const int nvec = a.H >> 3;
  // threads for V vectors each, a whole number of warps (and so of 128-blocks)
  auto threads = [&](int V) { return ((nvec + V - 1) / V + 31) / 32 * 32; };
  if (threads(1) <= 320) return launch_v<T, MODE, RES, 1>(a, threads(1), st);
  if (threads(2) <= 320) return launch_v<T, MODE, RES, 2>(a, threads(2), st);
  if (threads(4) <= 320) return launch_v<T, MODE, RES, 4>(a, threads(4), st);
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
