// Rotary positions on dims [offset, offset + n) of every head:
//
//   (u, v) -> (u c - v s, u s + v c),  c = scale cos(a), s = scale sin(a),  a = position * freq[i]
//
// for the n/2 pairs i of a head, (x[2i], x[2i+1]) in the interleaved layout and
// (x[i], x[i + n/2]) in the half layout; `inverse` turns the other way (which is
// also the gradient).  The other dims are copied (or stay, in place).
//
// Angles.  position * freq in fp32 is off by position * freq * 2^-24 radians,
// 0.06 at position 2^20; here freq comes in fp64 and is turned into a 64-bit
// fixed-point fraction of a turn, f = freq / (2 pi) * 2^64.  position * f in
// 64-bit integers keeps exactly the fraction (whole turns fall off the top),
// and only that fraction, in [-1/2, 1/2) turns, is rounded to fp32 for
// sincospif.  What is left of the error is freq's own 2^-53.
//
// HBM-bound: a CTA takes one token and a range of its heads, loads its 16-byte
// vectors first, computes the token's n/2 cos/sin pairs into shared memory
// while they are in flight, and rotates and stores.
#include "common.cuh"

namespace rope {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;
constexpr int kU = 4;           // 16-byte vectors (pairs of vectors in the half layout) in flight per thread

struct Args {
  const void* x;
  void* out;
  int64_t x_tok, x_head;        // strides in elements
  int64_t o_tok, o_head;
  const int64_t* pos64;         // one of the two
  const int* pos32;
  const double* freq;           // [n/2] radians per position
  int64_t tokens;
  int H, D, n, offset;
  int heads_per_cta;
  float scale;
  int inverse, copy;            // copy: the unrotated dims go to out as well
};

// One task of a head: a rotated vector (or pair of vectors), or a vector to copy.
template <typename T, bool HALF>
__global__ void __launch_bounds__(kThreads) rope_kernel(Args a) {
  constexpr int E = 16 / (int)sizeof(T);               // elements per vector
  __shared__ float2 cs[kMaxPairs];
  pdl_wait();
  const int64_t tok = blockIdx.x;
  const int h0 = blockIdx.y * a.heads_per_cta;
  const int nh = min(a.heads_per_cta, a.H - h0);
  const int nrot = HALF ? a.n / (2 * E) : a.n / E;
  const int per_head = nrot + (a.copy ? (a.D - a.n) / E : 0);
  const int tasks = nh * per_head;
  const T* x = reinterpret_cast<const T*>(a.x) + tok * a.x_tok + h0 * a.x_head;
  T* out = reinterpret_cast<T*>(a.out) + tok * a.o_tok + h0 * a.o_head;

  auto where = [&](int task, int& h, int& j, int& d) {   // head, index of the rotated vector (-1: copy), first dim
    h = task / per_head;
    const int k = task - h * per_head;
    if (k < nrot) {
      j = k;
      d = a.offset + k * E;
    } else {
      j = -1;
      const int e = (k - nrot) * E;
      d = e < a.offset ? e : e + a.n;
    }
  };
  bool first = true;
  for (int base = 0; base < tasks; base += kThreads * kU) {
    uint4 lo[kU], hi[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int task = base + u * kThreads + threadIdx.x;
      if (task < tasks) {
        int h, j, d;
        where(task, h, j, d);
        lo[u] = *reinterpret_cast<const uint4*>(x + h * a.x_head + d);
        if (HALF && j >= 0) hi[u] = *reinterpret_cast<const uint4*>(x + h * a.x_head + d + a.n / 2);
      }
    }
    if (first) {
      first = false;
      if (threadIdx.x < a.n / 2) {
        const int64_t p = a.pos64 ? a.pos64[tok] : (int64_t)a.pos32[tok];
        const double turn = a.freq[threadIdx.x] * 0.15915494309189533577;    // 1 / (2 pi)
        const double frac = turn - floor(turn);
        // frac < 1; 2^64 itself (frac rounded up) saturates to 2^64 - 1
        const unsigned long long f = __double2ull_rn(frac * 18446744073709551616.0);
        const long long t = (long long)((unsigned long long)p * f);
        float s, c;
        sincospif((float)t * 1.0842021724855044e-19f, &s, &c);               // 2^-63: fraction of a turn x 2
        cs[threadIdx.x] = make_float2(c * a.scale, (a.inverse ? -s : s) * a.scale);
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int task = base + u * kThreads + threadIdx.x;
      if (task < tasks) {
        int h, j, d;
        where(task, h, j, d);
        T* o = out + h * a.o_head + d;
        if (j >= 0) {
          float f[E];
          unpack<T>(lo[u], f);
          if (HALF) {
            float g[E], p[E], q[E];
            unpack<T>(hi[u], g);
#pragma unroll
            for (int i = 0; i < E; ++i) {
              const float2 t = cs[j * E + i];
              p[i] = f[i] * t.x - g[i] * t.y;
              q[i] = f[i] * t.y + g[i] * t.x;
            }
            *reinterpret_cast<uint4*>(o + a.n / 2) = pack<T>(q);
            lo[u] = pack<T>(p);
          } else {
            float p[E];
#pragma unroll
            for (int i = 0; i < E; i += 2) {
              const float2 t = cs[(j * E + i) >> 1];
              p[i] = f[i] * t.x - f[i + 1] * t.y;
              p[i + 1] = f[i] * t.y + f[i + 1] * t.x;
            }
            lo[u] = pack<T>(p);
          }
        }
        *reinterpret_cast<uint4*>(o) = lo[u];
      }
    }
  }
  pdl_launch_dependents();
}

}  // namespace rope

cudaError_t bs_launch_rope(rope::Args a, int dtype, int half, cudaStream_t st) {
  if (a.tokens == 0) return cudaSuccess;
  const int esz = dtype == BS_DT_F32 ? 4 : 2;
  // enough heads for about 16 KB of loads in each CTA
  const int64_t head_bytes = (int64_t)(a.copy ? a.D : a.n) * esz;
  int64_t hpc = 16384 / head_bytes;
  hpc = hpc < 1 ? 1 : (hpc > a.H ? a.H : hpc);
  a.heads_per_cta = (int)hpc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.tokens, (unsigned)((a.H + hpc - 1) / hpc));
  cfg.blockDim = dim3(rope::kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto go = [&](auto t) {
    using T = decltype(t);
    return half ? cudaLaunchKernelEx(&cfg, rope::rope_kernel<T, true>, a)
                : cudaLaunchKernelEx(&cfg, rope::rope_kernel<T, false>, a);
  };
  if (dtype == BS_DT_BF16) return go(__nv_bfloat16());
  if (dtype == BS_DT_F16) return go(__half());
  return go(float());
}
