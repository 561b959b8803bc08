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
// HBM-bound (8192 tokens x 40 heads x 128 bf16: 30 us, 0.85 of the copy
// bandwidth): a CTA takes a few tokens (or, when there are few, a range of one
// token's heads), loads its 16-byte vectors first, computes the tokens' cos/sin
// pairs into shared memory while they are in flight, rotates and stores.
#include "common.cuh"

namespace rope {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;
constexpr int kCs = 1024;        // cos/sin pairs of a CTA's tokens

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
  int tokens_per_cta, heads_per_cta;
  float scale;
  int inverse, copy;            // copy: the unrotated dims go to out as well
  BsDiv per_head, per_token, pairs;
};

// One task: a rotated vector of 16 bytes (in the half layout a pair of them), or a vector to copy.  U tasks per thread
// and pass are in flight.
template <typename T, bool HALF, int U>
__global__ void __launch_bounds__(kThreads) rope_kernel(const Args a) {
  constexpr int E = 16 / (int)sizeof(T);               // elements per vector
  constexpr int PV = HALF ? E : E / 2;                 // pairs of a task
  // Two pairs (cos, sin, cos, sin) in 16 bytes, a task's PV / 2 of them nrot apart: lanes next to each other read next
  // to each other.
  __shared__ float4 cs[kCs / 2];
  pdl_wait();
  const int64_t tok0 = (int64_t)blockIdx.x * a.tokens_per_cta;
  const int nt = (int)min((int64_t)a.tokens_per_cta, a.tokens - tok0);
  const int h0 = blockIdx.y * a.heads_per_cta;
  const int nh = min(a.heads_per_cta, a.H - h0);
  const int nrot = HALF ? a.n / (2 * E) : a.n / E;
  const int per_token = nh * (int)a.per_head.d;
  const int tasks = nt * per_token;
  const T* x = reinterpret_cast<const T*>(a.x) + tok0 * a.x_tok + h0 * a.x_head;
  T* out = reinterpret_cast<T*>(a.out) + tok0 * a.o_tok + h0 * a.o_head;
  const int np = a.n / 2;
  bool first = true;
  for (int base = 0; base < tasks; base += kThreads * U) {
    uint4 lo[U], hi[HALF ? U : 1];
    int64_t to[U];
    int at[U];                       // first cos/sin pairs, or -1: copy
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int task = base + u * kThreads + threadIdx.x;
      if (task < tasks) {
        // per_token is the divisor of a full range of heads; a CTA with several tokens has all of them
        const int t = nt > 1 ? bs_div(task, a.per_token) : 0;
        const int in = task - t * per_token;
        const int h = bs_div(in, a.per_head);
        const int k = in - h * (int)a.per_head.d;
        int d;
        if (k < nrot) {
          d = a.offset + k * E;
          at[u] = t * (np / 2) + k;
        } else {
          const int e = (k - nrot) * E;
          d = e < a.offset ? e : e + a.n;
          at[u] = -1;
        }
        const T* p = x + t * a.x_tok + h * a.x_head + d;
        to[u] = t * a.o_tok + h * a.o_head + d;
        lo[u] = *reinterpret_cast<const uint4*>(p);
        if (HALF && at[u] >= 0) hi[u] = *reinterpret_cast<const uint4*>(p + np);
      }
    }
    if (first) {
      first = false;
      for (int j = threadIdx.x; j < nt * np; j += kThreads) {
        const int t = bs_div(j, a.pairs), i = j - t * np;
        const int64_t p = a.pos64 ? a.pos64[tok0 + t] : (int64_t)a.pos32[tok0 + t];
        const double turn = a.freq[i] * 0.15915494309189533577;              // 1 / (2 pi)
        const double frac = turn - floor(turn);
        // frac < 1; 2^64 itself (frac rounded up) saturates to 2^64 - 1
        const unsigned long long f = __double2ull_rn(frac * 18446744073709551616.0);
        const long long v = (long long)((unsigned long long)p * f);
        float s, c;
        sincospif((float)v * 1.0842021724855044e-19f, &s, &c);               // 2^-63: fraction of a turn x 2
        const int k = i / PV, in = i - k * PV;
        reinterpret_cast<float2*>(cs)[(t * (np / 2) + (in / 2) * nrot + k) * 2 + (in & 1)] =
            make_float2(c * a.scale, (a.inverse ? -s : s) * a.scale);
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int task = base + u * kThreads + threadIdx.x;
      if (task < tasks) {
        T* o = out + to[u];
        if (at[u] >= 0) {
          float f[E];
          unpack<T>(lo[u], f);
          if (HALF) {
            float g[E], p[E], q[E];
            unpack<T>(hi[u], g);
#pragma unroll
            for (int i = 0; i < E; i += 2) {
              const float4 t = cs[at[u] + (i / 2) * nrot];
              p[i] = f[i] * t.x - g[i] * t.y;
              q[i] = f[i] * t.y + g[i] * t.x;
              p[i + 1] = f[i + 1] * t.z - g[i + 1] * t.w;
              q[i + 1] = f[i + 1] * t.w + g[i + 1] * t.z;
            }
            *reinterpret_cast<uint4*>(o + np) = pack<T>(q);
            lo[u] = pack<T>(p);
          } else {
            float p[E];
#pragma unroll
            for (int i = 0; i < E; i += 4) {
              const float4 t = cs[at[u] + (i / 4) * nrot];
              p[i] = f[i] * t.x - f[i + 1] * t.y;
              p[i + 1] = f[i] * t.y + f[i + 1] * t.x;
              p[i + 2] = f[i + 2] * t.z - f[i + 3] * t.w;
              p[i + 3] = f[i + 2] * t.w + f[i + 3] * t.z;
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
  const int esz = dtype == BS_DT_F32 ? 4 : 2, E = 16 / esz;
  const int per_head = (half ? a.n / (2 * E) : a.n / E) + (a.copy ? (a.D - a.n) / E : 0);
  // Tasks of a CTA: two per thread in the half layout (two vectors each), one in the interleaved one, of as many whole
  // tokens as that is (their cos/sin pairs have to fit) or of part of a token's heads; fewer when the CTAs would not
  // fill the GPU a few times.  More per thread costs registers, and with them loads in flight: 8192 tokens x 40 heads x
  // 128 bf16 take 30 us half (1: 41, 3: 42) and 43 to 46 us interleaved (2: 52, 4: 63); 64 tokens x 64 heads x 512 with 64
  // dims turned 2.9 us (2: 3.4, 4: 4.7).
  const int want = half ? 2 * rope::kThreads : rope::kThreads;
  const int64_t per_token = (int64_t)per_head * a.H;
  int64_t tpc = want / per_token, hpc = a.H;
  tpc = tpc < rope::kCs / (a.n / 2) ? tpc : rope::kCs / (a.n / 2);
  const int64_t even = a.tokens / (4 * 148);
  tpc = tpc < even ? tpc : even;
  if (tpc <= 1) {
    tpc = 1;
    const int64_t most = a.tokens < 4 * 148 ? rope::kThreads : want;   // few tokens: more, smaller CTAs
    if (per_token > most) hpc = most / per_head > 1 ? most / per_head : 1;
  }
  a.tokens_per_cta = (int)tpc;
  a.heads_per_cta = (int)hpc;
  a.per_head = bs_make_div(per_head);
  a.per_token = bs_make_div((uint32_t)(tpc > 1 ? per_token : 1));
  a.pairs = bs_make_div(a.n / 2);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.tokens + tpc - 1) / tpc), (unsigned)((a.H + hpc - 1) / hpc));
  cfg.blockDim = dim3(rope::kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto go = [&](auto t) {
    using T = decltype(t);
    return half ? cudaLaunchKernelEx(&cfg, rope::rope_kernel<T, true, 2>, a)
                : cudaLaunchKernelEx(&cfg, rope::rope_kernel<T, false, 1>, a);
  };
  if (dtype == BS_DT_BF16) return go(__nv_bfloat16());
  if (dtype == BS_DT_F16) return go(__half());
  return go(float());
}
