// New keys and values into a paged e4m3 cache with one scale per page and head.
//
//   cache [n_pages, Hkv, page, D] e4m3, scale [n_pages, Hkv] fp32; position p of
//   sequence b is slot p % page of page table[b][p / page].
//
// A page's scale s is the smallest power of two with amax / s <= 448 (amax at
// least 1e-4, as in act_quant, kernel_sm121.py:55-87) over what was written to
// it.  Tokens arrive a few at a time, so s may have to grow under codes that
// are there already: s' = max(s, needed), and the earlier codes are rounded
// again at s'.  Powers of two make that harmless: the ratio only moves the
// exponent, and a code changes its value only where it becomes subnormal.
// A page whose slot 0 is written by this call starts anew (whatever it held
// before does not count), and slots behind the new tokens are left alone.
// Infinities and NaN are stored as NaN and take no part in the scale.
//
// One CTA per (sequence, page it touches, head, key or value): it owns that
// page and head, so there are no atomics and the result does not depend on any
// order.  Two passes over its new rows: amax, then codes (the second reads
// hit the caches).  HBM-bound for prompts, latency for single tokens.
#include "common.cuh"

namespace kvc {

constexpr int kThreads = 128;

struct Args {
  const void* src[2];           // k, v: [B, S, Hkv, D], last dim contiguous
  int64_t sb[2], ss[2], sh[2];  // strides in elements
  uint8_t* cache[2];
  float* scale[2];
  const int* table;             // [B, max_pages]
  const int* start;             // [B] cached tokens before the new ones
  const int* new_lens;          // [B] or null
  int B, S, Hkv, D, page_log2, max_pages, n_pages, span;   // span: pages a sequence touches at most
};

// Smallest power of two s with amax / s <= 448 = 1.75 * 2^8, exactly: compare amax's significand with 1.75.
BS_DEVINL float pow2_scale(float amax) {
  const uint32_t b = __float_as_uint(fmaxf(amax, 1e-4f));
  const int e = (int)(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)e << 23);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) append_kernel(Args a) {
  constexpr int E = 16 / (int)sizeof(T);
  __shared__ float red[kThreads / 32];
  pdl_wait();
  int64_t u = blockIdx.x;
  const int h = (int)(u % a.Hkv);
  u /= a.Hkv;
  const int j = (int)(u % a.span);
  const int b = (int)(u / a.span);
  const int w = blockIdx.y;
  const int page = 1 << a.page_log2;
  int start = a.start[b];
  int nl = a.new_lens ? a.new_lens[b] : a.S;
  if (start < 0 || nl < 0 || nl > a.S) {      // not a length: nothing of this sequence is written
    if (threadIdx.x == 0) bs_set_error(BS_ERR_BAD_INDEX);
    return;
  }
  const int64_t pg = (int64_t)(start >> a.page_log2) + j;
  const int64_t first = pg << a.page_log2;
  const int64_t lo = max((int64_t)start, first), hi = min((int64_t)start + nl, first + page);
  if (lo >= hi) return;
  const int id = pg < a.max_pages ? a.table[(int64_t)b * a.max_pages + pg] : -1;
  if (id < 0 || id >= a.n_pages) {
    if (threadIdx.x == 0) bs_set_error(BS_ERR_BAD_INDEX);
    return;
  }
  const int m = (int)(hi - lo), before = (int)(lo - first);
  const int vrow = a.D / E;                   // 16-byte vectors per row
  const T* src = reinterpret_cast<const T*>(a.src[w]) + b * a.sb[w] + (lo - start) * a.ss[w] + h * a.sh[w];
  float amax = 0.0f;
  for (int i = threadIdx.x; i < m * vrow; i += kThreads) {
    const int r = i / vrow, d = (i - r * vrow) * E;
    float f[E];
    unpack<T>(*reinterpret_cast<const uint4*>(src + r * a.ss[w] + d), f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float v = fabsf(f[e]);
      if (v < __uint_as_float(0x7F800000u)) amax = fmaxf(amax, v);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  const int64_t sat = (int64_t)id * a.Hkv + h;
  const float old = a.scale[w][sat];
  __syncthreads();                            // also: every thread has read the old scale
#pragma unroll
  for (int k = 0; k < kThreads / 32; ++k) amax = fmaxf(amax, red[k]);
  float s = pow2_scale(amax);
  uint8_t* dst = a.cache[w] + sat * ((int64_t)a.D << a.page_log2);
  if (before > 0) {
    s = fmaxf(s, old);
    if (s > old) {
      const float f = __fdiv_rn(old, s);
      const int n16 = before * a.D / 16;
      for (int i = threadIdx.x; i < n16; i += kThreads) {
        uint4 c = reinterpret_cast<uint4*>(dst)[i];
        uint32_t* p = reinterpret_cast<uint32_t*>(&c);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t v = p[k];
          p[k] = bs_cvt_e4m3x2(bs_e4m3_to_f32(v & 0xFF) * f, bs_e4m3_to_f32((v >> 8) & 0xFF) * f) |
                 ((uint32_t)bs_cvt_e4m3x2(bs_e4m3_to_f32((v >> 16) & 0xFF) * f, bs_e4m3_to_f32(v >> 24) * f) << 16);
        }
        reinterpret_cast<uint4*>(dst)[i] = c;
      }
    }
  }
  if (threadIdx.x == 0) a.scale[w][sat] = s;
  dst += (int64_t)before * a.D;
  for (int i = threadIdx.x; i < m * vrow; i += kThreads) {
    const int r = i / vrow, d = (i - r * vrow) * E;
    float f[E];
    unpack<T>(*reinterpret_cast<const uint4*>(src + r * a.ss[w] + d), f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      f[e] = __fdiv_rn(f[e], s);
      if (fabsf(f[e]) == __uint_as_float(0x7F800000u)) f[e] = __uint_as_float(0x7FC00000u);
    }
    uint32_t q[E / 4];
#pragma unroll
    for (int e = 0; e < E / 4; ++e)
      q[e] = bs_cvt_e4m3x2(f[4 * e], f[4 * e + 1]) | ((uint32_t)bs_cvt_e4m3x2(f[4 * e + 2], f[4 * e + 3]) << 16);
    uint32_t* o = reinterpret_cast<uint32_t*>(dst + (int64_t)r * a.D + d);
    if constexpr (E == 8) *reinterpret_cast<uint2*>(o) = make_uint2(q[0], q[1]);
    else *o = q[0];
  }
  pdl_launch_dependents();
}

}  // namespace kvc

cudaError_t bs_launch_cache_append(const kvc::Args& a, int dtype, int both, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.span * a.Hkv), both ? 2 : 1);
  cfg.blockDim = dim3(kvc::kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (dtype == BS_DT_BF16) return cudaLaunchKernelEx(&cfg, kvc::append_kernel<__nv_bfloat16>, a);
  if (dtype == BS_DT_F16) return cudaLaunchKernelEx(&cfg, kvc::append_kernel<__half>, a);
  return cudaLaunchKernelEx(&cfg, kvc::append_kernel<float>, a);
}
