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
// Infinities and NaN are stored as NaN and take no part in the scale.  A page
// whose scale is NaN or infinite keeps it, with codes of NaN (new values over an
// infinite scale are zero), until its slot 0 is written.
//
// One CTA per (sequence, page it touches, head), for its keys and values: it owns that
// page and head, so there are no atomics and the result does not depend on any
// order.  Its new rows are read once into registers, the loads going out
// before the page's index and old scale are known; rows that do not fit there
// (long pages of wide heads) are read twice, the second time out of L2.
// 4 x 4001 tokens x 8 heads x 128 bf16 take 22 us (0.68 of the copy bandwidth;
// keys and values in CTAs of their own 24, with 8 vectors a thread 27 to 31):
// a CTA is a chain of dependent loads, its start, its rows and page index, with
// 128 KB of rows in flight per SM.  One token for each of 128 sequences: 3.9 us.
#include "common.cuh"

namespace kvc {

constexpr int kU = 4;             // 16-byte vectors of new rows in registers, for keys and for values

struct Args {
  const void* src[2];           // k, v: [B, S, Hkv, D], last dim contiguous
  int64_t sb[2], ss[2], sh[2];  // strides in elements
  uint8_t* cache[2];
  float* scale[2];
  const int* table;             // [B, max_pages]
  const int* start;             // [B] cached tokens before the new ones
  const int* new_lens;          // [B] or null
  int B, S, Hkv, D, page_log2, max_pages, n_pages, span;   // span: pages a sequence touches at most
  BsDiv vrow;                   // 16-byte vectors of a row
};

// Smallest power of two s with amax / s <= 448 = 1.75 * 2^8, exactly: compare amax's significand with 1.75.
BS_DEVINL float pow2_scale(float amax) {
  const uint32_t b = __float_as_uint(fmaxf(amax, 1e-4f));
  const int e = (int)(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)e << 23);
}

// Codes of a vector: x / s for a power of two s (exact) or, where the page came with another scale, any s.  `odd`: there
// are infinities among the new rows, which become NaN (the conversion would saturate them).
template <typename T>
BS_DEVINL void put_codes(uint8_t* dst, const uint4& raw, float s, float inv, bool pow2, bool odd) {
  constexpr int E = 16 / (int)sizeof(T);
  float f[E];
  unpack<T>(raw, f);
  if (pow2) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] *= inv;
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = __fdiv_rn(f[e], s);
  }
  if (odd) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (fabsf(f[e]) == __uint_as_float(0x7F800000u)) f[e] = __uint_as_float(0x7FC00000u);
  }
  uint32_t q[E / 4];
#pragma unroll
  for (int e = 0; e < E / 4; ++e)
    q[e] = bs_cvt_e4m3x2(f[4 * e], f[4 * e + 1]) | ((uint32_t)bs_cvt_e4m3x2(f[4 * e + 2], f[4 * e + 3]) << 16);
  if constexpr (E == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(q[0], q[1]);
  else *reinterpret_cast<uint32_t*>(dst) = q[0];
}

// Largest magnitude of a vector as bits (of T, for two values of 16 bits at once in both halves): for numbers without
// their sign integer order is float order, and infinities and NaN come out on top.
template <typename T>
BS_DEVINL uint32_t top_of(const uint4& v, uint32_t top) {
  if constexpr (sizeof(T) == 2) {
    constexpr uint32_t k = 0x7FFF7FFFu;
    top = max_u16x2(top, max_u16x2(max_u16x2(v.x & k, v.y & k), max_u16x2(v.z & k, v.w & k)));
  } else {
    constexpr uint32_t k = 0x7FFFFFFFu;
    top = max(top, max(max(v.x & k, v.y & k), max(v.z & k, v.w & k)));
  }
  return top;
}
template <typename T>
BS_DEVINL float top_value(uint32_t top) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(top);
  const uint16_t b = (uint16_t)max(top & 0xFFFFu, top >> 16);
  return bs_to_f32<T>(*reinterpret_cast<const T*>(&b));
}
// Largest finite magnitude (vectors with infinities or NaN).
template <typename T>
BS_DEVINL float finite_top(const uint4& raw, float amax) {
  constexpr int E = 16 / (int)sizeof(T);
  float f[E];
  unpack<T>(raw, f);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float v = fabsf(f[e]);
    if (v < __uint_as_float(0x7F800000u)) amax = fmaxf(amax, v);
  }
  return amax;
}

// W = 2: keys and values, whose loads go out together.
template <typename T, int W>
__global__ void __maxnreg__(64) append_kernel(const Args a) {
  constexpr int E = 16 / (int)sizeof(T);
  __shared__ float red[W][16];
  pdl_wait();
  const int nthr = blockDim.x, warps = nthr >> 5;
  unsigned u = blockIdx.x;
  const int h = (int)(u % (unsigned)a.Hkv);
  u /= (unsigned)a.Hkv;
  const int j = (int)(u % (unsigned)a.span);
  const int b = (int)(u / (unsigned)a.span);
  const int page = 1 << a.page_log2;
  const int start = a.start[b];
  const int nl = a.new_lens ? a.new_lens[b] : a.S;
  if (start < 0 || nl < 0 || nl > a.S) {      // not a length: nothing of this sequence is written
    if (threadIdx.x == 0) bs_set_error(BS_ERR_BAD_INDEX);
    return;
  }
  const int64_t pg = (int64_t)(start >> a.page_log2) + j;
  const int64_t first = pg << a.page_log2;
  const int64_t lo = max((int64_t)start, first), hi = min((int64_t)start + nl, first + page);
  if (lo >= hi) return;
  const int id = pg < a.max_pages ? a.table[(int64_t)b * a.max_pages + pg] : -1;
  const int m = (int)(hi - lo), before = (int)(lo - first);
  const int vrow = (int)a.vrow.d, nvec = m * vrow;   // 16-byte vectors
  const T* src[W];
#pragma unroll
  for (int w = 0; w < W; ++w)
    src[w] = reinterpret_cast<const T*>(a.src[w]) + b * a.sb[w] + (lo - start) * a.ss[w] + h * a.sh[w];
  auto vec = [&](int w, int i) {
    const int r = (int)bs_div(i, a.vrow);
    return *reinterpret_cast<const uint4*>(src[w] + r * a.ss[w] + (i - r * vrow) * E);
  };
  // a thread's vectors are threadIdx.x + k nthr; the first kU stay in registers
  uint4 raw[W][kU];
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const int i = threadIdx.x + k * nthr;
      if (i < nvec) raw[w][k] = vec(w, i);
    }
  float amax[W];
  auto over_cta = [&]() {
#pragma unroll
    for (int w = 0; w < W; ++w) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax[w] = nan_max(amax[w], __shfl_xor_sync(0xffffffffu, amax[w], o));
      if ((threadIdx.x & 31) == 0) red[w][threadIdx.x >> 5] = amax[w];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w)
      for (int k = 0; k < warps; ++k) amax[w] = nan_max(amax[w], red[w][k]);
  };
#pragma unroll
  for (int w = 0; w < W; ++w) {
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < kU; ++k)
      if ((int)threadIdx.x + k * nthr < nvec) top = top_of<T>(raw[w][k], top);
#pragma unroll 4
    for (int i = threadIdx.x + kU * nthr; i < nvec; i += nthr) top = top_of<T>(vec(w, i), top);
    amax[w] = top_value<T>(top);
  }
  over_cta();
  bool odd = false;
#pragma unroll
  for (int w = 0; w < W; ++w) odd |= !(amax[w] < __uint_as_float(0x7F800000u));
  if (odd) {                                  // infinities or NaN: the same for the whole CTA
#pragma unroll
    for (int w = 0; w < W; ++w) {
      amax[w] = 0.0f;
#pragma unroll
      for (int k = 0; k < kU; ++k)
        if ((int)threadIdx.x + k * nthr < nvec) amax[w] = finite_top<T>(raw[w][k], amax[w]);
      for (int i = threadIdx.x + kU * nthr; i < nvec; i += nthr) amax[w] = finite_top<T>(vec(w, i), amax[w]);
    }
    __syncthreads();
    over_cta();
  }
  if (id < 0 || id >= a.n_pages) {            // looked at this late, its load is behind the rows'
    if (threadIdx.x == 0) bs_set_error(BS_ERR_BAD_INDEX);
    return;
  }
  const int64_t sat = (int64_t)id * a.Hkv + h;
  float s[W];
#pragma unroll
  for (int w = 0; w < W; ++w) s[w] = pow2_scale(amax[w]);
  if (before > 0) {
    float old[W];
#pragma unroll
    for (int w = 0; w < W; ++w) old[w] = a.scale[w][sat];
    __syncthreads();                          // every thread has read the old scales
#pragma unroll
    for (int w = 0; w < W; ++w) {
      s[w] = nan_max(s[w], old[w]);
      // grown, or no number: its codes are none then either (max and quotient as the formula has them)
      if (s[w] != old[w] || !(s[w] < __uint_as_float(0x7F800000u))) {
        const float f = __fdiv_rn(old[w], s[w]);
        const int n16 = before * a.D / 16;
        uint4* dst = reinterpret_cast<uint4*>(a.cache[w] + sat * ((int64_t)a.D << a.page_log2));
#pragma unroll 4
        for (int i = threadIdx.x; i < n16; i += nthr) {
          uint4 c = dst[i];
          uint32_t* p = reinterpret_cast<uint32_t*>(&c);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t v = p[k];
            p[k] = bs_cvt_e4m3x2(bs_e4m3_to_f32(v & 0xFF) * f, bs_e4m3_to_f32((v >> 8) & 0xFF) * f) |
                   ((uint32_t)bs_cvt_e4m3x2(bs_e4m3_to_f32((v >> 16) & 0xFF) * f, bs_e4m3_to_f32(v >> 24) * f) << 16);
          }
          dst[i] = c;
        }
      }
    }
  }
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (threadIdx.x == 0) a.scale[w][sat] = s[w];
    // the new rows lie one behind the other there
    uint8_t* dst = a.cache[w] + sat * ((int64_t)a.D << a.page_log2) + (int64_t)before * a.D;
    const bool pow2 = (__float_as_uint(s[w]) & 0x7FFFFFu) == 0 && s[w] >= 1.1754944e-38f && s[w] < 1.7e38f;
    const float inv = pow2 ? bs_inv_pow2(s[w]) : 0.0f;
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const int i = threadIdx.x + k * nthr;
      if (i < nvec) put_codes<T>(dst + i * E, raw[w][k], s[w], inv, pow2, odd);
    }
#pragma unroll 4
    for (int i = threadIdx.x + kU * nthr; i < nvec; i += nthr) put_codes<T>(dst + i * E, vec(w, i), s[w], inv, pow2, odd);
  }
  pdl_launch_dependents();
}

}  // namespace kvc

cudaError_t bs_launch_cache_append(kvc::Args a, int dtype, int both, cudaStream_t st) {
  // threads: one 16-byte vector of a page's new rows in each of the kU registers, from a warp to 512
  const int E = dtype == BS_DT_F32 ? 4 : 8, page = 1 << a.page_log2;
  a.vrow = bs_make_div(a.D / E);
  const int64_t vecs = (int64_t)(a.S < page ? a.S : page) * a.D / E;
  int threads = 32;
  while (threads < 512 && (int64_t)threads * kvc::kU < vecs) threads *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.span * a.Hkv));
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto go = [&](auto t) {
    using T = decltype(t);
    return both ? cudaLaunchKernelEx(&cfg, kvc::append_kernel<T, 2>, a) : cudaLaunchKernelEx(&cfg, kvc::append_kernel<T, 1>, a);
  };
  if (dtype == BS_DT_BF16) return go(__nv_bfloat16());
  if (dtype == BS_DT_F16) return go(__half());
  return go(float());
}
