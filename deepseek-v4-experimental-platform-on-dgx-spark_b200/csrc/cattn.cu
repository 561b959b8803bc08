// Attention of each sequence's newest tokens over a paged e4m3 cache with one
// scale per page and head (grouped-query heads; or one latent that is key and
// value at once), with an optional sink logit per head.
//
//   o[b, s, h] = sum_t w_t v_t / (sum_t w_t + e^{sink_h}),   w_t = exp(scale q.k_t)
//   over the cached tokens t < seq_len[b] - new[b] + s + 1
//
// The cached codes go from HBM to the tensor cores without being touched by a
// thread: TMA brings 128 tokens x 128 bytes into 128B-swizzled shared memory,
// and that one tile is the K-major A operand of S^T = K Q^T and, for values,
// the MN-major A operand of O^T = V^T P^T.  A tcgen05.mma with M = 128 costs
// the same for any N up to 128, so the few query rows of a decode step sit in
// N, and what e4m3 would lose of Q and P is bought back with more columns:
//
//   x = c1 + c2/16 + c3/256,  c1 = e4m3(x), c2 = e4m3(16 (x - c1)), ...
//
// Rounding to e4m3 leaves at most 2^-4 of the value's power of two, after the
// second term 2^-9 and after the third 2^-14, so two terms hold a bf16 value
// (8 bits) exactly and three an f16 value (11 bits).  Rows of Q are first
// scaled by a power of two so that their amax lies in [128, 256): what the
// terms cannot hold is below 2^-22 of the row's amax for two terms and 2^-26
// for three.  P = exp2(s - ref) * (page's value scale / largest of the tile) *
// 256 is rounded to the same number of terms: with bf16 outputs to 2^-8 of the
// value at most (2^-9, and f16 on the way; half a step of bf16 itself is
// 2^-8), with f16 outputs to 2^-14.  The terms end at a step, so this holds for
// P above 2^-6; below, half that step is left, 2^-14 (bf16) or 2^-18 (f16),
// 2^-22 or 2^-26 of the largest P there can be.  Hence ref is the row's maximum
// in this tile, not the one so far: what a dominant key costs the small weights
// beside it ends with its 128 tokens.  (Only tiles more than kReach = 24 powers
// of two below the maximum so far use that minus kReach, so that sums stay in
// range: there weights below 2^-46 of the largest are lost.)  Where the value
// scales of a tile's pages differ by more than kSpread = 4, the largest may be
// that of a page which a row does not see or hardly weighs; in such tiles ref is
// the row's largest product of weight and scale (scales below 2^-kFar = 2^-64 of
// the largest count as that, so that weights stay in range).
// Accumulation is fp32 in TMEM; O is taken out after every tile and added, in
// fp32, to accumulators in registers, which follow ref from tile to tile (times
// 2^-kReach, so that they are never above the result's own size) and where the
// tile's value scale is applied.
//
// One work unit is a tile: 128 tokens of one (sequence, row tile, kv head);
// a row tile is R of the S * (H / Hkv) query rows of a kv head.  All tiles of
// the call lie in one line, every head's preceded by what its start and end
// cost (in tiles), and each resident CTA takes an equal stretch of the line,
// whatever the lengths; where a stretch ends inside a head's tokens, both
// sides leave partial results (unnormalised O, reference, sum) and a second kernel
// joins them.  Lengths are read on the device only.
//
// What bounds it: few rows, HBM (64 sequences of up to 16384 tokens, 8 kv heads
// of 128, 8 query heads each: 1.09 GB of codes in 186 to 192 us, 0.87 to 0.90 of
// the copy bandwidth; 200000 tokens f16, 3 terms: 77 to 79 us, 0.80 to 0.82); 64
// rows a tile, the instructions of the softmax (a chunk of 512 tokens on 8192:
// 291 us, issue slots 65 % busy, 32 instructions a score); a latent of 512 dims
// with 64 heads, the chain copy - S - softmax - O of a ring of two and a half
// tiles, each fetched twice, as its 64 rows take two row tiles (48 sequences of
// up to 8192: 85 us, 304 TFLOP/s).  Tiles of spread scales on every page: 187,
// 77, 338 and 87 us.
//
// Roles: one warpgroup with the TMA producer and an issuer for each of the two
// products; one softmax warpgroup, or from 32 rows on one for every 16 of them;
// one that stages Q and accumulates O, one head dim per thread and 128-dim
// chunk.  Shared memory: rings of 16 KB chunks, Q (this segment's and, where it
// fits, the next one's), two P buffers.
#include <type_traits>

#include "common.cuh"

namespace cattn {

constexpr int kTok = 128;
constexpr int kChunk = kTok * 128;
constexpr int kInfo = 16;          // tile info ring: above the tiles between the producer and the accumulators
constexpr int kSegRing = 5;        // row sums of finished segments: the softmax warps run at most four segments ahead
constexpr int kMaxSlots = 12;
constexpr float kReach = 24.0f;    // powers of two that a tile's reference may lie below the row's maximum
constexpr float kReachScale = 16777216.0f;
constexpr float kSpread = 4.0f;    // largest ratio of a tile's value scales that the maximum of the scores takes as one
constexpr float kFar = 64.0f;

struct Args {
  const void* q;
  int64_t q_sb, q_ss, q_sh;        // strides in elements
  const float* k_scale;
  const float* v_scale;            // [n_pages, Hkv]
  const int* table;                // [B, max_pages]
  const int* seq_lens;
  const int* new_lens;             // or null: S for every sequence
  const float* sink;               // [H] or null
  void* out;                       // [B, S, H, D]
  int* plan;                       // [1 + B * RT]: places per CTA, first place of each (sequence, row tile)
  float* part_ml;                  // [2 * grid][R][2]: reference, sum
  float* part_o;                   // [2 * grid][R][NC * 128]
  int B, S, H, Hkv, G, D, RT, page_log2, max_pages, n_pages;
  float scale_log2;                // softmax scale x log2(e)
  int seg_cost;                    // Cfg::kSegCost, for the joining kernel
  int shared;                      // values are the keys' codes
};

// Lengths of one sequence as the kernels use them; what is out of range reads as nothing and is recorded.
struct Seq {
  int len, nl;
};
BS_DEVINL Seq load_seq(const Args& a, int b, bool report) {
  Seq s;
  s.len = a.seq_lens[b];
  s.nl = a.new_lens ? a.new_lens[b] : a.S;
  const int64_t most = (int64_t)a.max_pages << a.page_log2;
  if (s.len < 0 || s.len > most || s.nl < 0 || s.nl > a.S) {
    if (report) bs_set_error(BS_ERR_BAD_INDEX);
    s.len = 0;
    s.nl = 0;
  }
  return s;
}
// Tokens that query token i sees (0 for a padded one).
BS_DEVINL int row_limit(const Seq& s, int i) { return i < s.nl ? max(0, s.len - s.nl + i + 1) : 0; }
// Tokens that any row of row tile rt sees: those of its last row.
BS_DEVINL int tile_limit(const Args& a, const Seq& s, int rt, int R) {
  const int last = min((rt + 1) * R, a.S * a.G) - 1;
  const int i = min(last / a.G, s.nl - 1);
  return i < rt * R / a.G ? 0 : row_limit(s, i);
}
BS_DEVINL int tiles_of(int limit) { return (limit + kTok - 1) / kTok; }

// A CTA's walk over its share: units (b, rt) in order, within a unit all kv heads, within a head its tiles.
struct Walk {
  int unit, h, t, nt;
  int b, rt, limit;
  Seq s;
  int left;
  bool fresh;                       // nothing of this segment has been taken yet
  BS_DEVINL void enter(const Args& a, int R) {
    b = unit / a.RT;
    rt = unit - b * a.RT;
    s = load_seq(a, b, false);
    limit = tile_limit(a, s, rt, R);
    nt = tiles_of(limit);
  }
  BS_DEVINL int seg_end() const { return min(nt, t + left); }
  BS_DEVINL void next(const Args& a, int R) {
    left -= seg_end() - t;
    t = 0;
    fresh = true;
    if (left <= 0) return;
    if (++h == a.Hkv) {
      h = 0;
      do {
        if (++unit >= a.B * a.RT) {   // left > 0 means a later unit has tiles, unless the lengths changed under the call
          left = 0;
          return;
        }
        enter(a, R);
      } while (nt == 0);
    }
  }
};

struct Info {                       // one tile, from the producer
  float ks[8];                      // per page of the tile
  float vr[8];                      // 256 x value scale / unit
  float unit;                       // largest |value scale| that is a number
  int valid;                        // bits of the pages that are there
  int t0;                           // first token
  int limit;                        // tokens that any row sees
  int first, last;                  // of its segment
  int mask;                         // 1: some row does not see all of the tile; 2: value scales (not 0) kSpread apart
  int nan;                          // bits of the pages whose value scale is NaN
};

__host__ __device__ constexpr int softmax_groups(int R) { return R >= 32 ? R / 16 : 1; }

template <int R, int PP, int NC>
struct Cfg {
  static constexpr int N = R * PP % 16 ? R * PP + 8 : R * PP;      // columns of one MMA
  static constexpr int WG = softmax_groups(R);                     // softmax warpgroups
  static constexpr int RW = R / WG;                                // rows of each
  static constexpr int kThreads = 128 * (2 + WG);
  static constexpr int kQBytes = NC * N * 128;
  static constexpr int kPBytes = N * kTok;
  static constexpr int QB = kQBytes >= 32768 ? 1 : 2;              // Q buffers
  // Places before a head's tiles on the line of work, for staging its rows, draining the pipeline and writing its
  // results.  Measured with 0 to 8: 1 is best for 64 ragged sequences of 8 rows a head (182 us then; 0: 184, 2: 183), 4 to 6
  // for a chunk of 512 tokens (301 us then; 2: 333, 8: 305), 6 to 8 with one Q buffer (latent: 89 us then; 2: 97).
  static constexpr int kSegCost = QB == 1 ? 7 : WG > 1 ? 5 : 1;
  static constexpr int OB = 2 * N + 2 * NC * N <= 512 ? 2 : 1;     // O buffers
  static constexpr int SB = 2 * N + OB * NC * N <= 512 ? 2 : 1;    // S buffers
  static constexpr int kCols = SB * N + OB * NC * N;
  static constexpr int kTmem = kCols <= 32 ? 32 : kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kCols <= 512 && N % 16 == 0 && N <= 256, "TMEM");
  struct alignas(16) Tail {         // behind the ring, Q and P
    Info info[kInfo];
    float qf[2][R];                 // 2^-k x |scale| x log2(e) of each row
    int lim[2][R];                  // tokens each row sees
    int64_t off[2][R];              // element offset of the row's output, -1: no row
    float wmax[2][R][4], alpha[4][R];
    float lsum[kSegRing][4][R], mfin[kSegRing][R], fin[2][R];
    int nanmin[kSegRing][NC * 128]; // first token with a NaN value in partly hidden tiles
    int nanseen[kSegRing];
    uint64_t full[kMaxSlots], empty[kMaxSlots];
    uint64_t s_full[2], s_empty[2], p_full[2], p_empty[2], o_full[2], o_empty[2], q_full[2], l_full[kSegRing], v_ready;
    uint32_t tmem;
    int abort;
    int2 scan[24];
    int first_tile, end_tile;       // its tiles on the line
    Walk start;                     // where this CTA's share begins
  };
  static constexpr int kFixed = 1024 + QB * kQBytes + 2 * kPBytes + (int)sizeof(Tail);
  // Two CTAs an SM for the small row tiles of a decode step: a tile's chain of waits (keys, S, maximum, P, O) is longer
  // than its bytes take, and two such chains overlap.
  static constexpr int kCtas = NC == 1 && R <= 16 ? 2 : 1;
  static_assert(kCtas * kTmem <= 512, "TMEM of the resident CTAs");
  static constexpr int kFit = ((kCtas == 2 ? 113 : 227) * 1024 - kFixed) / kChunk;
  static constexpr int kSlots = kFit < kMaxSlots ? kFit : kMaxSlots;
  // Separate rings for keys and values: each product's issuer then sees every phase of the barriers it waits for.  (In
  // one ring of mixed chunks a slot's previous phase could belong to the other product, still incomplete, and a parity
  // wait takes a phase two ahead for one that is over.)  Values that are the keys use one ring of all slots.
  static constexpr int kVSlots = kSlots / 2, kKSlots = kSlots - kVSlots;
  static_assert(kVSlots >= NC && kSlots + 4 <= kInfo, "rings");
  static constexpr int kSmem = kFixed + kSlots * kChunk;
};

// Descriptor of a 128-token x 128-byte tile (128B swizzle) read along tokens: M is the byte within a row, K the row.
// 8 rows (1024 bytes) to the next group along K; M = 128 is one swizzle atom wide.
BS_DEVINL uint64_t sdesc_mn_sw128(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFF);
  d |= (uint64_t)(1024 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// Descriptor of P: [N / 16][128 tokens][16 bytes], no swizzle; 128 bytes to the next 8 tokens, 2048 to the next 16 columns.
BS_DEVINL uint64_t sdesc_mn_plain(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFF);
  d |= (uint64_t)(128 >> 4) << 16;
  d |= (uint64_t)(2048 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  return d;
}

// mbar_wait behind a non-suspending probe.  A phase that is over costs 7 cycles this way and 70 with try_wait.
BS_DEVINL bool wait_quick(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return mbar_test_wait(bar, parity) || mbar_wait(bar, parity, abort);
}
// A whole warp waits, each lane for its own barrier (lanes with active = false for none).  The first probe does not
// diverge; lanes that have to wait for good then do so one after another.
BS_DEVINL bool warp_wait(uint64_t* bar, uint32_t parity, bool active, volatile int* abort) {
  bool ok = !active || mbar_test_wait(bar, parity);
  if (__all_sync(0xffffffffu, ok)) return true;
  if (!ok) ok = mbar_wait(bar, parity, abort);
  return __all_sync(0xffffffffu, ok);
}

// Barrier of one warpgroup that also says whether all of it is still alive.
BS_DEVINL bool group_all(int id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok), "r"(id)
      : "memory");
  return r != 0;
}
BS_DEVINL float lds_f32(uint32_t addr) {
  float v;
  asm("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
BS_DEVINL int64_t lds_s64(uint32_t addr) {
  int64_t v;
  asm("ld.shared.s64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
template <int N>
BS_DEVINL void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
BS_DEVINL void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// Two fp32 operations in one instruction.
BS_DEVINL float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
BS_DEVINL float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
BS_DEVINL float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
BS_DEVINL float2 both(float x) { return make_float2(x, x); }

// 2^x to 2 ulp; exponents below -126 give 0.
BS_DEVINL float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two e4m3 codes -> f16 (exact).
BS_DEVINL __half2 e4m3x2_to_h2(uint16_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  return *reinterpret_cast<__half2*>(&h);
}
BS_DEVINL uint16_t h2_to_e4m3x2(__half2 v) {
  uint16_t c;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(c) : "r"(*reinterpret_cast<uint32_t*>(&v)));
  return c;
}
// The PP terms of two values of Q: they are f16 numbers here (8 or 11 bits on a scale where the row's largest is in
// [128, 256); what f16 loses is below 2^-25 on that scale).  Differences of a value and its nearest e4m3 neighbour are
// exact.
template <int PP>
BS_DEVINL void split2h(float x, float y, uint16_t* c) {
  __half2 v = __floats2half2_rn(x, y);
#pragma unroll
  for (int p = 0; p < PP; ++p) {
    c[p] = h2_to_e4m3x2(v);
    if (p + 1 < PP) v = __hmul2(__hsub2(v, e4m3x2_to_h2(c[p])), __float2half2_rn(16.0f));
  }
}
// The same for two weights: with two terms (2^-9 of the value is left) through f16, whose 2^-11 is below that; with three
// (2^-14) in fp32.
template <int PP>
BS_DEVINL void split2p(float x, float y, uint16_t* c) {
  if constexpr (PP == 2) {
    split2h<PP>(x, y, c);
  } else {
#pragma unroll
    for (int p = 0; p < PP; ++p) {
      c[p] = bs_cvt_e4m3x2(x, y);
      if (p + 1 < PP) {
        const float2 b = __half22float2(e4m3x2_to_h2(c[p]));
        const float2 r = mul2(add2(make_float2(x, y), make_float2(-b.x, -b.y)), both(16.0f));
        x = r.x;
        y = r.y;
      }
    }
  }
}

// 16 TMEM lanes x 8 K columns: v[4g + 2i + j] is lane (thread / 4) + 8i, column 8g + 2 (thread % 4) + j.
template <int K>
BS_DEVINL void tmem_ld16x256(uint32_t taddr, uint32_t* v) {
  if constexpr (K == 1) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(taddr));
  } else {
    static_assert(K == 2, "16x256b.x2");
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr));
  }
}

// B of the R values of one TMEM lane out of their PP terms: columns term * R + row.
template <int R, int PP, int B>
BS_DEVINL void load_rows(uint32_t taddr, float* s) {
  if constexpr (R == 8) {
    uint32_t v[PP == 2 ? 16 : 32];             // all terms lie side by side
    if constexpr (PP == 2) BS_TMEM_LD16(taddr, v);
    else BS_TMEM_LD32(taddr, v);
    tmem_ld_wait();
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      float x = __uint_as_float(v[(PP - 1) * 8 + r]);
#pragma unroll
      for (int p = PP - 2; p >= 0; --p) x = fmaf(x, 0.0625f, __uint_as_float(v[p * 8 + r]));
      s[r] = x;
    }
  } else {
    static_assert(B == 16 || B == 32, "rows of a load");
    uint32_t v[PP][B];
#pragma unroll
    for (int p = 0; p < PP; ++p) {
      if constexpr (B == 16) BS_TMEM_LD16(taddr + p * R, v[p]);
      else BS_TMEM_LD32(taddr + p * R, v[p]);
    }
    tmem_ld_wait();
#pragma unroll
    for (int r = 0; r < B; r += 2) {
      float2 x = make_float2(__uint_as_float(v[PP - 1][r]), __uint_as_float(v[PP - 1][r + 1]));
#pragma unroll
      for (int p = PP - 2; p >= 0; --p)
        x = fma2(x, both(0.0625f), make_float2(__uint_as_float(v[p][r]), __uint_as_float(v[p][r + 1])));
      s[r] = x.x;
      s[r + 1] = x.y;
    }
  }
}

// Row of column r of P and O.  From 16 rows on, the columns of 16 rows are in the order in which the softmax threads hold
// them: rows 2i, 2i + 1, 2i + 8, 2i + 9 of thread i of 4 lie side by side, one 4-byte store.
template <int R>
__host__ __device__ constexpr int row_of(int r) {
  return R < 16 ? r : (r & ~15) + 8 * ((r >> 1) & 1) + 2 * ((r >> 2) & 3) + (r & 1);
}

// e4m3 NaN (0x7F or 0xFF) among four codes: bytes whose low seven bits are all set.
BS_DEVINL uint32_t nan_bytes(uint32_t v) { return ((v & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

template <int R, int PP, int NC>
__global__ void __launch_bounds__(Cfg<R, PP, NC>::kThreads, Cfg<R, PP, NC>::kCtas)
    cache_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Args a) {
  using C = Cfg<R, PP, NC>;
  constexpr int N = C::N, kThreads = C::kThreads;
  constexpr uint32_t SLOTS = C::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* qbuf = smem + SLOTS * kChunk;
  uint8_t* pbuf = qbuf + C::QB * C::kQBytes;
  typename C::Tail& T = *reinterpret_cast<typename C::Tail*>(pbuf + 2 * C::kPBytes);
  volatile int* abort_flag = &T.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < (int)SLOTS; ++i) {
      mbar_init(&T.full[i], 1);
      mbar_init(&T.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&T.s_full[i], 1);
      mbar_init(&T.s_empty[i], 4 * C::WG);
      mbar_init(&T.p_full[i], 4 * C::WG);
      mbar_init(&T.p_empty[i], 1);
      mbar_init(&T.o_full[i], 1);
      mbar_init(&T.o_empty[i], 4);
      mbar_init(&T.q_full[i], 4);
    }
    for (int i = 0; i < kSegRing; ++i) mbar_init(&T.l_full[i], 4 * C::WG);
    mbar_init(&T.v_ready, 1);
    T.abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_k);
    if (!a.shared) tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(&T.tmem, C::kTmem);
    tmem_relinquish();
  }
  // columns that hold no row stay zero
  if (N != R * PP) {
    for (int i = tid; i < C::QB * C::kQBytes / 16; i += kThreads) reinterpret_cast<uint4*>(qbuf)[i] = make_uint4(0, 0, 0, 0);
    for (int i = tid; i < 2 * C::kPBytes / 16; i += kThreads) reinterpret_cast<uint4*>(pbuf)[i] = make_uint4(0, 0, 0, 0);
  }
  pdl_launch_dependents();
  pdl_wait();

  // ---- the share of this CTA: tiles [start, start + count) of all
  const int units = a.B * a.RT;
  Walk mine;
  auto unit_tiles = [&](int u, bool report) -> int {
    if (u >= units) return 0;
    mine.unit = u;
    mine.enter(a, R);
    if (report && mine.rt == 0) load_seq(a, mine.b, true);
    return a.Hkv * mine.nt;
  };
  auto warp_sum = [&](int x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
  };
  // Lengths of the line: in places (tiles and the costs before them), and in tiles.
  int total = 0, tiles = 0;
  if (units > kThreads) {            // else one pass below sees them all
    int x = 0, y = 0;
    for (int u = tid; u < units; u += kThreads) {
      const int n = unit_tiles(u, false);
      y += n;
      x += n ? n + a.Hkv * C::kSegCost : 0;
    }
    x = warp_sum(x);
    y = warp_sum(y);
    if (lane == 0) T.scan[warp] = make_int2(x, y);
    __syncthreads();
    for (int i = 0; i < kThreads / 32; ++i) {
      total += T.scan[i].x;
      tiles += T.scan[i].y;
    }
    __syncthreads();
  }
  int start = 0, end = 0;
  int2 before = make_int2(0, 0);
  for (int u0 = 0; u0 == 0 || u0 < units; u0 += kThreads) {
    const int n = unit_tiles(u0 + tid, blockIdx.x == 0);
    const int2 x = make_int2(n ? n + a.Hkv * C::kSegCost : 0, n);
    int2 inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc.x, o), z = __shfl_up_sync(0xffffffffu, inc.y, o);
      if (lane >= o) {
        inc.x += y;
        inc.y += z;
      }
    }
    if (lane == 31) T.scan[warp] = inc;
    if (u0 == 0) {
      // the rest of the start-up, while the lengths are on their way
      for (int i = tid; i < kSegRing * NC * 128; i += kThreads) (&T.nanmin[0][0])[i] = 0x7FFFFFFF;
      if (tid < kSegRing) T.nanseen[tid] = 0;
      fence_proxy_async_smem();
      tc_fence_before();
    }
    __syncthreads();
    if (u0 == 0) tc_fence_after();
    int2 base = before, sum = make_int2(0, 0);
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
      const int2 y = T.scan[i];
      if (i < warp) {
        base.x += y.x;
        base.y += y.y;
      }
      sum.x += y.x;
      sum.y += y.y;
    }
    if (units <= kThreads) {
      total = sum.x;
      tiles = sum.y;
    }
    if (u0 == 0) {
      const int per = (total + (int)gridDim.x - 1) / (int)gridDim.x;
      start = min(per * (int)blockIdx.x, total);
      end = min(start + per, total);
      if (blockIdx.x == 0 && tid == 0) a.plan[0] = per;
      if (tid == 0 && start == total) T.first_tile = tiles;
      if (tid == 0 && end == total) T.end_tile = tiles;
    }
    const int first = base.x + inc.x - x.x, first_tile = base.y + inc.y - x.y;
    // tiles of the line before place p of this unit; h and t: the head and tile there
    auto place = [&](int p, int& h, int& t) {
      const int each = mine.nt + C::kSegCost;
      h = (p - first) / each;
      t = max(0, p - first - h * each - C::kSegCost);
      return first_tile + h * mine.nt + t;
    };
    if (start >= first && start < first + x.x) {
      T.first_tile = place(start, mine.h, mine.t);
      mine.fresh = true;
      T.start = mine;
    }
    if (end >= first && end < first + x.x) {
      int h, t;
      T.end_tile = place(end, h, t);
    }
    if (blockIdx.x == 0 && u0 + tid < units) a.plan[1 + u0 + tid] = first;
    before.x += sum.x;
    before.y += sum.y;
    __syncthreads();
    if (blockIdx.x != 0 && before.x > end) break;
  }
  const int count = T.end_tile - T.first_tile;
  const uint32_t tmem = T.tmem;
  // Slot of a running chunk number (tile x NC + c) and the parity of its phase.
  constexpr uint32_t KS = C::kKSlots, VS = C::kVSlots;
  auto k_slot = [&](uint32_t n) -> uint32_t { return a.shared ? n % SLOTS : n % KS; };
  auto k_par = [&](uint32_t n) -> uint32_t { return (a.shared ? n / SLOTS : n / KS) & 1; };
  auto v_slot = [&](uint32_t n) -> uint32_t { return a.shared ? n % SLOTS : KS + n % VS; };
  auto v_par = [&](uint32_t n) -> uint32_t { return (a.shared ? n / SLOTS : n / VS) & 1; };
  // Registers move from the issuing and softmax warpgroups to the accumulators; the shares add up to the launch's
  // 4 x 128 or 6 x 80.
  constexpr bool kSplitRegs = C::WG >= 2;
  constexpr int kIssueRegs = C::WG == 4 ? 64 : NC * R > 64 ? 72 : 120, kSoftRegs = C::WG == 4 ? 72 : NC * R > 64 ? 112 : 120,
                kAccRegs = C::WG == 4 ? 128 : NC * R > 64 ? 216 : 152;
  static_assert(!kSplitRegs || kIssueRegs + C::WG * kSoftRegs + kAccRegs == (C::WG == 4 ? 6 * 80 : 4 * 128), "registers");

  if (warp < 4) {
    if constexpr (kSplitRegs) reg_dec<kIssueRegs>();
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      const int ppt = kTok >> a.page_log2, page = 1 << a.page_log2;
      const int per_batch = 32 / ppt;            // tiles whose pages fit the lanes
      const int oob = a.n_pages * a.Hkv;         // a page row past the end: TMA fills zeros
      // Page rows and scales of the next tiles, one page per lane, loaded while the previous batch is sent.
      struct Batch {
        int prow, n, t, limit, low, first, last;
        uint32_t there;
        float ks, vs;
      };
      Walk w = T.start;
      w.left = count;
      auto load = [&](Batch& o) {
        o.n = 0;
        if (w.left <= 0) return;
        const int end = w.seg_end();
        o.t = w.t;
        o.n = min(end - w.t, per_batch);
        o.limit = w.limit;
        o.low = row_limit(w.s, w.rt * R / a.G);      // rows of the tile see at least the first row's tokens
        o.first = w.fresh;
        o.last = w.t + o.n == end;
        o.prow = oob;
        o.ks = o.vs = 0.0f;
        bool there = false;
        const int64_t p = (int64_t)o.t * ppt + lane;
        if (lane < o.n * ppt && (p << a.page_log2) < w.limit) {
          const int id = a.table[(int64_t)w.b * a.max_pages + p];
          there = id >= 0 && id < a.n_pages;
          if (there) {
            o.prow = id * a.Hkv + w.h;
            o.ks = a.k_scale[o.prow];
            o.vs = a.shared ? o.ks : a.v_scale[o.prow];
          } else {
            bs_set_error(BS_ERR_BAD_INDEX);
          }
        }
        o.there = __ballot_sync(0xffffffffu, there);
        if (o.last) {
          w.next(a, R);
        } else {
          w.t += o.n;
          w.left -= o.n;
          w.fresh = false;
        }
      };
      uint32_t k_sent = 0, v_sent = 0;           // chunks
      bool ok = true;
      auto chunk = [&](const CUtensorMap* m, uint32_t slot, uint32_t parity, int x, int prow) {
        ok = ok && __all_sync(0xffffffffu, wait_quick(&T.empty[slot], parity ^ 1, abort_flag));
        if (!ok) return;
        if (lane == 0) mbar_arrive_expect_tx(&T.full[slot], kChunk);
        __syncwarp();
        if (lane < ppt) tma_load_3d(smem + slot * kChunk + lane * page * 128, m, &T.full[slot], x, 0, prow);
        __syncwarp();
      };
      auto k_chunks = [&](int prow) {
        for (int c = 0; c < NC && ok; ++c) {
          chunk(&tm_k, k_slot(k_sent), k_par(k_sent), c * 128, prow);
          k_sent += ok;
        }
      };
      auto v_chunks = [&](int prow) {
        for (int c = 0; c < NC && ok; ++c) {
          chunk(&tm_v, v_slot(v_sent), v_par(v_sent), c * 128, prow);
          v_sent += ok;
        }
      };
      Batch cur, nxt;
      load(cur);
      load(nxt);
      int v_prow = 0;                            // the previous tile's page row of this lane, for its values
      bool v_pending = false;
      uint32_t tile = 0;
      while (cur.n > 0 && ok) {
        for (int k = 0; k < cur.n && ok; ++k, ++tile) {
          const int src = (k * ppt + (lane & (ppt - 1))) & 31;
          const int prow = __shfl_sync(0xffffffffu, cur.prow, src);
          const float ks = __shfl_sync(0xffffffffu, cur.ks, src), vs = __shfl_sync(0xffffffffu, cur.vs, src);
          const uint32_t valid = (cur.there >> (k * ppt)) & ((1u << ppt) - 1u);
          float unit = vs == vs ? fabsf(vs) : 0.0f;   // a NaN scale stays with its page
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) unit = fmaxf(unit, __shfl_xor_sync(0xffffffffu, unit, o));
          // the first slot of the tile free: the entry's last reader is far behind
          ok = __all_sync(0xffffffffu, wait_quick(&T.empty[k_slot(k_sent)], k_par(k_sent) ^ 1, abort_flag));
          if (!ok) break;
          Info& in = T.info[tile % kInfo];
          // a NaN scale makes its page's weights NaN where every row sees the tile; else they are 0, and the softmax
          // warps note the page's tokens as NaN values
          const bool spread = __any_sync(0xffffffffu, vs != 0.0f && fabsf(vs) * kSpread < unit);
          const bool mask = (cur.t + k + 1) * kTok > cur.low || valid != (1u << ppt) - 1u;
          const uint32_t nan = __ballot_sync(0xffffffffu, vs != vs) & ((1u << ppt) - 1u);
          if (lane < 8) {
            in.ks[lane] = ks;
            in.vr[lane] = vs != vs ? (mask ? 0.0f : vs) : unit > 0.0f ? 256.0f * (vs / unit) : 0.0f;
          }
          if (lane == 0) {
            const int t = cur.t + k;
            in.unit = unit;
            in.valid = (int)valid;
            in.t0 = t * kTok;
            in.limit = cur.limit;
            in.first = cur.first && k == 0;
            in.last = cur.last && k + 1 == cur.n;
            in.mask = (mask ? 1 : 0) | (spread ? 2 : 0);
            in.nan = (int)nan;
          }
          __syncwarp();
          k_chunks(prow);
          if (!a.shared) {
            if (v_pending && ok) v_chunks(v_prow);
            v_prow = prow;
            v_pending = true;
          }
        }
        cur = nxt;
        load(nxt);
      }
      if (v_pending && ok) v_chunks(v_prow);
      // on the way out after a timeout: the copies in flight still write this CTA's shared memory
      if (!ok) {
        auto drain = [&](uint32_t slot, uint32_t parity) {
          uint64_t t0 = 0;
          for (uint32_t j = 0; j < BS_SPIN_LIMIT; ++j)
            if (mbar_try_wait(&T.full[slot], parity) || bs_wait_expired(j, &t0)) break;
        };
        const uint32_t nk = min(k_sent, a.shared ? SLOTS : KS), nv = min(v_sent, VS);
        for (uint32_t k = 1; k <= nk; ++k) drain(k_slot(k_sent - k), k_par(k_sent - k));
        for (uint32_t k = 1; k <= nv; ++k) drain(v_slot(v_sent - k), v_par(v_sent - k));
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- S = K Q^T
      // One lane per barrier: the waits of a tile one after another, in one warp for both products, took longer than
      // its products (1925 cycles a tile of 128 x 128).
      constexpr uint32_t idesc = idesc_f8f6f4(0, 0, 128, N);
      const uint64_t dk = sdesc_k128_sw128(smem_u32(smem));
      const uint64_t dq = sdesc_k128_sw128(smem_u32(qbuf));
      int seg = -1;
      for (uint32_t i = 0; i < (uint32_t)count; ++i) {
        const uint32_t sb = i % C::SB;
        if (!warp_wait(lane ? &T.s_empty[sb] : &T.full[k_slot(i * NC)], lane ? ((i / C::SB) & 1) ^ 1 : k_par(i * NC), lane < 2,
                       abort_flag))
          break;
        if (T.info[i % kInfo].first) {
          ++seg;
          if (!warp_wait(&T.q_full[seg % C::QB], (seg / C::QB) & 1, true, abort_flag)) break;
        }
        bool ok = true;
#pragma unroll
        for (int c = 0; c < NC; ++c) {         // each chunk as it comes in
          const uint32_t slot = k_slot(i * NC + c);
          if (c > 0) ok = ok && warp_wait(&T.full[slot], k_par(i * NC + c), true, abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t da = dk + (uint64_t)(slot * kChunk >> 4);
            const uint64_t db = dq + (uint64_t)(((seg % C::QB) * C::kQBytes + c * N * 128) >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) tc_mma_f8f6f4(tmem + sb * N, da + 2 * k, db + 2 * k, idesc, (c | k) != 0);
            if (!a.shared) tc_commit(&T.empty[slot]);
            if (c == NC - 1) tc_commit(&T.s_full[sb]);
          }
          __syncwarp();
        }
        if (!ok) break;
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------- O = V^T P^T
      constexpr uint32_t idesc = idesc_f8f6f4(0, 0, 128, N) | (1u << 15) | (1u << 16);   // A and B along M / N
      const uint64_t dv = sdesc_mn_sw128(smem_u32(smem));
      const uint64_t dp = sdesc_mn_plain(smem_u32(pbuf));
      for (uint32_t i = 0; i < (uint32_t)count; ++i) {
        const uint32_t pb = i & 1, ob = i % C::OB;
        const uint32_t at = i * NC + min(lane, NC - 1);
        if (!warp_wait(&T.full[v_slot(at)], v_par(at), lane < NC, abort_flag)) break;
        // the softmax warps look the values of a partly hidden tile over before they hand in its weights
        if (lane == 0 && (T.info[i % kInfo].mask & 1)) mbar_arrive(&T.v_ready);
        __syncwarp();
        if (!warp_wait(lane ? &T.o_empty[ob] : &T.p_full[pb], lane ? ((i / C::OB) & 1) ^ 1 : (i >> 1) & 1, lane < 2, abort_flag))
          break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t db = dp + (uint64_t)(pb * C::kPBytes >> 4);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const uint32_t slot = v_slot(i * NC + c);
            const uint64_t da = dv + (uint64_t)(slot * kChunk >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)        // 32 tokens each: 4096 bytes of V, 512 of P
              tc_mma_f8f6f4(tmem + C::SB * N + (ob * NC + c) * N, da + (4096 >> 4) * k, db + (512 >> 4) * k, idesc, k != 0);
            tc_commit(&T.empty[slot]);
          }
          tc_commit(&T.p_empty[pb]);
          tc_commit(&T.o_full[ob]);
        }
        __syncwarp();
      }
    }
  } else if (warp < 4 + 4 * C::WG) {
    // ------------------------------------------------------------ softmax
    // A thread holds tokens tok0 + 8k (k = 0..3) of rows row0 + 8g + {0, 1} (g < K).
    if constexpr (kSplitRegs) reg_dec<kSoftRegs>();
    constexpr int RW = C::RW, K = RW / 8;
    const int wg = (warp >> 2) - 1, quad = warp & 3;
    const int tok0 = quad * 32 + (lane >> 2);
    const int row0 = wg * RW + 2 * (lane & 3);
    const uint32_t t_lane = tmem + ((uint32_t)(quad * 32) << 16) + wg * RW;
    float2 l[K], m[K], ref[K], qf[K];    // sum relative to 2^ref, maximum so far
    int seg = -1, masked = 0;
    bool dead = false;
    for (int i = 0; i < count; ++i) {
      const int sb = i % C::SB, pb = i & 1;
      const Info& in = T.info[i % kInfo];
      const bool ok = warp_wait(lane ? &T.p_empty[pb] : &T.s_full[sb], lane ? ((i >> 1) & 1) ^ 1 : (i / C::SB) & 1,
                                lane < 2, abort_flag) &&
                      !dead;
      float2 s[K][4];
      if (ok) {
        tc_fence_after();
        {
          uint32_t v[2][PP][4 * K];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int p = 0; p < PP; ++p) tmem_ld16x256<K>(t_lane + ((uint32_t)(16 * h) << 16) + sb * N + p * R, v[h][p]);
          if (in.first) {
            ++seg;
#pragma unroll
            for (int g = 0; g < K; ++g) {
              qf[g] = *reinterpret_cast<const float2*>(&T.qf[seg & 1][row0 + 8 * g]);
              m[g] = ref[g] = both(-INFINITY);
              l[g] = both(0.0f);
            }
          }
          float ks[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) ks[k] = in.ks[(tok0 + 8 * k) >> a.page_log2];
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&T.s_empty[sb]);
#pragma unroll
          for (int g = 0; g < K; ++g)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int at = 4 * g + 2 * (k & 1);
              auto term = [&](int p) {
                return make_float2(__uint_as_float(v[k >> 1][p][at]), __uint_as_float(v[k >> 1][p][at + 1]));
              };
              float2 x = term(PP - 1);
#pragma unroll
              for (int p = PP - 2; p >= 0; --p) x = fma2(x, both(0.0625f), term(p));
              s[g][k] = mul2(x, both(ks[k]));
            }
        }
        // Maxima of the thread's 2K rows over its tokens, then over the warp's 32, in a butterfly that halves the rows with
        // the lanes: lane group (lane / 4) % 2K ends up with row 8 (v / 2) + v % 2 of v = that number.
        float x[2 * K];
        auto over_tokens = [&](auto of) {
#pragma unroll
          for (int g = 0; g < K; ++g) {
            x[2 * g] = fmaxf(fmaxf(of(s[g][0].x, 0, qf[g].x), of(s[g][1].x, 1, qf[g].x)),
                             fmaxf(of(s[g][2].x, 2, qf[g].x), of(s[g][3].x, 3, qf[g].x)));
            x[2 * g + 1] = fmaxf(fmaxf(of(s[g][0].y, 0, qf[g].y), of(s[g][1].y, 1, qf[g].y)),
                                 fmaxf(of(s[g][2].y, 2, qf[g].y), of(s[g][3].y, 3, qf[g].y)));
          }
        };
        if (in.mask) {
#pragma unroll
          for (int g = 0; g < K; ++g) {
            const int2 lim = *reinterpret_cast<const int2*>(&T.lim[seg & 1][row0 + 8 * g]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int tok = tok0 + 8 * k, t = in.t0 + tok;
              const bool there = (in.valid >> (tok >> a.page_log2)) & 1;
              if (!there || t >= lim.x) s[g][k].x = -INFINITY;
              if (!there || t >= lim.y) s[g][k].y = -INFINITY;
            }
          }
          // (asked here, not for every tile: beside this choice the code of all tiles came out 12 % slower)
          if (in.mask & 2) {         // of score and the scale's logarithm (x is multiplied by qf afterwards)
            float lv[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              lv[k] = fmaxf(__log2f(fabsf(in.vr[(tok0 + 8 * k) >> a.page_log2]) * (1.0f / 256.0f)), -kFar);
            over_tokens([&](float y, int k, float q) { return y + __fdividef(lv[k], q); });
          } else {
            over_tokens([](float y, int, float) { return y; });
          }
        } else {
          over_tokens([](float y, int, float) { return y; });
        }
        int n = 2 * K;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          if (n > 1) {
            const bool odd = lane & o;
#pragma unroll
            for (int q = 0; q < n / 2; ++q)
              x[q] = fmaxf(odd ? x[2 * q + 1] : x[2 * q], __shfl_xor_sync(0xffffffffu, odd ? x[2 * q] : x[2 * q + 1], o));
            n /= 2;
          } else {
            x[0] = fmaxf(x[0], __shfl_xor_sync(0xffffffffu, x[0], o));
          }
        }
        const int v = (lane >> 2) & (2 * K - 1);
        if (lane < 8 * K) T.wmax[i & 1][row0 + 8 * (v >> 1) + (v & 1)][quad] = x[0];
      }
      // one barrier a tile: wmax has two buffers
      if (!group_all(1 + wg, ok)) break;
      const bool last = in.last;
#pragma unroll
      for (int g = 0; g < K; ++g) {
        const float4 x = *reinterpret_cast<const float4*>(T.wmax[i & 1][row0 + 8 * g]);
        const float4 y = *reinterpret_cast<const float4*>(T.wmax[i & 1][row0 + 8 * g + 1]);
        const float2 top = mul2(make_float2(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)), fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w))), qf[g]);
        m[g] = make_float2(fmaxf(m[g].x, top.x), fmaxf(m[g].y, top.y));
        const float2 now = make_float2(fmaxf(top.x, m[g].x - kReach), fmaxf(top.y, m[g].y - kReach));
        // rows that have seen no token yet: -inf - 0
        const float2 use = make_float2(now.x == -INFINITY ? 0.0f : now.x, now.y == -INFINITY ? 0.0f : now.y);
        const float2 al = make_float2(ex2(ref[g].x - use.x), ex2(ref[g].y - use.y));
        ref[g] = now;
        const float2 neg = make_float2(-use.x, -use.y);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 e = fma2(s[g][k], qf[g], neg);
          s[g][k] = make_float2(ex2(e.x), ex2(e.y));
        }
        l[g] = fma2(l[g], al, add2(add2(s[g][0], s[g][1]), add2(s[g][2], s[g][3])));
        if (quad == 0 && lane < 4) *reinterpret_cast<float2*>(&T.alpha[i & 3][row0 + 8 * g]) = al;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int tok = tok0 + 8 * k;
        const float2 ratio = both(in.vr[tok >> a.page_log2]);
        uint8_t* p = pbuf + pb * C::kPBytes + tok * 16;
        uint16_t c[K][PP];
#pragma unroll
        for (int g = 0; g < K; ++g) {
          const float2 w = mul2(s[g][k], ratio);
          split2p<PP>(w.x, w.y, c[g]);
        }
#pragma unroll
        for (int t = 0; t < PP; ++t) {
          if constexpr (K == 1) {
            const int n = t * R + row0;
            *reinterpret_cast<uint16_t*>(p + (n >> 4) * 2048 + (n & 15)) = c[0][t];
          } else {
            // the thread's four rows next to each other (row_of)
            *reinterpret_cast<uint32_t*>(p + (t * (R / 16) + wg) * 2048 + 4 * (lane & 3)) =
                (uint32_t)c[0][t] | ((uint32_t)c[1][t] << 16);
          }
        }
      }
      if ((in.mask & 1) && wg == 0) {
        // Values that some row must not see: 0 x NaN would reach its sum.  Rows that no query sees become zero; a NaN
        // in a row that only some see becomes zero too, and is put back for those when the segment ends.
        const int tok = quad * 32 + lane, t = in.t0 + tok;
        dead = !__all_sync(0xffffffffu, wait_quick(&T.v_ready, masked++ & 1, abort_flag));
        if (in.nan && ((in.nan >> (tok >> a.page_log2)) & 1) && t < in.limit) {
          T.nanseen[seg % kSegRing] = 1;
          for (int d = 0; d < NC * 128; ++d) atomicMin(&T.nanmin[seg % kSegRing][d], t);
        }
        for (int c = 0; c < NC && !dead; ++c) {
          uint4* row16 = reinterpret_cast<uint4*>(smem + v_slot(i * NC + c) * kChunk + tok * 128);
          for (int k = 0; k < 8; ++k) {
            // the swizzle has the row's dims 16 k .. 16 k + 15 in this 16-byte unit
            uint4* vr = row16 + (k ^ (tok & 7));
            if (t >= in.limit) {
              *vr = make_uint4(0, 0, 0, 0);
            } else {
              uint4 x = *vr;
              uint32_t* xs = reinterpret_cast<uint32_t*>(&x);
              if (nan_bytes(x.x) | nan_bytes(x.y) | nan_bytes(x.z) | nan_bytes(x.w)) {
                T.nanseen[seg % kSegRing] = 1;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t nb = nan_bytes(xs[e]);
#pragma unroll
                  for (int y = 0; y < 4; ++y)
                    if ((nb >> (8 * y + 7)) & 1) {
                      atomicMin(&T.nanmin[seg % kSegRing][c * 128 + 16 * k + 4 * e + y], t);
                      xs[e] &= ~(0xFFu << (8 * y));
                    }
                }
                *vr = x;
              }
            }
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&T.p_full[pb]);
      if (last) {
#pragma unroll
        for (int g = 0; g < K; ++g) {
          float2 x = l[g];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1)
            x = add2(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)));
          if (lane < 4) {
            *reinterpret_cast<float2*>(&T.lsum[seg % kSegRing][quad][row0 + 8 * g]) = x;
            if (quad == 0) *reinterpret_cast<float2*>(&T.mfin[seg % kSegRing][row0 + 8 * g]) = ref[g];
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&T.l_full[seg % kSegRing]);
      }
    }
  } else {
    // ------------------------------------------------------------ Q in, O out
    if constexpr (kSplitRegs) reg_inc<kAccRegs>();
    const int quad = warp & 3;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    // One warp per row: amax, power-of-two scale, terms, swizzled store.  Lane k works out where the warp's k-th row
    // lies; the loads of RB rows go out together.
    constexpr int RB = R / 4 < 4 ? R / 4 : 4;
    auto stage = [&](const Walk& w, int seg) {
      uint8_t* qb = qbuf + (seg % C::QB) * C::kQBytes;
      const int buf = seg & 1;
      int64_t from = -1;
      if (lane < R / 4) {
        const int r = quad + 4 * lane, rr = w.rt * R + r;
        int lim = 0;
        int64_t off = -1;
        if (rr < a.S * a.G) {
          const int i = rr / a.G, head = w.h * a.G + rr - i * a.G;
          lim = row_limit(w.s, i);
          from = (int64_t)w.b * a.q_sb + (int64_t)i * a.q_ss + (int64_t)head * a.q_sh;
          if (i < w.s.nl) off = (((int64_t)w.b * a.S + i) * a.H + head) * a.D;
        }
        T.lim[buf][r] = lim;
        T.off[buf][r] = off;
      }
#pragma unroll 1
      for (int k0 = 0; k0 < R / 4; k0 += RB) {
        uint2 raw[RB][NC];
#pragma unroll
        for (int k = 0; k < RB; ++k) {
          const int64_t at = __shfl_sync(0xffffffffu, from, k0 + k);
          const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + at + lane * 4;
#pragma unroll
          for (int c = 0; c < NC; ++c)
            raw[k][c] = at >= 0 && c * 128 + lane * 4 < a.D ? *reinterpret_cast<const uint2*>(q + c * 128) : make_uint2(0, 0);
        }
#pragma unroll
        for (int k = 0; k < RB; ++k) {
          const int r = quad + 4 * (k0 + k);
          // amax of 16-bit numbers without their sign, two at a time: integer order is float order, NaN on top
          uint32_t top = 0;
#pragma unroll
          for (int c = 0; c < NC; ++c) top = max_u16x2(top, max_u16x2(raw[k][c].x & 0x7FFF7FFFu, raw[k][c].y & 0x7FFF7FFFu));
          const uint32_t bits = __reduce_max_sync(0xffffffffu, max(top & 0xFFFFu, top >> 16));
          const float amax = PP == 3 ? __half2float(__ushort_as_half((uint16_t)bits)) : __uint_as_float(bits << 16);
          // 2^e with amax * 2^e in [128, 256); zero rows and tiny ones keep to the exponents that exist; a row with
          // infinities or NaN becomes NaN (e4m3 would saturate it)
          int e = 134 - (int)(__float_as_uint(amax) >> 23);
          e = amax == 0.0f ? 0 : min(max(e, -120), 120);
          float up = __uint_as_float((uint32_t)(127 + e) << 23);
          const float down = __uint_as_float((uint32_t)(127 - e) << 23);
          if (!(amax < __uint_as_float(0x7F800000u))) up = __uint_as_float(0x7FC00000u);
          if (a.scale_log2 < 0.0f) up = -up;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            uint16_t t[2][PP];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint32_t u = y ? raw[k][c].y : raw[k][c].x;
              float2 x;
              if (PP == 3) x = __half22float2(*reinterpret_cast<const __half2*>(&u));
              else x = make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
              x = mul2(x, both(up));
              split2h<PP>(x.x, x.y, t[y]);
            }
#pragma unroll
            for (int p = 0; p < PP; ++p) {
              const int n = p * R + r;
              *reinterpret_cast<uint32_t*>(qb + c * N * 128 + n * 128 + ((lane * 4) ^ ((n & 7) << 4))) =
                  (uint32_t)t[0][p] | ((uint32_t)t[1][p] << 16);
            }
          }
          // not zero: a hidden token's -inf times it has to stay -inf
          if (lane == 0) T.qf[buf][r] = fmaxf(down * fabsf(a.scale_log2), 1e-35f);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&T.q_full[seg % C::QB]);
    };
    Walk w = T.start;
    w.left = count;
    if (w.left > 0) stage(w, 0);
    int i = 0;
    bool ok = true;
    for (int seg = 0; w.left > 0 && ok; ++seg) {
      const int t0 = w.t, t1 = w.seg_end(), nt = w.nt;
      w.next(a, R);
      // The next rows' places go where those of the segment before this one were: all four warps are done with them.
      if (seg > 0) group_all(8, true);
      // the other Q buffer: its last products are behind the O tiles taken out before
      if (C::QB == 2 && w.left > 0) stage(w, seg + 1);
      float acc[NC][R];
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[c][r] = 0.0f;
      for (int t = t0; t < t1; ++t, ++i) {
        const int ob = i % C::OB;
        ok = __all_sync(0xffffffffu, wait_quick(&T.o_full[ob], (i / C::OB) & 1, abort_flag));
        if (!ok) break;               // out of the tile loop; the group's barrier below ends the role
        tc_fence_after();
        const float unit = T.info[i % kInfo].unit * (1.0f / 256.0f / kReachScale);
        const float* al = T.alpha[i & 3];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          constexpr int B = R == 64 ? 16 : R;   // rows at a time: the registers of 64 would not fit
#pragma unroll
          for (int b = 0; b < R; b += B) {
            float o[B];
            load_rows<R, PP, B>(tmem + lane_base + C::SB * N + (ob * NC + c) * N + b, o);
#pragma unroll
            for (int r = 0; r < B; r += 2) {
              const float2 x = fma2(make_float2(acc[c][b + r], acc[c][b + r + 1]), *reinterpret_cast<const float2*>(al + row_of<R>(b + r)),
                                    mul2(make_float2(o[r], o[r + 1]), both(unit)));
              acc[c][b + r] = x.x;
              acc[c][b + r + 1] = x.y;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&T.o_empty[ob]);
      }
      if (C::QB == 1 && ok && w.left > 0) stage(w, seg + 1);
      const int sr = seg % kSegRing, buf = seg & 1;
      ok = ok && __all_sync(0xffffffffu, wait_quick(&T.l_full[sr], (seg / kSegRing) & 1, abort_flag));
      const bool whole = t0 == 0 && t1 == nt;
      const int64_t slot = 2 * (int64_t)blockIdx.x + (seg == 0 ? 0 : 1);
      // Row r's factor (1 over its sum), once, by thread r; partial results keep their sum and reference instead.
      const int row = quad * 32 + lane;
      if (ok && row < R) {
        const float lr = T.lsum[sr][0][row] + T.lsum[sr][1][row] + T.lsum[sr][2][row] + T.lsum[sr][3][row];
        const float m = T.mfin[sr][row];
        float f = 1.0f;
        if (!whole) {
          *reinterpret_cast<float2*>(&a.part_ml[(slot * R + row) * 2]) = make_float2(m, lr);
        } else {
          const int64_t at = T.off[buf][row];
          float z = lr;
          if (a.sink && at >= 0) {
            const float sk = a.sink[(at / a.D) % a.H] * 1.4426950408889634f;
            const float M = fmaxf(m, sk);
            f = m == -INFINITY ? 0.0f : exp2f(m - M);
            z = lr * f + (sk == -INFINITY ? 0.0f : exp2f(sk - M));
          }
          f = z == 0.0f ? 0.0f : f / z * kReachScale;
        }
        T.fin[buf][row] = f;
      }
      if (!group_all(8, ok)) break;
      if (T.nanseen[sr]) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int first_nan = T.nanmin[sr][c * 128 + quad * 32 + lane];
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (first_nan < T.lim[buf][row_of<R>(r)]) acc[c][r] = __uint_as_float(0x7FC00000u);
          T.nanmin[sr][c * 128 + quad * 32 + lane] = 0x7FFFFFFF;
        }
      }
      // Shared memory is read by its 32-bit address here: loads through T are generic ones, which wait for the global
      // stores before them (1000 cycles a row, 60000 at the end of a segment of 64 rows).
      const uint32_t fin = smem_u32(&T.fin[buf][0]), off = smem_u32(&T.off[buf][0]);
      const int d0 = quad * 32 + lane;
      if (whole) {
        uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + d0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int64_t at = lds_s64(off + 8 * row_of<R>(r));
          const float f = lds_f32(fin + 4 * row_of<R>(r));
          if (at < 0) continue;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            if (c * 128 + d0 < a.D) {
              const float x = acc[c][r] * f;
              out[at + c * 128] = PP == 3 ? __half_as_ushort(__float2half_rn(x)) : __bfloat16_as_ushort(__float2bfloat16_rn(x));
            }
          }
        }
      } else {
        float* po = a.part_o + slot * (R * NC * 128) + d0;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int c = 0; c < NC; ++c) po[row_of<R>(r) * (NC * 128) + c * 128] = acc[c][r];
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmem);
  }
}

// Joins the partial results of heads that several CTAs share, and writes zeros for rows that see nothing (empty
// sequences, padded query tokens).  A row is one warp's, or with SPLIT (few rows) a CTA's, whose warps then share the
// partial results.  A lane weighs one partial result and holds four dims of each chunk.
template <typename T, int NC, bool SPLIT>
__global__ void __launch_bounds__(256) merge_kernel(const Args a, int R, int rows) {
  __shared__ float4 part_acc[SPLIT ? 8 : 1][SPLIT ? NC * 32 : 1];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = a.plan[0], cost = a.seg_cost;
  for (int id = SPLIT ? blockIdx.x : blockIdx.x * 8 + warp; id < rows; id += gridDim.x * (SPLIT ? 1 : 8)) {
    const int item = id / R, r = id - item * R;
    const int unit = item / a.Hkv, h = item - unit * a.Hkv;
    const int start = a.plan[1 + unit];
    const int b = unit / a.RT, rt = unit - b * a.RT;
    const int rr = rt * R + r;
    if (rr >= a.S * a.G) continue;
    const int i = rr / a.G, g = rr - i * a.G;
    const Seq s = load_seq(a, b, false);
    const int nt = tiles_of(tile_limit(a, s, rt, R));
    T* out = reinterpret_cast<T*>(a.out) + (((int64_t)b * a.S + i) * a.H + h * a.G + g) * a.D;
    const bool empty = row_limit(s, i) == 0;
    const int place = start + h * (nt + cost), first = place + cost;
    const int c0 = empty ? 0 : first / per, c1 = empty ? 0 : (first + nt - 1) / per;
    if (!empty && c0 == c1) continue;            // one CTA had it all
    float4 acc[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (!empty) {
      // a CTA's first segment is in its slot 0, its last one in slot 1
      auto part = [&](int c) { return (int64_t)(2 * c + (c * per >= place ? 0 : 1)) * R + r; };
      const float sk = a.sink ? a.sink[h * a.G + g] * 1.4426950408889634f : -INFINITY;
      float M = sk, z = 0.0f;
      for (int c = c0 + lane; c <= c1; c += 32) {   // this lane's running maximum and sum
        const float2 ml = *reinterpret_cast<const float2*>(&a.part_ml[part(c) * 2]);
        const float m = fmaxf(M, ml.x);
        if (m != -INFINITY) z = z * exp2f(M - m) + ml.y * exp2f(ml.x - m);
        M = m;
      }
      float top = M;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float use = top == -INFINITY ? 0.0f : top;
      z *= exp2f(M - use);                       // no part: 0 x exp2(-inf) = 0
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      if (sk != -INFINITY) z += exp2f(sk - use);
      const float f = z == 0.0f ? 0.0f : kReachScale / z;
      constexpr int step = SPLIT ? 8 : 1;
      for (int cb = c0 + (SPLIT ? warp : 0); cb <= c1; cb += 32 * step) {
        const int n = min(32, (c1 - cb) / step + 1);
        float w = 0.0f;
        if (lane < n) w = exp2f(a.part_ml[part(cb + lane * step) * 2] - use) * f;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
          const float wj = __shfl_sync(0xffffffffu, w, j);
          const float4* po = reinterpret_cast<const float4*>(a.part_o + part(cb + j * step) * (NC * 128)) + lane;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const float4 v = po[c * 32];
            acc[c].x = fmaf(v.x, wj, acc[c].x);
            acc[c].y = fmaf(v.y, wj, acc[c].y);
            acc[c].z = fmaf(v.z, wj, acc[c].z);
            acc[c].w = fmaf(v.w, wj, acc[c].w);
          }
        }
      }
    }
    auto put = [&](int d, float4 x) {
      if (d < a.D) {
        T v[4] = {bs_from_f32<T>(x.x), bs_from_f32<T>(x.y), bs_from_f32<T>(x.z), bs_from_f32<T>(x.w)};
        *reinterpret_cast<uint2*>(out + d) = *reinterpret_cast<const uint2*>(v);
      }
    };
    if constexpr (SPLIT) {
#pragma unroll
      for (int c = 0; c < NC; ++c) part_acc[warp][c * 32 + lane] = acc[c];
      __syncthreads();                           // a row's course is the same for all threads
      if ((int)threadIdx.x < NC * 32) {
        float4 x = part_acc[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < 8; ++k) {
          const float4 y = part_acc[k][threadIdx.x];
          x.x += y.x;
          x.y += y.y;
          x.z += y.z;
          x.w += y.w;
        }
        put(threadIdx.x * 4, x);
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) put(c * 128 + lane * 4, acc[c]);
    }
  }
}

bool make_map(CUtensorMap* m, const void* cache, int64_t D, int64_t page, int64_t rows) {
  auto enc = moe::encode_fn();
  if (!enc) return false;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)page, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)D, (cuuint64_t)(D * page)};
  cuuint32_t box[3] = {128u, (cuuint32_t)page, 1u};          // dims past D are filled with zeros
  cuuint32_t estr[3] = {1u, 1u, 1u};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(cache), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Largest row tile: what TMEM, registers and shared memory carry.
__host__ __device__ constexpr int most_rows(int PP, int NC) {
  return NC == 1 ? (PP == 3 ? 32 : 64) : NC == 2 ? 32 : (PP == 3 ? 16 : 32);
}
// Rows of a tile: the smallest R that holds a kv head's rows, up to that.
int rows_per_tile(int64_t rows, int NC, int f16) {
  const int most = most_rows(f16 ? 3 : 2, NC);
  int R = 8;
  while (R < most && R < rows) R *= 2;
  return R;
}

int sm_count() {
  static int slots[hostcache::kMaxDevices];
  const int n = hostcache::device_attr(slots, cudaDevAttrMultiProcessorCount);
  return n > 0 ? n : 148;
}

struct Layout {
  int R, NC, RT, grid;
  size_t plan, ml, o, total;
};
Layout layout(int64_t B, int64_t S, int H, int Hkv, int D, int f16) {
  Layout l;
  l.NC = (D + 127) / 128;
  const int64_t rows = S * (H / Hkv);
  l.R = rows_per_tile(rows, l.NC, f16);
  l.RT = (int)((rows + l.R - 1) / l.R);
  l.grid = sm_count() * (l.NC == 1 && l.R <= 16 ? 2 : 1);
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  l.plan = up((1 + (size_t)B * l.RT) * 4);
  l.ml = up((size_t)2 * l.grid * l.R * 2 * 4);
  l.o = (size_t)2 * l.grid * l.R * l.NC * 128 * 4;
  l.total = l.plan + l.ml + l.o;
  return l;
}

template <int R, int PP, int NC>
cudaError_t launch(const CUtensorMap& mk, const CUtensorMap& mv, Args& a, int grid, cudaStream_t st) {
  using C = Cfg<R, PP, NC>;
  a.seg_cost = C::kSegCost;
  auto kern = cache_attn_kernel<R, PP, NC>;
  static int done[hostcache::kMaxDevices];
  cudaError_t e = (cudaError_t)hostcache::get(done, [&] {
    return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, mk, mv, a);
}

template <int PP, int NC>
cudaError_t launch_r(int R, const CUtensorMap& mk, const CUtensorMap& mv, Args& a, int grid, cudaStream_t st) {
  if (R == 8) return launch<8, PP, NC>(mk, mv, a, grid, st);
  if (R == 16) return launch<16, PP, NC>(mk, mv, a, grid, st);
  if constexpr (most_rows(PP, NC) >= 32)
    if (R == 32) return launch<32, PP, NC>(mk, mv, a, grid, st);
  if constexpr (most_rows(PP, NC) >= 64)
    if (R == 64) return launch<64, PP, NC>(mk, mv, a, grid, st);
  return cudaErrorInvalidConfiguration;
}

}  // namespace cattn

size_t bs_cache_attn_ws(int64_t B, int64_t S, int H, int Hkv, int D, int f16) {
  return cattn::layout(B, S, H, Hkv, D, f16).total;
}

// 0 ok, BS_ERR_UNSUPPORTED (descriptor), or a CUDA error in *cerr
int bs_launch_cache_attn(cattn::Args a, const void* k_cache, const void* v_cache, int f16, void* ws, cudaStream_t st,
                         cudaError_t* cerr) {
  *cerr = cudaSuccess;
  const cattn::Layout l = cattn::layout(a.B, a.S, a.H, a.Hkv, a.D, f16);
  // tiles and rows are counted in 32 bits
  const int64_t most = (((int64_t)a.max_pages << a.page_log2) + 127) / 128 + 8;
  if ((int64_t)a.B * l.RT * a.Hkv > 0x7fffffff / (most > l.R ? most : l.R) - 1024) return BS_ERR_UNSUPPORTED;
  a.RT = l.RT;
  a.plan = (int*)ws;
  a.part_ml = (float*)((char*)ws + l.plan);
  a.part_o = (float*)((char*)ws + l.plan + l.ml);
  const int64_t page = (int64_t)1 << a.page_log2;
  CUtensorMap mk, mv;
  if (!cattn::make_map(&mk, k_cache, a.D, page, (int64_t)a.n_pages * a.Hkv)) return BS_ERR_UNSUPPORTED;
  if (!cattn::make_map(&mv, a.shared ? k_cache : v_cache, a.D, page, (int64_t)a.n_pages * a.Hkv)) return BS_ERR_UNSUPPORTED;
  cudaError_t e;
  if (f16)
    e = l.NC == 1 ? cattn::launch_r<3, 1>(l.R, mk, mv, a, l.grid, st) : l.NC == 2 ? cattn::launch_r<3, 2>(l.R, mk, mv, a, l.grid, st)
      : l.NC == 3 ? cattn::launch_r<3, 3>(l.R, mk, mv, a, l.grid, st) : cattn::launch_r<3, 4>(l.R, mk, mv, a, l.grid, st);
  else
    e = l.NC == 1 ? cattn::launch_r<2, 1>(l.R, mk, mv, a, l.grid, st) : l.NC == 2 ? cattn::launch_r<2, 2>(l.R, mk, mv, a, l.grid, st)
      : l.NC == 3 ? cattn::launch_r<2, 3>(l.R, mk, mv, a, l.grid, st) : cattn::launch_r<2, 4>(l.R, mk, mv, a, l.grid, st);
  if (e != cudaSuccess) {
    *cerr = e;
    return BS_ERR_CUDA;
  }
  const int64_t rows = (int64_t)a.B * a.RT * a.Hkv * l.R;
  cudaLaunchConfig_t cfg = {};
  const bool split = rows <= 4 * 148;        // few rows: a CTA each
  const int64_t want = split ? rows : (rows + 7) / 8;
  cfg.gridDim = dim3((unsigned)(want < 148 * 8 ? want : 148 * 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto merge_n = [&](auto t, auto nc) {
    using T = decltype(t);
    constexpr int NC = decltype(nc)::value;
    return split ? cudaLaunchKernelEx(&cfg, cattn::merge_kernel<T, NC, true>, a, l.R, (int)rows)
                 : cudaLaunchKernelEx(&cfg, cattn::merge_kernel<T, NC, false>, a, l.R, (int)rows);
  };
  auto merge = [&](auto t) {
    return l.NC == 1   ? merge_n(t, std::integral_constant<int, 1>())
           : l.NC == 2 ? merge_n(t, std::integral_constant<int, 2>())
           : l.NC == 3 ? merge_n(t, std::integral_constant<int, 3>())
                       : merge_n(t, std::integral_constant<int, 4>());
  };
  e = f16 ? merge(__half()) : merge(__nv_bfloat16());
  *cerr = e;
  return e == cudaSuccess ? 0 : BS_ERR_CUDA;
}
