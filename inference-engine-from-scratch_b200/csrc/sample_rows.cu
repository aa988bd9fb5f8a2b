// Draws from given random numbers: temperature, top-k, top-p and min-p over rows of logits.
//
// With m = max x and w_i = exp((x_i - m) / T), the kept tokens are the first n of the descending
// order (equal logits: lowest id first), n the least of
//   top-k:  k;
//   top-p:  the tokens whose mass before them is below top_p times the mass of the top-k tokens;
//   min-p:  the tokens with w_i >= min_p (the largest weight is 1);
// and at least 1. The token is the first kept id, in ascending order, whose prefix mass exceeds
// u times the kept mass.
//
// A row is a cluster of CTAs, each with a slice of the row in shared memory, so the logits are read
// from memory once. Cuts are found by a radix select over ordered integer keys (larger key = larger
// logit), 1024 bins a pass, counts and masses added over the cluster; a vector of 16 bytes whose
// largest logit is below the search is passed over. A border is
// decided by sums over the whole vocabulary, so weights are good to about 2e-9 (an error of 1e-7, as
// plain fp32 gives, moves the border of a flat distribution past a token) and summed in steps of 2^-45,
// whose sums do not depend on their order: the same inputs give the same tokens.
//
// Where a lower bound of all cuts (from the quarter warps' maxima, or min-p) leaves at most 2,048 tokens,
// they are gathered and sorted by one CTA; else the cuts are selected over the row. Bound by instructions and
// their latency (2 of 4 issue slots used), not by the 97 MB: 320 rows of 151,936 bf16 logits, replayed with the
// logits in L2, take 41 us greedy, 72 to 92 with top-k or min-p, 135 without a filter, 270 with top-p 0.9 at
// temperature 0.8 and 670 with top-p 0.999 at 1.5 (every third token a candidate), 176 with all of these mixed
// (176 to 188 as calls, by the inputs); one row 14 to 73. With 64 registers, for two CTAs an SM, ptxas spills 180 bytes stored
// and 392 loaded (bf16; fp32 20 and 80).
#include <cooperative_groups.h>

#include "sampling.cuh"

namespace ne {

namespace {

namespace cg = cooperative_groups;

constexpr int RT = 512;               // threads per CTA
constexpr int RW = RT / 32;
constexpr int BINS = 1024;
constexpr int MOST = 2048;            // tokens of a list
constexpr int BANDS = 12;
constexpr int MOST_CHUNKS = 18;       // (MAX_SLICE_BYTES over 16 warps of 32 vectors)
constexpr int MAX_CLUSTER = 8;
constexpr unsigned ALL = 0xFFFFFFFFu;
// 2^(31 + i / 64), rounded
__device__ const uint32_t POW2[64] = {
    2147483648u, 2170868212u, 2194507417u, 2218404036u, 2242560872u, 2266980759u, 2291666561u, 2316621173u,
    2341847524u, 2367348571u, 2393127307u, 2419186755u, 2445529972u, 2472160047u, 2499080105u, 2526293303u,
    2553802834u, 2581611923u, 2609723834u, 2638141863u, 2666869345u, 2695909648u, 2725266179u, 2754942382u,
    2784941738u, 2815267765u, 2845924021u, 2876914102u, 2908241642u, 2939910317u, 2971923842u, 3004285971u,
    3037000500u, 3070071267u, 3103502151u, 3137297074u, 3171459999u, 3205994934u, 3240905930u, 3276197082u,
    3311872529u, 3347936457u, 3384393094u, 3421246719u, 3458501653u, 3496162267u, 3534232978u, 3572718252u,
    3611622603u, 3650950594u, 3690706840u, 3730896002u, 3771522796u, 3812591987u, 3854108391u, 3896076880u,
    3938502376u, 3981389855u, 4024744348u, 4068570940u, 4112874773u, 4157661043u, 4202935003u, 4248701965u};
constexpr double FIX = 35184372088832.0;          // 2^45
constexpr unsigned long long ONE = 1ull << 45;    // a weight of 1
constexpr int MAX_VOCAB = 1 << 18;        // 262,144 weights of at most 1 sum to at most 2^63
constexpr size_t MAX_SLICE_BYTES = 132 << 10;  // MAX_VOCAB / MAX_CLUSTER tokens in fp32, and a padded vector
static_assert((MAX_SLICE_BYTES / 16 + RW - 1) / RW <= 32 * MOST_CHUNKS, "a warp's chunks");
constexpr size_t MID_SLICE_BYTES = 80 << 10;  // largest slice of clusters below the largest (launch_sample_rows)
constexpr int MOST_SLICE = MID_SLICE_BYTES / 2 > MAX_VOCAB / MAX_CLUSTER ? MID_SLICE_BYTES / 2 : MAX_VOCAB / MAX_CLUSTER;
static_assert((unsigned long long)MOST_SLICE << 15 <= 0xFFFFFFFFull, "pieces of a bin");

// Ordered key of a logit, in the low bits: 16 for bf16, 32 for fp32. NaN and -inf: never drawn.
// A vector is 16 bytes of a row; ``top`` is its largest logit (NaN aside).
template <typename T>
struct Keys;
template <>
struct Keys<__nv_bfloat16> {
  static constexpr int PER = 8;
  static constexpr uint32_t NONE = 0x007Fu;  // the key of -inf; keys up to it hold no token
  static __device__ __forceinline__ uint32_t key(uint32_t b) {
    if ((b & 0x7FFFu) > 0x7F80u) return 0u;  // NaN
    if (b == 0x8000u) b = 0u;                // -0 equals 0
    return (b & 0x8000u) ? (~b & 0xFFFFu) : (b | 0x8000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    const uint32_t b = (k & 0x8000u) ? (k & 0x7FFFu) : (~k & 0xFFFFu);
    return __uint_as_float(b << 16);
  }
  static __device__ __forceinline__ uint32_t key_of(float x) { return key(__float_as_uint(x) >> 16); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float top(const uint4& v) {
    const uint32_t m = max2(max2(v.x, v.y), max2(v.z, v.w));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t at(const uint4& v, int j) {  // (j a constant)
    const uint32_t w = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
    return key(j & 1 ? w >> 16 : w & 0xFFFFu);
  }
  static __device__ __forceinline__ float logit(const uint4& v, int j) {
    const uint32_t w = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
    return __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16);
  }
  static constexpr uint16_t PAD = 0xFF80u;  // -inf
  using Raw = uint16_t;
};
template <>
struct Keys<float> {
  static constexpr int PER = 4;
  static constexpr uint32_t NONE = 0x007FFFFFu;
  static __device__ __forceinline__ uint32_t key(uint32_t b) {
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
    if (b == 0x80000000u) b = 0u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
  }
  static __device__ __forceinline__ uint32_t key_of(float x) { return key(__float_as_uint(x)); }
  static __device__ __forceinline__ float top(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ uint32_t at(const uint4& v, int j) {
    return key(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ float logit(const uint4& v, int j) {
    return __uint_as_float(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w);
  }
  static constexpr uint32_t PAD = 0xFF800000u;
  using Raw = uint32_t;
};

// Fixed-point masses of a bin in three 15-bit pieces (the upper one up to 2^15): those of a CTA's 40,960
// tokens at most add up in 32 bits each, by the 32-bit shared-memory atomics (a 64-bit one took a pass from 15 to 90 us a row).
struct Bins {
  uint32_t count[BINS], piece[3][BINS];
};
// The tokens at or above a lower bound of all cuts, where they are few: gathered into the first CTA.
struct List {
  unsigned long long entry[MOST], mass[MOST];
};
// (The slice lies behind it: begun 16 bytes past a 32-byte boundary, 320 rows of 151,936 take 4 us more.)
struct alignas(128) Shared {
  union {
    Bins bins[2];
    List list;
    float column[BANDS][RT];  // a thread's sums of the weights in (4^-(b + 1), 4^-b]
  };
  unsigned long long chunk[RW][MOST_CHUNKS];  // kept mass of a warp's part, 32 vectors at a time
  unsigned long long red64[RW];
  uint32_t red32[RW];
  uint2 pow2[64];  // 2^(31 + i / 64) in 32 bits (2^32 - 1 at most), and an eighth of it as a float
  // published to the cluster
  unsigned long long pub_sum[3], pub_above;
  float pub_band[BANDS];
  uint32_t pub_best, pub_low, pub_ties, pub_listed, bound;
  uint32_t pub_tops[4 * RW];               // the largest key of each quarter warp
  alignas(16) uint32_t tops[4 * RW * MAX_CLUSTER];  // (the cluster's)
  int pub_id;
  // the bin a select pass chose
  int sel_bin;
  uint32_t sel_count;
  unsigned long long sel_mass;
};

// A cut of the descending order: tokens with a key above ``key``, and the first ``keep`` (by id) of
// the ``ties`` tokens that have it.
struct Cut {
  uint32_t key, keep, ties;
};

// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  return (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// (0 for 64 places and more, which C++ leaves open)
__device__ __forceinline__ unsigned long long shift_right(unsigned long long v, int by) {
  unsigned long long d;
  asm("shr.u64 %0, %1, %2;" : "=l"(d) : "l"(v), "r"(by));
  return d;
}

template <typename T>
struct Row {
  const uint4* vecs;   // this CTA's slice: vector v holds tokens PER v .. of it, padded with -inf
  int count;           // its vectors
  uint32_t top;        // the row's largest key
  bool inf;            // it alone has a weight
  bool careful;        // (a temperature so high that masked logits have to be told apart by their keys)
  float least;         // a logit whose weight is 2^-59 or less
  float scale, minus;  // 1, or what keeps differences and c1 in range; minus the largest logit times it
  float c1, c2;        // log2(e) / (temperature x scale) = c1 + c2
  const uint2* pow2;

  // exp((x - m) / T) in steps of 2^-45: 2^t, t = (x - m) log2(e) / T = n / 64 + r, |r| <= 1/128, as the
  // table's 2^(n / 64) times the series of 2^r to the fourth power. On the FMA and integer pipes: the
  // difference and its product with c are taken with their rounding errors, so that t is off by less than
  // 2^-30 whatever the largest logit; the weight by about 2e-9 of itself, each logit's differently.
  // (The same in fp64 took a pass over a row from 6 to 25 us.) A logit below ``least``, -inf or NaN
  // weighs 2^-59 or less, which is 0.
  __device__ __forceinline__ void power2(float logit_a, float logit_b, unsigned long long& wa, unsigned long long& wb,
                                         int* band = nullptr, float* approx = nullptr) const {
    constexpr uint64_t MINUS = 0xBF800000BF800000ull;         // (-1, -1): a - b as fma(b, -1, a), one rounding
    const uint64_t x = pair(fmaxf(logit_a, least), fmaxf(logit_b, least)), c = pair(c1, c1), m2 = pair(minus, minus);
    const uint64_t s = fma2(x, pair(scale, scale), m2), z = fma2(x, pair(-scale, -scale), s);  // x - m = s + err
    const uint64_t err = add2(fma2(x, pair(scale, scale), fma2(s, MINUS, z)), fma2(z, MINUS, m2));
    const uint64_t p = mul2(s, c), e = fma2(s, c, mul2(p, MINUS));  // s c1 = p + e
    const uint64_t low = fma2(err, c, fma2(s, pair(c2, c2), e));
    constexpr float MAGIC = 196608.f;                         // 1.5 x 2^17: p rounded to 1 / 64
    const uint64_t u = add2(p, pair(MAGIC, MAGIC));
    const uint64_t r = add2(fma2(add2(u, pair(-MAGIC, -MAGIC)), MINUS, p), low);
    uint64_t y = fma2(r, pair(0.009618129f, 0.009618129f), pair(0.05550411f, 0.05550411f));
    y = fma2(y, r, pair(0.24022651f, 0.24022651f));
    y = mul2(fma2(y, r, pair(0.69314718f, 0.69314718f)), r);  // 2^r - 1
    const int na = (int)(uint32_t)u - 0x48400000, nb = (int)(uint32_t)(u >> 32) - 0x48400000;
    const uint2 ta = pow2[na & 63], tb = pow2[nb & 63];       // 2^(31 + n / 64), and an eighth as a float
    const uint64_t t8 = (uint64_t)ta.y | (uint64_t)tb.y << 32;
    // (|y| < 0.0055: the product is below 2^22, where 1.5 x 2^23 rounds it to an integer)
    const uint64_t i = fma2(y, t8, pair(12582912.f, 12582912.f));
    const uint32_t va = ta.x + ((uint32_t)i - 0x4B400000u) * 8u, vb = tb.x + ((uint32_t)(i >> 32) - 0x4B400000u) * 8u;
    wa = shift_right((unsigned long long)va << 14, -(na >> 6));
    wb = shift_right((unsigned long long)vb << 14, -(nb >> 6));
    if (band) {  // for a coarse sum by weight: the band of 4^-b, and the weight times 2^28 in fp32
      const uint64_t f = fma2(y, t8, t8);
      band[0] = min(-na >> 7, BANDS - 1);
      band[1] = min(-nb >> 7, BANDS - 1);
      approx[0] = __int_as_float((int)(uint32_t)f + (na >> 6) * (1 << 23));
      approx[1] = __int_as_float((int)(uint32_t)(f >> 32) + (nb >> 6) * (1 << 23));
    }
  }
  __device__ __forceinline__ unsigned long long power(float logit) const {
    unsigned long long a, b;
    power2(logit, logit, a, b);
    return a;
  }
  // (an infinite largest logit: all for it, nothing for the rest)
  __device__ __forceinline__ unsigned long long fixed(uint32_t k) const {
    if (inf) return k == top ? ONE : 0ull;
    return k <= Keys<T>::NONE ? 0ull : power(Keys<T>::value(k));
  }
  // the masses of a vector's tokens, side by side
  __device__ __forceinline__ void masses(const uint4& v, unsigned long long (&w)[Keys<T>::PER]) const {
    if (careful) {
#pragma unroll
      for (int j = 0; j < Keys<T>::PER; ++j) w[j] = fixed(Keys<T>::at(v, j));
    } else {
#pragma unroll
      for (int j = 0; j < Keys<T>::PER; j += 2) power2(Keys<T>::logit(v, j), Keys<T>::logit(v, j + 1), w[j], w[j + 1]);
    }
  }
  __device__ __forceinline__ unsigned long long vector_mass(const uint4& v) const {
    unsigned long long w[Keys<T>::PER], sum = 0;
    masses(v, w);
#pragma unroll
    for (int j = 0; j < Keys<T>::PER; ++j) sum += w[j];
    return sum;
  }

  // f(token of the slice, key) for every token with a key of at least ``lo`` (above NONE)
  template <typename F>
  __device__ __forceinline__ void above(uint32_t lo, F&& f) const {
    const float least = Keys<T>::value(lo);
    for (int v = threadIdx.x; v < count; v += RT) {
      const uint4 x = vecs[v];
      if (!(Keys<T>::top(x) >= least)) continue;
#pragma unroll
      for (int j = 0; j < Keys<T>::PER; ++j) {
        const uint32_t k = Keys<T>::at(x, j);
        if (k >= lo) f(v * Keys<T>::PER + j, k);
      }
    }
  }
};

__device__ __forceinline__ unsigned long long warp_add(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
  return v;
}

// Sum over the CTA, then over the cluster; every thread of the cluster gets it.
// Each call of a row has a place of its own (``turn``), so that none is set while another CTA reads it.
__device__ unsigned long long cluster_sum(cg::cluster_group& cl, Shared& sh, unsigned long long v, int turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_add(v);
  if (lane == 0) sh.red64[warp] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned long long t = 0;
    for (int w = 0; w < RW; ++w) t += sh.red64[w];
    sh.pub_sum[turn] = t;
  }
  cl.sync();
  unsigned long long total = 0;
  for (unsigned r = 0; r < cl.num_blocks(); ++r) total += *cl.map_shared_rank(&sh.pub_sum[turn], r);
  return total;
}

// The cut at which the tokens with larger keys, and some of the ties, first reach ``limit``: a count
// (MASS false) or a mass in fixed point. It is looked for in [lo, hi] (a mass above hi is added up);
// with no ties it is not there. At the bottom of all cuts (``last``) it is the lowest key present
// where the limit is not reached.
template <typename T, bool MASS>
__device__ Cut select_cut(cg::cluster_group& cl, Shared& sh, const Row<T>& row, uint32_t lo, uint32_t hi,
                          unsigned long long limit, bool last = true) {
  unsigned long long above = 0;
  bool first = true;
  // The first pass of masses cuts a wide range evenly by the logits: keys are even by their logarithm,
  // and put most of a row into a few bins around the bulk, whose atomics then queue (58,000 cycles a
  // pass). Later passes take the tokens of the chosen ``slot`` by the same arithmetic.
  const float x_hi = Keys<T>::value(hi), x_lo = Keys<T>::value(lo);
  const float per = (float)BINS / (x_hi - x_lo);
  const bool even = MASS && hi - lo >= BINS && per > 0.f && per < 1e30f;
  auto slot_of = [&](uint32_t k) -> int {
    return BINS - 1 - min(BINS - 1, (int)((x_hi - Keys<T>::value(k)) * per));
  };
  int slot = -1;
  int buf = 0;
  uint32_t ties = 0;
  for (;;) {
    const uint32_t range = hi - lo;
    const int shift = max(0, 32 - __clz(range) - 10);
    Bins& bins = sh.bins[buf];
    for (int i = threadIdx.x; i < BINS; i += RT) {
      bins.count[i] = 0u;
      if (MASS) bins.piece[0][i] = bins.piece[1][i] = bins.piece[2][i] = 0u;
    }
    __syncthreads();
    // (a bin of one key needs no masses: they are its count times the key's)
    const bool start = MASS && first, pieces = MASS && shift > 0;
    unsigned long long outer = 0;
    const uint32_t least = max(lo, Keys<T>::NONE + 1u);
    const float least_value = Keys<T>::value(least), hi_value = Keys<T>::value(hi);
    for (int v = threadIdx.x; v < row.count; v += RT) {
      const uint4 x = row.vecs[v];
      const float t = Keys<T>::top(x);
      if (!(t >= least_value)) continue;
      unsigned long long f[Keys<T>::PER];
      if (pieces || (start && t > hi_value)) row.masses(x, f);  // (side by side: one at a time, behind each
#pragma unroll                                                  // test, took three times as long)
      for (int j = 0; j < Keys<T>::PER; ++j) {
        const uint32_t k = Keys<T>::at(x, j);
        if (k < least) continue;
        if (k > hi) {
          if (start) outer += f[j];
          continue;
        }
        if (slot >= 0 && slot_of(k) != slot) continue;
        const uint32_t b = even && first ? (uint32_t)slot_of(k) : (k - lo) >> shift;
        atomicAdd(&bins.count[b], 1u);
        if (pieces) {
          atomicAdd(&bins.piece[0][b], (uint32_t)f[j] & 0x7FFFu);
          atomicAdd(&bins.piece[1][b], (uint32_t)(f[j] >> 15) & 0x7FFFu);
          atomicAdd(&bins.piece[2][b], (uint32_t)(f[j] >> 30));
        }
      }
    }
    if (start) {
      outer = warp_add(outer);
      if ((threadIdx.x & 31) == 0) sh.red64[threadIdx.x >> 5] = outer;
      __syncthreads();
      if (threadIdx.x == 0) {
        unsigned long long t = 0;
        for (int x = 0; x < RW; ++x) t += sh.red64[x];
        sh.pub_above = t;
      }
    }
    cl.sync();
    // every CTA adds the cluster's bins: thread t owns bins 2 t and 2 t + 1
    uint32_t c[2] = {0u, 0u};
    unsigned long long w[2] = {0ull, 0ull};
#pragma unroll 4
    for (unsigned r = 0; r < cl.num_blocks(); ++r) {
      const Bins* remote = cl.map_shared_rank(&bins, r);
      const uint2 rc = reinterpret_cast<const uint2*>(remote->count)[threadIdx.x];
      c[0] += rc.x;
      c[1] += rc.y;
      if (start) above += *cl.map_shared_rank(&sh.pub_above, r);
      if (pieces) {
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          const uint2 rp = reinterpret_cast<const uint2*>(remote->piece[q])[threadIdx.x];
          w[0] += (unsigned long long)rp.x << (15 * q);
          w[1] += (unsigned long long)rp.y << (15 * q);
        }
      }
    }
    if (MASS && !pieces) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (c[j]) w[j] = c[j] * row.fixed(lo + 2 * threadIdx.x + j);
    }
    const unsigned long long v[2] = {MASS ? w[0] : c[0], MASS ? w[1] : c[1]};
    // mass (or count) of the bins above this thread's: an exclusive suffix sum
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long incl = v[0] + v[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long t = __shfl_down_sync(ALL, incl, o);
      if (lane + o < 32) incl += t;
    }
    if (lane == 0) sh.red64[warp] = incl;
    if (threadIdx.x == 0) sh.sel_bin = -1;
    __syncthreads();
    unsigned long long before = above + incl - (v[0] + v[1]);
    unsigned long long all = 0;
    for (int x = 0; x < RW; ++x) {
      const unsigned long long t = sh.red64[x];
      if (x > warp) before += t;
      all += t;
    }
    if (start && !last && above + all < limit) return Cut{lo, 0u, 0u};
    // the lowest non-empty bin whose tokens start below the limit: each thread offers its own
    int mine = -1;
    unsigned long long mine_before = 0;
    const unsigned long long before_lo = before + v[1];
    if (c[0] && before_lo < limit) {
      mine = 2 * threadIdx.x;
      mine_before = before_lo;
    } else if (c[1] && before < limit) {
      mine = 2 * threadIdx.x + 1;
      mine_before = before;
    }
    // the lowest offered bin: bins are ascending in thread order
    uint32_t low = mine >= 0 ? (uint32_t)mine : 0xFFFFFFFFu;
    low = __reduce_min_sync(ALL, low);
    if (lane == 0) sh.red32[warp] = low;
    __syncthreads();
    uint32_t best = 0xFFFFFFFFu;
    for (int x = 0; x < RW; ++x) best = min(best, sh.red32[x]);
    if (mine >= 0 && (uint32_t)mine == best) {
      sh.sel_bin = mine;
      sh.sel_mass = mine_before;
      sh.sel_count = c[mine & 1];
    }
    __syncthreads();
    const int bin = sh.sel_bin;
    if (bin < 0) return Cut{lo, 0u, 0u};  // (the limit lies above hi)
    above = sh.sel_mass;
    ties = sh.sel_count;
    if (even && first) {
      // keys that the slot's tokens lie between, with a margin for the slots' arithmetic
      slot = bin;
      const float d = (float)(BINS - 1 - bin);
      const uint32_t a = Keys<T>::key_of(x_hi - (d + 1.01f) / per), z = Keys<T>::key_of(x_hi - (d - 0.01f) / per);
      lo = max(lo, a > 0u ? a - 1u : 0u);
      hi = max(lo, min(hi, z + 1u));
      first = false;
      buf ^= 1;
      continue;
    }
    const uint32_t nlo = lo + ((uint32_t)bin << shift);
    const uint32_t last = nlo + ((1u << shift) - 1u);
    hi = last < nlo ? hi : min(hi, last);
    lo = nlo;
    first = false;
    buf ^= 1;  // (the other CTAs may still read this buffer)
    if (shift == 0) break;
  }
  Cut cut{lo, ties, ties};
  if (!MASS) {
    cut.keep = (uint32_t)min((unsigned long long)ties, limit - above);
  } else {
    const unsigned long long w = row.fixed(lo);
    // tie j starts at above + j w and is kept while that is below the limit
    if (w > 0ull) cut.keep = (uint32_t)min((unsigned long long)ties, (limit - above - 1ull) / w + 1ull);
  }
  return cut;
}

// Ascending (UP) or descending bitonic sort of the first ``size`` (a power of two) entries, by the CTA.
template <bool UP>
__device__ void sort_entries(unsigned long long* e, int size) {
  if (size <= 64) {  // a pair a lane
    if (threadIdx.x < 32) {
      const int i = threadIdx.x;
      for (int width = 2; width <= size; width *= 2) {
        for (int stride = width / 2; stride > 0; stride /= 2) {
          const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
          const unsigned long long a = i < size / 2 ? e[lo] : 0ull, b = i < size / 2 ? e[hi] : 0ull;
          if (i < size / 2 && (a > b) == (((lo & width) == 0) == UP)) {
            e[lo] = b;
            e[hi] = a;
          }
          __syncwarp();
        }
      }
    }
    __syncthreads();
    return;
  }
  for (int width = 2; width <= size; width *= 2) {
    for (int stride = width / 2; stride > 0; stride /= 2) {
      for (int i = threadIdx.x; i < size / 2; i += RT) {
        const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const unsigned long long a = e[lo], b = e[hi];
        if ((a > b) == (((lo & width) == 0) == UP)) {
          e[lo] = b;
          e[hi] = a;
        }
      }
      __syncthreads();
    }
  }
}

// Inclusive prefix sums of f(0), f(1), .. f(size - 1) (size a power of two up to MOST): each thread gets
// its entries' in ``out``, thread t entries t * per .. of them; block-wide, returns per.
template <typename F>
__device__ int scan_entries(Shared& sh, int size, F&& f, unsigned long long (&out)[MOST / RT]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = max(1, size / RT);
  unsigned long long run = 0;
#pragma unroll
  for (int i = 0; i < MOST / RT; ++i) {
    const int at = threadIdx.x * per + i;
    if (i < per && at < size) run += f(at);
    out[i] = run;
  }
  unsigned long long incl = run;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(ALL, incl, o);
    if (lane >= o) incl += t;
  }
  __syncthreads();
  if (lane == 31) sh.red64[warp] = incl;
  __syncthreads();
  unsigned long long before = incl - run;
  for (int w = 0; w < warp; ++w) before += sh.red64[w];
#pragma unroll
  for (int i = 0; i < MOST / RT; ++i) out[i] += before;
  return per;
}

// Everything behind the list, by the first CTA alone: the cuts are places in the sorted list, and the
// draw is a second sort, of the kept tokens by id.
template <typename T>
__device__ void draw_from_list(Shared& sh, const Row<T>& row, int n, int k, float tp, unsigned long long floor_w, float u,
                               int32_t* token, float* prob) {
  List& list = sh.list;
  int size = 32;
  while (size < n) size *= 2;
  for (int i = n + threadIdx.x; i < size; i += RT) list.entry[i] = 0ull;
  __syncthreads();
  sort_entries<false>(list.entry, size);  // largest key first, lowest id first among equals
  const int n_k = k > 0 ? min(k, n) : n;
  for (int i = threadIdx.x; i < size; i += RT)
    list.mass[i] = i < n_k ? row.fixed((uint32_t)(list.entry[i] >> 32)) : 0ull;
  __syncthreads();
  unsigned long long sum[MOST / RT];
  int per = scan_entries(sh, size, [&](int i) { return list.mass[i]; }, sum);
  // the number of kept tokens: those that start below the limit and weigh enough (each a prefix)
  unsigned long long limit = ~0ull;
  if (tp < 1.f) {
    unsigned long long z = 0;
    for (int w = 0; w < RW; ++w) z += sh.red64[w];
    const double edge = ceil((double)fmaxf(tp, 0.f) * (double)z);
    limit = edge < 1.0 ? 1ull : (unsigned long long)edge;
  }
  int kept = 0;
#pragma unroll
  for (int i = 0; i < MOST / RT; ++i) {
    const int at = threadIdx.x * per + i;
    if (i < per && at < n_k)
      kept += sum[i] - list.mass[at] < limit && list.mass[at] >= floor_w;
  }
  kept = __reduce_add_sync(ALL, kept);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.red32[threadIdx.x >> 5] = kept;
  __syncthreads();
  kept = 0;
  for (int w = 0; w < RW; ++w) kept += sh.red32[w];
  kept = max(kept, 1);
  // the kept tokens by id: id in the upper bits, the place in the sorted list below
  size = 32;
  while (size < kept) size *= 2;
  for (int i = threadIdx.x; i < size; i += RT)
    list.entry[i] = i < kept ? (unsigned long long)(0xFFFFFFFFu - (uint32_t)list.entry[i]) << 32 | i : ~0ull;
  __syncthreads();
  sort_entries<true>(list.entry, size);
  per = scan_entries(sh, size, [&](int i) { return i < kept ? list.mass[(uint32_t)list.entry[i]] : 0ull; }, sum);
  unsigned long long total = 0;
  for (int w = 0; w < RW; ++w) total += sh.red64[w];
  const double want = u > 0.f ? floor((double)u * (double)total) : 0.0;
  const unsigned long long target = want >= (double)total ? total - 1ull : (unsigned long long)want;
#pragma unroll
  for (int i = 0; i < MOST / RT; ++i) {
    const int at = threadIdx.x * per + i;
    if (i >= per || at >= kept) continue;
    const unsigned long long w = list.mass[(uint32_t)list.entry[at]];
    if (sum[i] > target && sum[i] - w <= target) {
      *token = (int32_t)(list.entry[at] >> 32);
      if (prob) *prob = (float)((double)w / (double)total);
    }
  }
}

// The row of cluster ``place``: the rows whose cuts are selected over the whole row first, each kind in
// ascending order. They take up to ten times the others, and one that starts last holds the launch.
__device__ int row_at(Shared& sh, int place, int rows, int listed, const float* temperature, const int32_t* top_k,
                      const float* top_p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto slow = [&](int r) {  // (the three loads side by side)
    r = min(r, rows - 1);
    const float p = top_p[r], t = temperature ? temperature[r] : 1.f;
    const int k = top_k ? top_k[r] : 0;
    return p < 1.f & t > 0.f & !(k > 0 & k <= listed);
  };
  int many = 0;
  bool mine = slow(threadIdx.x);
  uint32_t votes = __ballot_sync(ALL, mine & threadIdx.x < rows);
  if (lane == 0) sh.red32[warp] = __popc(votes);
  __syncthreads();
  for (int w = 0; w < RW; ++w) many += sh.red32[w];
  for (int r0 = RT; r0 < rows; r0 += RT) many += __syncthreads_count(slow(r0 + threadIdx.x) & r0 + threadIdx.x < rows);
  const bool want = place < many;
  int before = want ? 0 : many;
  for (int r0 = 0; r0 < rows; r0 += RT) {
    const int r = r0 + threadIdx.x;
    if (r0 > 0) mine = slow(r);
    mine = (mine == want) & r < rows;
    votes = __ballot_sync(ALL, mine);
    __syncthreads();
    if (lane == 0) sh.red32[warp] = __popc(votes);
    __syncthreads();
    int at = before + __popc(votes & ((1u << lane) - 1u));
    for (int w = 0; w < RW; ++w) {
      if (w < warp) at += sh.red32[w];
      before += sh.red32[w];
    }
    if (mine & at == place) sh.pub_id = r;
  }
  __syncthreads();
  const int row = sh.pub_id;
  __syncthreads();
  return row;
}

template <typename T>
__global__ void __launch_bounds__(RT, 2)
    sample_rows_kernel(const T* __restrict__ logits, long long row_stride, int vocab, int slice, int ordered_rows,
                       const float* __restrict__ temperature, const int32_t* __restrict__ top_k,
                       const float* __restrict__ top_p, const float* __restrict__ min_p,
                       const float* __restrict__ uniform, int32_t* __restrict__ tokens,
                       float* __restrict__ probs, int* status) {
  using K = Keys<T>;
  using Raw = typename K::Raw;
  pdl_prologue();
  __shared__ Shared sh;
  extern __shared__ __align__(16) uint8_t slice_smem[];
  cg::cluster_group cl = cg::this_cluster();
  const int ctas = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  int r = blockIdx.x / ctas;
  if (ordered_rows > 0) r = row_at(sh, r, ordered_rows, 4 * RW * ctas, temperature, top_k, top_p);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = min(vocab, rank * slice), n = min(vocab, first + slice) - first;
  if (tid < 64) sh.pow2[tid] = make_uint2(POW2[tid], __float_as_uint((float)POW2[tid] * 0.125f));

  // ---- the slice into shared memory; 16-byte loads from the first aligned logit on. Vector 0 of the
  // slice starts at that boundary's token or before: ``skew`` places of it are padding
  constexpr int PER = K::PER;
  const Raw* src = reinterpret_cast<const Raw*>(logits) + (long long)r * row_stride + first;
  const int skew = (int)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(Raw));
  uint4* vecs = reinterpret_cast<uint4*>(slice_smem);
  const int count = n > 0 ? (skew + n + PER - 1) / PER : 0;
  const uint4* vsrc = reinterpret_cast<const uint4*>(src - skew);
  float top = -INFINITY;
  for (int v = tid; v < count; v += RT) {
    if ((v > 0 || skew == 0) && (v + 1) * PER <= skew + n) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(vecs + v)), "l"(vsrc + v) : "memory");
    } else {  // the first or last vector, in part
      union {
        uint4 v;
        Raw e[PER];
      } part;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = v * PER + j - skew;
        part.e[j] = i >= 0 && i < n ? src[i] : K::PAD;
      }
      vecs[v] = part.v;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");  // (a thread reads its own vectors until the first barrier)
  for (int v = tid; v < count; v += RT) top = fmaxf(top, K::top(vecs[v]));

  // ---- the row's largest logit, and the largest of each eight lanes' tokens
  uint32_t top_key = K::key_of(top);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top_key = max(top_key, __shfl_xor_sync(ALL, top_key, o));
  if ((lane & 7) == 0) sh.pub_tops[4 * warp + (lane >> 3)] = top_key;
  const uint32_t warp_top = __reduce_max_sync(ALL, top_key), thread_low = __reduce_min_sync(ALL, K::key_of(top));
  if (lane == 0) sh.red64[warp] = (unsigned long long)warp_top << 32 | thread_low;
  __syncthreads();
  if (tid == 0) {
    uint32_t best = 0u, tl = 0xFFFFFFFFu;
    for (int w = 0; w < RW; ++w) {
      best = max(best, (uint32_t)(sh.red64[w] >> 32));
      tl = min(tl, (uint32_t)sh.red64[w]);
    }
    sh.pub_best = best;
    sh.pub_low = tl;
    sh.pub_id = 0x7FFFFFFF;
    sh.pub_listed = 0u;
    sh.bound = 0u;
  }
  cl.sync();
  uint32_t low = 0xFFFFFFFFu, row_top = 0u;
  for (int q = 0; q < ctas; ++q) {
    row_top = max(row_top, *cl.map_shared_rank(&sh.pub_best, q));
    low = min(low, *cl.map_shared_rank(&sh.pub_low, q));
  }
  Row<T> row;
  row.vecs = vecs;
  row.count = count;
  row.top = row_top;
  row.pow2 = sh.pow2;
  const float T_row = temperature ? temperature[r] : 1.f;
  const float m = K::value(row_top);
  constexpr float LOG2E_1 = 1.442695041f, LOG2E_2 = 1.925963e-8f;  // log2(e) in two parts
  // (differences of logits may overflow where they matter, log2(e) / T does at subnormal temperatures)
  row.scale = T_row > 1e30f ? 0.5f : T_row < 1e-20f ? 18446744073709551616.f : 1.f;
  const float T_scaled = T_row * row.scale;
  row.c1 = LOG2E_1 / T_scaled;
  row.c2 = isinf(T_row) ? 0.f : (fmaf(-row.c1, T_scaled, LOG2E_1) + LOG2E_2) / T_scaled;
  row.minus = -m * row.scale;
  // At a temperature below 2^-29 or so of the largest logit, the next lower fp32 number weighs less than
  // 2^-46: the largest logit alone has a weight.
  row.inf = isinf(m) || !(fabsf(row.minus) * row.c1 < 7.7e8f);
  row.careful = row.inf || T_row > 1e30f;
  row.least = m - 41.6f * T_row;  // (60 ln 2)
  if (m - row.least < 41.f * T_row) row.least = nextafterf(row.least, -INFINITY);
  row.least = fmaxf(row.least, -3.4028234663852886e38f);
  // the key of a logit that weighs w, or of one a little lighter (the logarithm's error is a bound's)
  auto key_at = [&](float w) -> uint32_t {
    const float x = m + T_row * (logf(w) - 1e-3f);
    const uint32_t f = x > -3.0e38f ? K::key_of(x) : 0u;
    return min(f > 0u ? f - 1u : 0u, row_top);
  };
  const bool empty = row_top <= K::NONE;
  if (empty || !(T_row > 0.f)) {  // nothing to draw, or greedy: the lowest id of the largest logit
    if (!empty) {
      row.above(row_top, [&](int i, uint32_t) { atomicMin(cl.map_shared_rank(&sh.pub_id, 0), first + i - skew); });
    }
    cl.sync();
    if (rank == 0 && tid == 0) {
      tokens[r] = empty ? -1 : sh.pub_id;
      if (probs) probs[r] = empty ? 0.f : 1.f;
      if (empty) report(status, NE_DEV_BAD_TOKEN);
    }
    return;
  }

  // ---- the cuts
  const int k = top_k ? top_k[r] : 0;
  const float tp = top_p ? top_p[r] : 1.f, mp = min_p ? min_p[r] : 0.f;
  const unsigned long long floor_w = mp > 0.f ? (unsigned long long)ceil(fmin((double)mp, 1.0) * FIX) : 0ull;
  const bool some = k > 0 && k < vocab;
  // A lower bound of all cuts: the k-th largest of the quarter warps' maxima (or of the warps', where
  // they are enough), each of which is a token, is no larger than the k-th largest token, and little
  // less. Without top-p, whose mass counts the tokens that min-p cuts, min-p is a bound too (a key
  // lower for the rounding of the logarithm).
  uint32_t bound = 0u;
  if (some && k <= 4 * RW * ctas) {
    const int pool = k <= RW * ctas ? RW * ctas : 4 * RW * ctas;
    uint32_t mine = 0u;
    if (tid < pool) {
      const uint32_t* theirs = cl.map_shared_rank(&sh.pub_tops[0], tid / (pool / ctas));
      const int at = tid % (pool / ctas);
      if (pool == RW * ctas)
        mine = max(max(theirs[4 * at], theirs[4 * at + 1]), max(theirs[4 * at + 2], theirs[4 * at + 3]));
      else
        mine = theirs[at];
      sh.tops[tid] = mine;
    }
    __syncthreads();
    if (tid < pool) {
      int at_least = 0;
      for (int i = 0; i < pool; i += 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(&sh.tops[i]);
        at_least += (x.x >= mine) + (x.y >= mine) + (x.z >= mine) + (x.w >= mine);
      }
      if (at_least >= k) atomicMax(&sh.bound, mine);
    }
    __syncthreads();
    bound = sh.bound;
  }
  if (mp > 0.f && !(tp < 1.f)) {
    bound = max(bound, key_at(fminf(mp, 1.f)));
  }
  if (bound > K::NONE) {
    uint32_t have = 0;
    row.above(bound, [&](int, uint32_t) { ++have; });
    const unsigned long long n_list = cluster_sum(cl, sh, have, 0);
    if (n_list <= MOST) {
      row.above(bound, [&](int i, uint32_t key) {
        const uint32_t at = atomicAdd(cl.map_shared_rank(&sh.pub_listed, 0), 1u);
        cl.map_shared_rank(&sh.list, 0)->entry[at] =
            (unsigned long long)key << 32 | (0xFFFFFFFFu - (uint32_t)(first + i - skew));
      });
      cl.sync();
      if (rank == 0)
        draw_from_list(sh, row, (int)n_list, some ? k : 0, tp, mp > 1.f ? ~0ull : floor_w, uniform[r], tokens + r,
                       probs ? probs + r : nullptr);
      return;
    }
  }
  Cut cut{K::NONE + 1u, 0xFFFFFFFFu, 0u};  // every token (all ties of the lowest key)
  if (mp > 1.f) {
    cut = select_cut<T, false>(cl, sh, row, row_top, row_top, 1ull);
  } else {
    if (some) {  // (the threads' maxima bound the k-th largest too)
      const uint32_t lo = max(max(bound, k <= ctas * RT ? low : 0u), K::NONE + 1u);
      cut = select_cut<T, false>(cl, sh, row, lo, row_top, (unsigned long long)k);
    }
    if (tp < 1.f) {
      unsigned long long z = 0;
      // with top-k the few tokens that are left; else every token, and where their mass lies by bands of
      // the weight: a column of sums a thread, in shared memory, without atomics
      const bool banded = !cut.ties && !row.careful;
      if (cut.ties) {
        row.above(cut.key, [&](int, uint32_t key) {
          if (key > cut.key) z += row.fixed(key);
        });
      } else if (!banded) {
        for (int v = tid; v < count; v += RT) z += row.vector_mass(vecs[v]);
      } else {
#pragma unroll
        for (int x = 0; x < BANDS; ++x) sh.column[x][tid] = 0.f;
        for (int v = tid; v < count; v += RT) {
          const uint4 x = vecs[v];
          int band[PER];
          float approx[PER];
#pragma unroll
          for (int j = 0; j < PER; j += 2) {
            unsigned long long a, b;
            row.power2(K::logit(x, j), K::logit(x, j + 1), a, b, &band[j], &approx[j]);
            z += a + b;
          }
#pragma unroll
          for (int j = 0; j < PER; ++j) sh.column[band[j]][tid] += approx[j];
        }
        __syncthreads();
        if (warp < BANDS) {
          float t = 0.f;
#pragma unroll
          for (int i = 0; i < RT / 32; ++i) t += sh.column[warp][i * 32 + lane];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(ALL, t, o);
          if (lane == 0) sh.pub_band[warp] = t;
        }
      }
      z = cluster_sum(cl, sh, z, 1);
      if (cut.ties) z += (unsigned long long)cut.keep * row.fixed(cut.key);
      const double edge = ceil((double)fmaxf(tp, 0.f) * (double)z);
      const unsigned long long limit = edge < 1.0 ? 1ull : (unsigned long long)edge;
      // tokens below w0 = (1 - top_p) z / vocab hold less than (1 - top_p) z together: the cut is at or
      // above w0
      const float w0 = (1.f - fmaxf(tp, 0.f)) * ((float)((double)z / FIX) / vocab * 0.999f);
      const uint32_t lo = max(cut.key, w0 > 0.f ? key_at(w0) : 0u);
      Cut found{lo, 0u, 0u};
      if (banded) {
        // the bands whose running sum passes the limit, give or take the sums' error
        const float want = (float)((double)limit / FIX) * 268435456.f;  // (the bands' weights are times 2^28)
        int b0 = BANDS, b1 = BANDS;
        float run = 0.f;
        for (int x = 0; x < BANDS; ++x) {
          for (int q = 0; q < ctas; ++q) run += cl.map_shared_rank(&sh.pub_band[0], q)[x];
          if (b0 == BANDS && run >= want * 0.999f) b0 = x;
          if (b1 == BANDS && run >= want * 1.001f) b1 = x;
        }
        if (b1 < BANDS - 1) {
          const float above = b0 > 0 ? m + T_row * (-1.3862944f * b0 + 0.02f) : m;  // (a band is rounded by 1 / 128)
          const uint32_t band_hi = b0 > 0 ? min(K::key_of(above) + 1u, row_top) : row_top;
          const uint32_t band_lo = max(lo, key_at(exp2f(-2.f * b1 - 2.02f)));
          if (band_lo <= band_hi) found = select_cut<T, true>(cl, sh, row, band_lo, band_hi, limit, band_lo == lo);
          if (!found.ties) cl.sync();  // (not there after all: look everywhere)
        }
      }
      if (!found.ties) found = select_cut<T, true>(cl, sh, row, lo, row_top, limit);
      cut = found;
    }
  }
  const bool partial = cut.ties != 0u && cut.keep < cut.ties;  // the cut divides its ties

  // ---- the draw: warp w of CTA c walks the w-th part of slice c, a vector a lane, in ascending id order
  const int len = (count + RW - 1) / RW, begin = min(count, warp * len), end = min(count, begin + len);
  const float least = K::value(cut.key);
  uint32_t tie_base = 0;
  if (partial) {  // ties before this warp's part
    uint32_t ties = 0;
    for (int v = begin + lane; v < end; v += 32) {
      const uint4 x = vecs[v];
      if (!(K::top(x) >= least)) continue;
#pragma unroll
      for (int j = 0; j < PER; ++j) ties += K::at(x, j) == cut.key;
    }
    ties = __reduce_add_sync(ALL, ties);
    __syncthreads();
    if (lane == 0) sh.red32[warp] = ties;
    __syncthreads();
    uint32_t all = 0;
    for (int w = 0; w < RW; ++w) {
      if (w < warp) tie_base += sh.red32[w];
      all += sh.red32[w];
    }
    if (tid == 0) sh.pub_ties = all;
    cl.sync();
    for (int q = 0; q < rank; ++q) tie_base += *cl.map_shared_rank(&sh.pub_ties, q);
  }
  // the kept mass of a lane's vector (``ranked``: ties before it); each(j, mass) in id order
  auto kept = [&](const uint4& x, uint32_t ranked, auto&& each) {
    if (!(K::top(x) >= least)) return;
    unsigned long long w[PER];
    row.masses(x, w);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t key = K::at(x, j);
      if (key < cut.key) continue;
      if (key == cut.key && partial && ranked++ >= cut.keep) continue;
      if (w[j] >= floor_w) each(j, w[j]);
    }
  };
  // ties in the lanes before this one's, and in all of them (only where the cut divides its ties)
  auto rank_of = [&](const uint4& x, uint32_t& before) -> uint32_t {
    if (!partial) return 0u;
    uint32_t mine = 0;
    if (K::top(x) >= least) {
#pragma unroll
      for (int j = 0; j < PER; ++j) mine += K::at(x, j) == cut.key;
    }
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(ALL, incl, o);
      if (lane >= o) incl += t;
    }
    const uint32_t at = before + incl - mine;
    before += __shfl_sync(ALL, incl, 31);
    return at;
  };
  union {
    Raw e[PER];
    uint4 v;
  } none;
#pragma unroll
  for (int j = 0; j < PER; ++j) none.e[j] = K::PAD;
  const bool whole = !cut.ties && floor_w == 0ull;  // every token is kept
  unsigned long long sum = 0;
  uint32_t before_ties = tie_base;
  for (int b = begin; b < end; b += 32) {
    const uint4 x = b + lane < end ? vecs[b + lane] : none.v;
    unsigned long long part = 0;
    if (whole) {
      part = row.vector_mass(x);
    } else {
      const uint32_t ranked = rank_of(x, before_ties);
      kept(x, ranked, [&](int, unsigned long long w) { part += w; });
    }
    part = warp_add(part);
    if (lane == 0) sh.chunk[warp][(b - begin) >> 5] = part;
    sum += part;
  }
  __syncthreads();
  if (lane == 0) sh.red64[warp] = sum;
  __syncthreads();
  unsigned long long mine = 0;
  for (int w = 0; w < RW; ++w) mine += sh.red64[w];
  if (tid == 0) sh.pub_sum[2] = mine;
  cl.sync();
  unsigned long long total = 0, before = 0;
  for (int q = 0; q < ctas; ++q) {
    const unsigned long long t = *cl.map_shared_rank(&sh.pub_sum[2], q);
    if (q < rank) before += t;
    total += t;
  }
  for (int w = 0; w < warp; ++w) before += sh.red64[w];
  const float u = uniform[r];
  const double want = u > 0.f ? floor((double)u * (double)total) : 0.0;
  const unsigned long long target = want >= (double)total ? total - 1ull : (unsigned long long)want;
  if (before <= target && before + sum > target) {  // one warp of the cluster
    before_ties = tie_base;
    unsigned long long run = before;
    for (int b = begin; b < end; b += 32) {
      const unsigned long long part = sh.chunk[warp][(b - begin) >> 5];
      const uint4 x = b + lane < end ? vecs[b + lane] : none.v;
      const uint32_t ranked = rank_of(x, before_ties);
      if (run + part <= target) {
        run += part;
        continue;
      }
      unsigned long long w = 0;
      kept(x, ranked, [&](int, unsigned long long f) { w += f; });
      unsigned long long incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(ALL, incl, o);
        if (lane >= o) incl += t;
      }
      const uint32_t hit = __ballot_sync(ALL, run + incl > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          unsigned long long at = run + incl - w;
          bool done = false;
          kept(x, ranked, [&](int j, unsigned long long f) {
            at += f;
            if (done || at <= target) return;
            done = true;
            tokens[r] = first - skew + (b + lane) * PER + j;
            if (probs) probs[r] = (float)((double)f / (double)total);
          });
        }
        break;
      }
      run += __shfl_sync(ALL, incl, 31);
    }
  }
  cl.sync();  // (no CTA leaves while another may read its shared memory)
}

// Shared memory of a slice: a padded vector at either end.
template <typename T>
size_t slice_bytes(int vocab, int ctas) {
  return ((size_t)((vocab + ctas - 1) / ctas) * sizeof(T) + 47) / 16 * 16;
}
// The largest slice that leaves room for two CTAs on an SM.
size_t max_pair_bytes(int dev) {
  int per_sm = 0, reserved = 0;
  cudaDeviceGetAttribute(&per_sm, cudaDevAttrMaxSharedMemoryPerMultiprocessor, dev);
  cudaDeviceGetAttribute(&reserved, cudaDevAttrReservedSharedMemoryPerBlock, dev);
  const size_t one = (size_t)per_sm / 2;
  return one > reserved + sizeof(Shared) ? one - reserved - sizeof(Shared) : 0;
}

template <typename T>
int launch_sample_rows(const void* logits, int rows, int vocab, long long row_stride, const float* temperature,
                       const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform,
                       int32_t* tokens, float* probs, int* status, cudaStream_t stream) {
  int dev = 0, sms = 148, ctas = 1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NE_ERR_CUDA;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  // Slices that two CTAs an SM have room for, as far as clusters of four (fp32: of two) give them, then
  // slices of up to 80 KB: the barriers of a larger cluster cost more than its shorter slices save (measured, 320
  // rows of 151,936 bf16, top-k 20: 2 / 4 / 8 CTAs 97 / 79 / 123 us), but half the CTAs an SM cost more than the
  // next size does: 320 rows of 80,000 bf16 in 2 / 4 CTAs, mixed settings 166 / 142 us, top-k 20 88 / 74, top-p
  // 221 / 206; 640 of 40,000 in 1 / 2 162 / 148, 91 / 90, 225 / 206; 640 of 20,000 fp32 in 1 / 2 131 / 125,
  // 86 / 86, 184 / 184. Not so for 320 of 160,000 bf16 in 4 / 8 (279 / 287, 137 / 137, 412 / 438), nor for 40,000
  // fp32 in 2 / 4, where top-p's selection passes lose more than the rest gains (127 / 119, 82 / 72, 176 / 209).
  // Few rows leave SMs idle, and slices above 8,192 tokens are halved then; where every SM has one CTA, above
  // 14,000 (measured, rows of mixed settings: slices of 16,000 / 19,000 / 20,000 tokens halved take 60 -> 47,
  // 125 -> 90 and 70 -> 55 us, of 12,500 58 -> 67).
  const size_t pair_bytes = max_pair_bytes(dev);
  const int paired = sizeof(T) == 2 ? 4 : 2;
  while (ctas < MAX_CLUSTER && slice_bytes<T>(vocab, ctas) > (ctas < paired ? pair_bytes : MID_SLICE_BYTES)) ctas *= 2;
  while (ctas < MAX_CLUSTER && (long long)rows * ctas <= sms &&
         vocab > (2LL * rows * ctas <= sms ? 8192 : 14000) * ctas)
    ctas *= 2;
  const int slice = (vocab + ctas - 1) / ctas;
  const size_t smem = slice_bytes<T>(vocab, ctas);
  // rows that do not all start at once are put in order (320 rows of mixed settings 228 -> 176 us; of one
  // setting, where the order gains nothing, 33 -> 41 to 660 -> 670)
  const int resident = smem <= pair_bytes ? 2 : 1;
  const int ordered = top_p && (long long)rows * ctas > (long long)resident * sms && rows <= 4096 ? rows : 0;
  if (smem > MAX_SLICE_BYTES) return NE_ERR_UNSUPPORTED;
  static bool done[64] = {};
  if (!done[dev]) {
    if (cudaFuncSetAttribute(sample_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)MAX_SLICE_BYTES) != cudaSuccess)
      return NE_ERR_CUDA;
    done[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * ctas);
  cfg.blockDim = dim3(RT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[3];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = add_common_attrs(attr, 1);
  return cudaLaunchKernelEx(&cfg, sample_rows_kernel<T>, static_cast<const T*>(logits), row_stride, vocab, slice, ordered,
                            temperature, top_k, top_p, min_p, uniform, tokens, probs, status) == cudaSuccess
             ? NE_OK
             : NE_ERR_CUDA;
}

}  // namespace

}  // namespace ne

extern "C" NE_API int ne_sample_logits(const void* logits, int logits_fp32, int rows, int vocab, long long row_stride,
                                       const float* temperature, const int32_t* top_k, const float* top_p,
                                       const float* min_p, const float* uniform, int32_t* tokens, float* probs,
                                       int32_t* status, void* stream) {
  if (!logits || !uniform || !tokens || rows < 0 || rows > (1 << 24) || vocab < 1 || vocab > ne::MAX_VOCAB ||
      row_stride < vocab || (reinterpret_cast<uintptr_t>(logits) & (logits_fp32 ? 3u : 1u)))
    return NE_ERR_INVALID;
  if (rows == 0) return NE_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return logits_fp32 ? ne::launch_sample_rows<float>(logits, rows, vocab, row_stride, temperature, top_k, top_p, min_p,
                                                     uniform, tokens, probs, status, s)
                     : ne::launch_sample_rows<__nv_bfloat16>(logits, rows, vocab, row_stride, temperature, top_k,
                                                             top_p, min_p, uniform, tokens, probs, status, s);
}
