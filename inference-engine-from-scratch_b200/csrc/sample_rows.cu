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
// A row is a cluster of CTAs, each with a slice of the row in shared memory as ordered integer keys
// (larger key = larger logit), so the logits are read from memory once. Cuts are found by a radix
// select over the keys, 1024 bins a pass, counts and masses added over the cluster. A border is
// decided by sums over the whole vocabulary, so weights are computed in 64 bits (an error of 1e-7
// in a weight, as fp32 gives, moves the border of a flat distribution past a token) and summed as
// 2^-45 fixed point, whose sums do not depend on their order: the same inputs give the same tokens.
#include <cooperative_groups.h>

#include "sampling.cuh"

namespace ne {

namespace {

namespace cg = cooperative_groups;

constexpr int RT = 512;               // threads per CTA
constexpr int RW = RT / 32;
constexpr int BINS = 1024;
constexpr int MAX_CLUSTER = 8;
constexpr unsigned ALL = 0xFFFFFFFFu;
constexpr double FIX = 35184372088832.0;  // 2^45
constexpr int MAX_VOCAB = 1 << 18;        // 262,144 weights of at most 1 sum to at most 2^63
constexpr size_t MAX_SLICE_BYTES = 200 << 10;

// Ordered key of a logit, in the low bits: 16 for bf16, 32 for fp32. NaN and -inf: never drawn.
template <typename T>
struct Keys;
template <>
struct Keys<__nv_bfloat16> {
  using Raw = uint16_t;
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
  static __device__ __forceinline__ uint32_t floor_key(float x) {  // a key no larger than any logit >= x has
    return key(__float_as_uint(x) >> 16);                          // (truncated towards 0: rounded down below)
  }
};
template <>
struct Keys<float> {
  using Raw = uint32_t;
  static constexpr uint32_t NONE = 0x007FFFFFu;
  static __device__ __forceinline__ uint32_t key(uint32_t b) {
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
    if (b == 0x80000000u) b = 0u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
  }
  static __device__ __forceinline__ uint32_t floor_key(float x) { return key(__float_as_uint(x)); }
};

struct Shared {
  unsigned long long mass[2][BINS];
  uint32_t count[2][BINS];
  unsigned long long red64[RW];
  uint32_t red32[RW];
  // published to the cluster
  unsigned long long pub_best, pub_sum;
  uint32_t pub_low[2], pub_ties;
  // the bin a select pass chose
  int sel_bin;
  uint32_t sel_count;
  unsigned long long sel_mass;
  uint32_t sel_here;
  unsigned long long sel_here_mass;
};

// A cut of the descending order: tokens with a key above ``key``, and the first ``keep`` (by id) of
// the ``ties`` tokens that have it.
struct Cut {
  uint32_t key, keep, ties;
};

template <typename T>
struct Row {
  const typename Keys<T>::Raw* keys;  // this CTA's slice
  int n;                              // its tokens
  uint32_t top;                       // the row's largest key
  double m, temp;                     // its value; the temperature

  __device__ __forceinline__ double weight(uint32_t k) const {
    if (k == top) return 1.0;
    if (k <= Keys<T>::NONE) return 0.0;
    return exp(((double)Keys<T>::value(k) - m) / temp);
  }
  __device__ __forceinline__ unsigned long long fixed(uint32_t k) const { return __double2ull_rn(weight(k) * FIX); }
};

__device__ __forceinline__ unsigned long long warp_add(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
  return v;
}

// Sum over the CTA, then over the cluster; every thread of the cluster gets it.
__device__ unsigned long long cluster_sum(cg::cluster_group& cl, Shared& sh, unsigned long long v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_add(v);
  if (lane == 0) sh.red64[warp] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned long long t = 0;
    for (int w = 0; w < RW; ++w) t += sh.red64[w];
    sh.pub_sum = t;
  }
  cl.sync();
  unsigned long long total = 0;
  for (unsigned r = 0; r < cl.num_blocks(); ++r) total += *cl.map_shared_rank(&sh.pub_sum, r);
  cl.sync();  // read everywhere before the next use
  return total;
}

// The cut at which the tokens with larger keys, and some of the ties, first reach ``limit``: a count
// (MASS false) or a mass in fixed point. Only keys in [lo, hi] are looked at; the tokens above hi
// are none, and those in [lo, hi] reach the limit (or the cut is the lowest key present).
template <typename T, bool MASS>
__device__ Cut select_cut(cg::cluster_group& cl, Shared& sh, const Row<T>& row, uint32_t lo, uint32_t hi,
                          unsigned long long limit) {
  unsigned long long above = 0;
  int buf = 0;
  uint32_t ties = 0;
  for (;;) {
    const uint32_t range = hi - lo;
    const int shift = max(0, 32 - __clz(range) - 10);
    for (int i = threadIdx.x; i < BINS; i += RT) {
      sh.count[buf][i] = 0u;
      if (MASS) sh.mass[buf][i] = 0ull;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < row.n; i += RT) {
      const uint32_t k = row.keys[i];
      if (k < lo || k > hi || k <= Keys<T>::NONE) continue;
      const uint32_t b = (k - lo) >> shift;
      atomicAdd(&sh.count[buf][b], 1u);
      if (MASS) atomicAdd(&sh.mass[buf][b], row.fixed(k));
    }
    cl.sync();
    // every CTA adds the cluster's bins: thread t owns bins 2 t and 2 t + 1
    uint32_t c[2] = {0u, 0u};
    unsigned long long w[2] = {0ull, 0ull};
    for (unsigned r = 0; r < cl.num_blocks(); ++r) {
      const uint32_t* rc = cl.map_shared_rank(&sh.count[buf][0], r);
      const unsigned long long* rm = cl.map_shared_rank(&sh.mass[buf][0], r);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        c[j] += rc[2 * threadIdx.x + j];
        if (MASS) w[j] += rm[2 * threadIdx.x + j];
      }
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
    for (int x = warp + 1; x < RW; ++x) before += sh.red64[x];
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
    if (bin < 0) break;  // no token in the range (not reached: the largest key starts at 0)
    above = sh.sel_mass;
    ties = sh.sel_count;
    const uint32_t nlo = lo + ((uint32_t)bin << shift);
    const uint32_t last = nlo + ((1u << shift) - 1u);
    hi = last < nlo ? hi : min(hi, last);
    lo = nlo;
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

template <typename T>
__global__ void __launch_bounds__(RT)
    sample_rows_kernel(const T* __restrict__ logits, long long row_stride, int vocab, int slice,
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
  const int r = blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = min(vocab, rank * slice), n = min(vocab, first + slice) - first;

  // ---- the slice into shared memory, as keys; 16-byte loads from the first aligned logit on
  constexpr int PER = 16 / sizeof(Raw);
  const Raw* src = reinterpret_cast<const Raw*>(logits) + (long long)r * row_stride + first;
  const int skew = (int)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(Raw));  // tokens past a boundary
  Raw* keys = reinterpret_cast<Raw*>(slice_smem) + skew;
  const int head = min(n, (PER - skew) & (PER - 1));
  const int vecs = (n - head) / PER;
  uint32_t top = 0u;
  int top_at = 0;
  auto take = [&](int i, uint32_t raw) {
    const uint32_t k = K::key(raw);
    if (k > top) {
      top = k;
      top_at = i;
    }
    return (Raw)k;
  };
  if (tid < head) keys[tid] = take(tid, src[tid]);
  const uint4* vsrc = reinterpret_cast<const uint4*>(src + head);
#pragma unroll 4
  for (int v = tid; v < vecs; v += RT) {
    const uint4 x = vsrc[v];
    union {
      uint4 v;
      Raw e[PER];
    } in, out;
    in.v = x;
#pragma unroll
    for (int j = 0; j < PER; ++j) out.e[j] = take(head + v * PER + j, in.e[j]);
    *reinterpret_cast<uint4*>(keys + head + v * PER) = out.v;
  }
  for (int i = head + vecs * PER + tid; i < n; i += RT) keys[i] = take(i, src[i]);

  // ---- the row's largest key (lowest id among equals), and lower bounds that hold 1 token each
  unsigned long long best = ((unsigned long long)top << 32) | (0xFFFFFFFFu - (uint32_t)(first + top_at));
  const uint32_t thread_low = __reduce_min_sync(ALL, top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long t = __shfl_xor_sync(ALL, best, o);
    best = t > best ? t : best;
  }
  if (lane == 0) {
    sh.red64[warp] = best;
    sh.red32[warp] = thread_low;
  }
  __syncthreads();
  if (tid == 0) {
    unsigned long long b = 0;
    uint32_t wl = 0xFFFFFFFFu, tl = 0xFFFFFFFFu;
    for (int w = 0; w < RW; ++w) {
      b = sh.red64[w] > b ? sh.red64[w] : b;
      wl = min(wl, (uint32_t)(sh.red64[w] >> 32));
      tl = min(tl, sh.red32[w]);
    }
    sh.pub_best = b;
    sh.pub_low[0] = wl;
    sh.pub_low[1] = tl;
  }
  cl.sync();
  uint32_t low[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
  best = 0;
  for (int q = 0; q < ctas; ++q) {
    const unsigned long long b = *cl.map_shared_rank(&sh.pub_best, q);
    best = b > best ? b : best;
    const uint32_t* l = cl.map_shared_rank(&sh.pub_low[0], q);
    low[0] = min(low[0], l[0]);
    low[1] = min(low[1], l[1]);
  }
  const uint32_t row_top = (uint32_t)(best >> 32);
  const float T_row = temperature ? temperature[r] : 1.f;
  const bool empty = row_top <= K::NONE;
  if (empty || !(T_row > 0.f)) {  // nothing to draw, or greedy: the largest logit
    if (rank == 0 && tid == 0) {
      tokens[r] = empty ? -1 : (int32_t)(0xFFFFFFFFu - (uint32_t)best);
      if (probs) probs[r] = empty ? 0.f : 1.f;
      if (empty) report(status, NE_DEV_BAD_TOKEN);
    }
    cl.sync();  // (no CTA leaves while another may read its shared memory)
    return;
  }
  Row<T> row;
  row.keys = keys;
  row.n = n;
  row.top = row_top;
  row.m = (double)K::value(row_top);
  row.temp = (double)T_row;

  // ---- the cuts
  const int k = top_k ? top_k[r] : 0;
  const float tp = top_p ? top_p[r] : 1.f, mp = min_p ? min_p[r] : 0.f;
  Cut cut{K::NONE + 1u, 0xFFFFFFFFu, 0u};  // every token (all ties of the lowest key)
  bool partial = false;                    // the cut divides its ties
  if (mp > 1.f) {
    cut = select_cut<T, false>(cl, sh, row, row_top, row_top, 1ull);
  } else {
    if (k > 0 && k < vocab) {
      // ctas * RW warps (ctas * RT threads) each hold a token of at least the lowest warp (thread)
      // maximum: with k of them or fewer the k-th largest is no lower
      uint32_t lo = k <= ctas * RW ? low[0] : k <= ctas * RT ? low[1] : 0u;
      lo = max(lo, K::NONE + 1u);
      cut = select_cut<T, false>(cl, sh, row, lo, row_top, (unsigned long long)k);
    }
    if (tp < 1.f) {
      unsigned long long z = 0;
      for (int i = tid; i < n; i += RT) {
        const uint32_t key = keys[i];
        if (key > cut.key || (key == cut.key && !cut.ties)) z += row.fixed(key);
      }
      z = cluster_sum(cl, sh, z);
      if (cut.ties) z += (unsigned long long)cut.keep * row.fixed(cut.key);
      const double edge = ceil((double)fmaxf(tp, 0.f) * (double)z);
      const unsigned long long limit = edge < 1.0 ? 1ull : (unsigned long long)edge;
      // tokens below w0 = (1 - top_p) z / vocab hold less than (1 - top_p) z together: the cut is
      // at or above w0 (taken a little lower for the rounding of the logarithm)
      const double w0 = (1.0 - (double)fmaxf(tp, 0.f)) * ((double)z / FIX) / vocab * 0.999;
      uint32_t lo = cut.key;
      const double x0 = row.m + row.temp * log(w0);
      if (x0 > -3.0e38) {
        const float xf = __double2float_rd(x0);
        uint32_t f = K::floor_key(xf);
        f = f > 0u ? f - 1u : 0u;
        lo = max(lo, min(f, row_top));
      }
      cut = select_cut<T, true>(cl, sh, row, lo, row_top, limit);
    }
  }
  partial = cut.ties != 0u && cut.keep < cut.ties;
  const double floor_w = mp > 0.f && mp <= 1.f ? (double)mp : 0.0;

  // ---- the draw: warp w of CTA c walks the w-th part of slice c in ascending id order
  const int len = ((n + RT - 1) / RT) * 32, begin = min(n, warp * len), end = min(n, begin + len);
  uint32_t tie_base = 0;
  if (partial) {  // ties before this warp's part
    uint32_t ties = 0;
    for (int i = begin + lane; i < end; i += 32) ties += keys[i] == cut.key;
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
  // token i's mass if it is kept (``rank_at``: ties before it); warp-collective
  auto kept_mass = [&](int i, uint32_t& rank_at) -> unsigned long long {
    const bool in = i < end;
    const uint32_t key = in ? (uint32_t)keys[i] : 0u;
    const uint32_t tie = __ballot_sync(ALL, in && key == cut.key);
    bool keep = in && key > cut.key;
    if (in && key == cut.key) keep = !partial || rank_at + __popc(tie & ((1u << lane) - 1u)) < cut.keep;
    rank_at += __popc(tie);
    if (!keep) return 0ull;
    const double w = row.weight(key);
    return w >= floor_w ? __double2ull_rn(w * FIX) : 0ull;
  };
  unsigned long long sum = 0;
  uint32_t at = tie_base;
  for (int b = begin; b < end; b += 32) sum += kept_mass(b + lane, at);
  sum = warp_add(sum);
  __syncthreads();
  if (lane == 0) sh.red64[warp] = sum;
  __syncthreads();
  unsigned long long mine = 0;
  for (int w = 0; w < RW; ++w) mine += sh.red64[w];
  if (tid == 0) sh.pub_sum = mine;
  cl.sync();
  unsigned long long total = 0, before = 0;
  for (int q = 0; q < ctas; ++q) {
    const unsigned long long t = *cl.map_shared_rank(&sh.pub_sum, q);
    if (q < rank) before += t;
    total += t;
  }
  for (int w = 0; w < warp; ++w) before += sh.red64[w];
  const float u = uniform[r];
  const double want = u > 0.f ? floor((double)u * (double)total) : 0.0;
  const unsigned long long target = want >= (double)total ? total - 1ull : (unsigned long long)want;
  if (before <= target && before + sum > target) {  // one warp of the cluster
    at = tie_base;
    unsigned long long run = before;
    for (int b = begin; b < end; b += 32) {
      const unsigned long long w = kept_mass(b + lane, at);
      unsigned long long incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(ALL, incl, o);
        if (lane >= o) incl += t;
      }
      const uint32_t hit = __ballot_sync(ALL, run + incl > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          tokens[r] = first + b + lane;
          if (probs) probs[r] = (float)((double)w / (double)total);
        }
        break;
      }
      run += __shfl_sync(ALL, incl, 31);
    }
  }
  cl.sync();
}

template <typename T>
int launch_sample_rows(const void* logits, int rows, int vocab, long long row_stride, const float* temperature,
                       const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform,
                       int32_t* tokens, float* probs, int* status, cudaStream_t stream) {
  int ctas = 1;
  // about 8,192 tokens a CTA: below that the cluster's barriers cost more than the shorter slices save
  while (ctas < MAX_CLUSTER && vocab > 8192 * ctas) ctas *= 2;
  const int slice = (vocab + ctas - 1) / ctas;
  const size_t smem = ((size_t)slice + 16) * sizeof(T);
  if (smem > MAX_SLICE_BYTES) return NE_ERR_UNSUPPORTED;
  static bool done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NE_ERR_CUDA;
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
  return cudaLaunchKernelEx(&cfg, sample_rows_kernel<T>, static_cast<const T*>(logits), row_stride, vocab, slice,
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
