// Paged attention for a batch whose sequences share prompt prefixes (include/nespec.h,
// ne_prefix_attention), in three launches:
//
// * prefix_kernel: every group's query vectors, gathered over its entries, against its prefix:
//   tcgen05 tiles of 128 vectors x 128 keys, persistent CTAs that divide all prefixes' tiles evenly.
// * own_tokens_kernel: every entry against the tokens that are its own (all of them for an entry
//   without a group), 16 query vectors a tile on mma.sync, one CTA per (entry, KV head, tiles). It
//   starts on the SMs that prefix_kernel's first CTAs leave.
// * join_kernel: o = sum O_i 2^(m_i - m) / sum l_i 2^(m_i - m) over a vector's parts i, each an
//   unnormalised sum O_i of values, its sum of weights l_i and the (log2) reference m_i of both. (The
//   join inside own_tokens_kernel was measured and is slower: a CTA's few warps then wait for every
//   vector's parts in turn, 11,000 to 30,000 cycles.)
#include <algorithm>

#include "attention.cuh"
#include "attention_tile.cuh"
#include "gemm_tc.cuh"

namespace ne {

namespace {

constexpr int MAX_SEQS = 1024;   // entries of a launch (the plan of prefix_kernel is in shared memory)
constexpr int MAX_GROUP = 32;    // query heads per KV head
constexpr int TILE = 128;        // query vectors, and keys, of a tensor-core tile
constexpr unsigned ALL = 0xFFFFFFFFu;

// ---------------------------------------------------------------- the parts of a call, in its workspace
struct Parts {
  // own tokens: [split][row][head]
  float *own_o, *own_m, *own_l;
  // prefixes: per part up to 256 vectors at an offset of their own (prefix_offset)
  float *pre_o, *pre_m, *pre_l;
  // the plan, written by prefix_kernel's first CTA for the join
  int32_t* entry_at;      // [num_seqs] the entry's first row among its group's
  int32_t* group_work;    // [num_groups + 1] units of work before group g
  int32_t* group_vec;     // [num_groups + 1] vectors of one KV head before group g
  int splits, pre_ctas;
};

constexpr size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

struct Layout {
  size_t own_o, own_m, own_l, pre_o, pre_m, pre_l, entry_at, group_work, group_vec, total;
};

// Vectors of the prefixes' parts: every vector once, and 256 more for each CTA (see prefix_offset).
inline long long prefix_part_vectors(long long max_rows, int nh, int ctas) { return max_rows * nh + 256LL * (ctas + 1); }

inline Layout layout_of(long long max_rows, int num_seqs, int num_groups, int nh, int splits, int ctas) {
  Layout l;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += align256(bytes);
    return p;
  };
  const size_t own = (size_t)splits * max_rows * nh;
  const size_t pre = num_groups > 0 ? (size_t)prefix_part_vectors(max_rows, nh, ctas) : 0;
  l.own_o = take(own * D * 4);
  l.own_m = take(own * 4);
  l.own_l = take(own * 4);
  l.pre_o = take(pre * D * 4);
  l.pre_m = take(pre * 4);
  l.pre_l = take(pre * 4);
  l.entry_at = take((size_t)num_seqs * 4);
  l.group_work = take(((size_t)num_groups + 1) * 4);
  l.group_vec = take(((size_t)num_groups + 1) * 4);
  l.total = at;
  return l;
}

// ---------------------------------------------------------------- entries and groups
struct Entry {
  int rows, start, group;  // rows 0: nothing to do; group -1: no shared prefix
};

// Entry b as every kernel of the call sees it. Rows outside the host's bounds are reported and left
// out; a group is taken only if the entry's first row (its positions ascend) sees its whole prefix.
__device__ __forceinline__ Entry entry_of(const ne_rows& rows, const ne_prefix_groups& groups, int b, int* status) {
  Entry e{rows.q_len[b], rows.q_start[b], -1};
  const int g = groups.num_groups > 0 ? groups.entry_group[b] : -1;
  if (e.rows <= 0) return Entry{0, 0, -1};
  if (e.rows > rows.max_q_len || e.start < 0 || e.start > rows.max_rows - e.rows) {
    report(status, NE_DEV_BAD_SLOT);
    return Entry{0, 0, -1};
  }
  const int first = rows.positions[e.start];
  if (g >= 0 && g < groups.num_groups) {
    const int blocks = groups.prefix_blocks[g];
    if (blocks > 0 && blocks <= min(rows.block_table_stride, groups.max_prefix_blocks) && first >= blocks * 16 - 1) e.group = g;
  }
  return e;
}

__device__ __forceinline__ const int32_t* table_of(const ne_rows& rows, int b) {
  return rows.block_tables + (long long)(rows.table_index ? rows.table_index[b] : b) * rows.block_table_stride;
}

// The larger value; NaN if one is.
__device__ __forceinline__ float max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// ---------------------------------------------------------------- prefixes: the division of the work
// A group's vectors of one KV head are cut into items of up to 256: one or two query tiles, which share
// every tile of 128 keys. A key tile costs an item 3 units of work with one query tile and 4 with two
// (measured, bf16: 3,000 and 4,000 cycles). An int8 pool is divided by the same units although its tiles take
// 6,900 and 7,400: there a share of single query tiles takes up to a quarter longer than one of pairs. The
// units of all (group, head, item) in turn are divided evenly over the CTAs: CTA c does the key tiles that
// start in its ceil(W / CTAs) units from c ceil(W / CTAs) on.
__device__ __forceinline__ int key_tiles(int blocks) { return (blocks + 7) / 8; }
__device__ __forceinline__ int item_units(int vec) { return vec > TILE ? 4 : 3; }
// units of one KV head
__device__ __forceinline__ int head_work(int vec, int blocks) {
  const int rest = vec % 256;
  return key_tiles(blocks) * (4 * (vec / 256) + (rest ? item_units(rest) : 0));
}
// Where the part of (CTA c, item) lies: behind the vectors of the items before it and 256 for each CTA
// before it; a part has at most 256, so that consecutive ones do not overlap.
__device__ __forceinline__ long long prefix_offset(long long vec_at, int nkv, int h, int vec, int item, int cta) {
  return vec_at * nkv + (long long)h * vec + 256LL * item + 256LL * cta;
}

// ---------------------------------------------------------------- the join of a vector's parts
// A warp's running sums of one query vector: four dimensions a lane.
struct Sums {
  float m = -INFINITY, l = 0.f;
  float4 o = {0.f, 0.f, 0.f, 0.f};

  // Up to 32 parts, lane p's at position ``at`` of (po, m, l); m -inf: an empty part, whose sums were
  // never written. Every lane reads its part's m and l at once, then all lanes each part's values.
  __device__ __forceinline__ void add(const float* po, float pm, float pl, long long at, int count) {
    const int lane = threadIdx.x & 31;
    float top = pm;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = max2(top, __shfl_xor_sync(ALL, top, x));
    const float mn = max2(m, top);
    if (mn == NEG_INF) return;
    const float keep = m == NEG_INF ? 0.f : exp2f(m - mn), f = pm == NEG_INF ? 0.f : exp2f(pm - mn);
    float sum = pm == NEG_INF ? 0.f : f * pl;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(ALL, sum, x);
    l = l * keep + sum;
    m = mn;
    o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
#pragma unroll 4
    for (int p = 0; p < count; ++p) {
      const float fp = __shfl_sync(ALL, f, p);
      const long long ap = __shfl_sync(ALL, at, p);
      if (fp == 0.f) continue;
      const float4 y = *reinterpret_cast<const float4*>(po + ap * D + 4 * lane);
      o = make_float4(o.x + fp * y.x, o.y + fp * y.y, o.z + fp * y.z, o.w + fp * y.w);
    }
  }
  __device__ __forceinline__ void store(__nv_bfloat16* out) const {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // (l is 0 only for a row that sees no key; NaN stays NaN)
    __nv_bfloat162 y[2] = {__floats2bfloat162_rn(l == 0.f ? 0.f : o.x * inv, l == 0.f ? 0.f : o.y * inv),
                           __floats2bfloat162_rn(l == 0.f ? 0.f : o.z * inv, l == 0.f ? 0.f : o.w * inv)};
    *reinterpret_cast<uint2*>(out + 4 * (threadIdx.x & 31)) = *reinterpret_cast<uint2*>(y);
  }
};

// Adds the prefix parts of query head ``h * G + hq`` of row ``j`` of entry b, whose prefix has ``blocks``.
__device__ __forceinline__ void add_prefix(Sums& sums, const Parts& parts, int num_groups, int g, int blocks, int b,
                                           int j, int h, int hq, int G, int nkv) {
  const int work = parts.group_work[num_groups], tiles = key_tiles(blocks);
  const int vec_at = parts.group_vec[g], vec = parts.group_vec[g + 1] - vec_at;
  const int v = (parts.entry_at[b] + j) * G + hq, item = v / 256;
  if (work == 0) return;
  const int nv = min(256, vec - 256 * item), u = item_units(nv), per = (work + parts.pre_ctas - 1) / parts.pre_ctas;
  // the CTAs whose units meet the item's
  const int from = parts.group_work[g] + h * head_work(vec, blocks) + 4 * tiles * item, to = from + u * tiles;
  const long long at0 = prefix_offset(vec_at, nkv, h, vec, item, 0) + v - 256 * item;
  for (int c0 = from / per; c0 * per < to; c0 += 32) {
    const int c = c0 + (threadIdx.x & 31);
    const int count = min(32, (to - c0 * per + per - 1) / per);
    // (a CTA does the key tiles whose first unit is among its own)
    const int first = max(c * per - from, 0) + u - 1, last = (c + 1) * per - from + u - 1;
    const bool has = c * per < to && first / u < min(tiles, last / u);
    const long long at = at0 + 256LL * c;
    sums.add(parts.pre_o, has ? parts.pre_m[at] : NEG_INF, has ? parts.pre_l[at] : 0.f, at, count);
  }
}

// ---------------------------------------------------------------- own tokens
// One 16-token block (logical index kb) against the tile, as tile_block, but values at masked keys do
// not reach the sums whatever they are, and an int8 block holds its integers as they are: the K scale
// (``scales``: lane t token t's, lane 16 + t its V scale) multiplies the scores, the V scale the
// weights, both in fp32. The weights are rounded to bf16 for the product with V (2^-8 of each at most), as
// tile_block rounds them, since the tensor cores take both operands in V's type; their sum is of the fp32 ones.
template <bool INT8>
__device__ __forceinline__ void own_block(TileState& ts, uint32_t k_s, uint32_t v_s, int kb, uint32_t scales,
                                          int lane) {
  float s[2][4];
  float mx[2] = {NEG_INF, NEG_INF};
  bool masked = false;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; kk += 2) {
      uint32_t b[4];
      const int tok = 8 * j + (lane & 7);
      const int col = 16 * kk + 8 * (lane >> 3);
      ldsm_x4(b, kv_addr<false>(k_s, tok, col));
      mma16816(s[j], ts.qa[kk], b[0], b[1]);
      mma16816(s[j], ts.qa[kk + 1], b[2], b[3]);
    }
    float ks[2] = {SCALE_LOG2, SCALE_LOG2};
    if (INT8) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
        ks[x] *= __uint_as_float(__shfl_sync(ALL, scales, 8 * j + 2 * (lane & 3) + x) << 16);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = e >> 1;
      const int key = kb * 16 + 8 * j + 2 * (lane & 3) + (e & 1);
      float v = s[j][e] * ks[e & 1];
      if (key > ts.pos[r]) {
        v = NEG_INF;
        masked |= ts.pos[r] >= 0;  // (a row without keys has no sums to keep clean)
      }
      s[j][e] = v;
      mx[r] = max2(mx[r], v);
    }
  }
  float corr[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    mx[r] = max2(mx[r], __shfl_xor_sync(ALL, mx[r], 1));
    mx[r] = max2(mx[r], __shfl_xor_sync(ALL, mx[r], 2));
    const float m_new = max2(ts.m[r], mx[r]);
    corr[r] = (m_new == NEG_INF || ts.m[r] == NEG_INF) ? (m_new == NEG_INF ? 1.f : 0.f) : exp2f(ts.m[r] - m_new);
    ts.m[r] = m_new;
  }
  float psum[2] = {0.f, 0.f}, p[2][4];
  uint32_t pa[4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = e >> 1;
      p[j][e] = (s[j][e] == NEG_INF) ? 0.f : exp2f(s[j][e] - ts.m[r]);
      psum[r] += p[j][e];
    }
    if (INT8) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float vs = __uint_as_float(__shfl_sync(ALL, scales, 16 + 8 * j + 2 * (lane & 3) + (e & 1)) << 16);
        p[j][e] = (s[j][e] == NEG_INF) ? 0.f : p[j][e] * vs;
      }
    }
    pa[2 * j] = pack_bf16(p[j][0], p[j][1]);
    pa[2 * j + 1] = pack_bf16(p[j][2], p[j][3]);
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    psum[r] += __shfl_xor_sync(ALL, psum[r], 1);
    psum[r] += __shfl_xor_sync(ALL, psum[r], 2);
    ts.l[r] = ts.l[r] * corr[r] + psum[r];
  }
  if (__any_sync(ALL, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      ts.o[t][0] *= corr[0];
      ts.o[t][1] *= corr[0];
      ts.o[t][2] *= corr[1];
      ts.o[t][3] *= corr[1];
    }
  }
  // a block with masked keys (the last one or two of an entry): 0 x inf or 0 x NaN must stay out
  bool plain = true;
  if (!INT8 && __any_sync(ALL, masked)) {
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int x = lane + 32 * i;  // 16 tokens x 16 chunks of 8 values
      uint32_t w[4];
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "r"(kv_addr<false>(v_s, x >> 4, 8 * (x & 15))));
#pragma unroll
      for (int y = 0; y < 4; ++y)
        odd |= (w[y] & 0x7F80u) == 0x7F80u || (w[y] & 0x7F800000u) == 0x7F800000u;
    }
    plain = !__any_sync(ALL, odd);
  }
  if (plain) {
#pragma unroll
    for (int t = 0; t < 16; t += 2) {
      uint32_t b[4];
      const int tok = (lane & 7) + 8 * ((lane >> 3) & 1);
      const int col = 8 * t + 8 * (lane >> 4);
      ldsm_x4_t(b, kv_addr<false>(v_s, tok, col));
      mma16816(ts.o[t], pa, b[0], b[1]);
      mma16816(ts.o[t + 1], pa, b[2], b[3]);
    }
    return;
  }
#pragma unroll
  for (int tok = 0; tok < 16; ++tok) {  // (seldom: some value of the block is infinite or NaN)
    const int from = (lane & ~3) | ((tok & 7) >> 1);
    float w[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) w[r] = bf16r(__shfl_sync(ALL, p[tok >> 3][2 * r + (tok & 1)], from));
    const int key = kb * 16 + tok;
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      uint32_t v;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(kv_addr<false>(v_s, tok, 8 * t) + 4 * (lane & 3)));
      const float v0 = __uint_as_float(v << 16), v1 = __uint_as_float(v & 0xFFFF0000u);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (key > ts.pos[r]) continue;
        ts.o[t][2 * r] += w[r] * v0;
        ts.o[t][2 * r + 1] += w[r] * v1;
      }
    }
  }
}

// NW groups of NT warps: group w takes every NW-th block of the split into two cp.async stages of its
// own, its warp t serves query tile t, and the groups merge their sums at the end.
template <int NW, int NT>
constexpr size_t own_smem() {
  return (size_t)NT * BLOCK_BYTES + 128 + (size_t)NW * 4 * BLOCK_BYTES;
}
static_assert((2 * 4 * 16 * D + 2 * 2 * 4 * 16) * 4 <= 4 * 4 * BLOCK_BYTES, "merge area");

// Each block is read once per CTA, a CTA's first loads go out before its query tile. Bound by the latency
// of a warp's own chain: a block takes it 1,300 to 1,700 cycles (QK products, maximum, weights, PV) and
// 600 to 900 to issue its loads, for which it then waits 60 at most; the CTA's first loads come 6,000
// cycles after its start (entry, positions, table). 256 entries of 100 own tokens on average and 8 KV heads,
// alone and from DRAM: 39 us, 115 MB. Three or four stages a warp, two blocks a softmax step, heads as the
// fastest grid axis, and CTAs beside prefix_kernel's (which then slows as much) were measured: none is faster.
// Spills, by ptxas, in the variants of two query tiles alone (128 registers): bf16 64 bytes stored and 56 loaded,
// int8 144 and 104.
template <bool INT8, int NW, int NT>
__global__ void __launch_bounds__(32 * NW * NT, NT == 2 ? 2 : NW == 8 ? 1 : NW == 4 ? 3 : 5)
    own_tokens_kernel(const __nv_bfloat16* __restrict__ q, const void* __restrict__ kc, const void* __restrict__ vc,
                      const __nv_bfloat16* __restrict__ ks, const __nv_bfloat16* __restrict__ vs, ne_rows rows,
                      ne_prefix_groups groups, int nh, int nkv, long long num_cache_slots, Parts parts, int chunks,
                      int late_wait, int* status) {
  // behind prefix_kernel, whose CTAs let this launch start only after they waited for the launch
  // before them, no input is still being written; the wait for that kernel itself comes at the end
  if (!late_wait) pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t smem[];
  const int b = blockIdx.x, h = blockIdx.y, chunk = blockIdx.z % chunks, split = blockIdx.z / chunks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = warp % NW, tile = warp / NW;
  const Entry e = entry_of(rows, groups, b, tid == 0 && chunk == 0 && h == 0 && split == 0 ? status : nullptr);
  Ctx c{};
  c.G = nh / nkv;
  c.nvec = e.rows * c.G;
  const int v_base = 16 * NT * chunk;
  if (v_base >= c.nvec) {
    pdl_wait();
    return;
  }
  c.q = q;
  c.kc = kc;
  c.vc = vc;
  c.ks = ks;
  c.vs = vs;
  c.table = table_of(rows, b);
  c.nh = nh;
  c.nkv = nkv;
  c.h = h;
  c.r0 = e.start;
  c.num_cache_slots = num_cache_slots;
  c.status = status;
  uint8_t* q_s = smem;
  int* spos = reinterpret_cast<int*>(smem + NT * BLOCK_BYTES);
  uint8_t* buf = smem + NT * BLOCK_BYTES + 128;
  const uint32_t wbuf = smem_u32(buf) + group * 4 * BLOCK_BYTES;
  const int v_end = min(c.nvec, v_base + 16 * NT);
  const int last = rows.positions[c.r0 + (v_end - 1) / c.G];  // the chunk's last row sees the most
  const int nblk = last >= 0 ? last / 16 + 1 : 0;
  const int kb_first = e.group >= 0 ? groups.prefix_blocks[e.group] : 0;
  const int n = max(0, nblk - kb_first), per_split = (n + parts.splits - 1) / parts.splits;
  const int kb0 = kb_first + split * per_split, kb1 = min(nblk, kb0 + per_split);
  const int stride = rows.block_table_stride;
  auto group_sync = [&] {
    if (NT == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * NT) : "memory");
  };
  // this group's blocks kb0 + group + NW j; the table entries of 32 of them in the lanes of a register
  const int count = kb0 + group < kb1 ? (kb1 - kb0 - group + NW - 1) / NW : 0;
  auto table_chunk = [&](int j0) -> int {
    const int kb = kb0 + group + NW * (j0 + lane);
    return kb < kb1 && kb < stride ? c.table[kb] : -1;
  };
  int tbl = table_chunk(0);
  auto block_at = [&](int j) -> long long {  // (warp-uniform; an id that names no block is reported)
    if ((j & 31) == 0 && j > 0) tbl = table_chunk(j);
    return checked_block(c, __shfl_sync(ALL, tbl, j & 31));
  };
  uint32_t scales = 0, next_scales = 0;
  auto stage = [&](int j, long long blk) {
    if (blk >= 0) {
      if (INT8) {
        if (tile == 0) stage_raw_int8(c, blk, wbuf + (j & 1) * 4096, lane);
        next_scales = load_scales_int8(c, blk, lane);
      } else {
        const uint32_t at = wbuf + (j & 1) * 2 * BLOCK_BYTES;
        stage_block<false>(c, blk, at, at + BLOCK_BYTES, lane + 32 * tile, 32 * NT);
      }
    }
    cp_commit();
  };
  long long blk = count > 0 ? block_at(0) : -1;
  stage(0, blk);
  if (tid < 16 * NT) spos[tid] = v_base + tid < c.nvec ? rows.positions[c.r0 + (v_base + tid) / c.G] : -1;
  {  // the query tiles: 16 chunks of 16 bytes a vector, every load issued before the first store
    constexpr int PER = 256 * NT / (32 * NW * NT);
    uint4 x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int v = v_base + ((tid + i * 32 * NW * NT) >> 4), ch = tid & 15;
      x[i] = make_uint4(0, 0, 0, 0);
      if (v < c.nvec)
        x[i] = *reinterpret_cast<const uint4*>(c.q + ((long long)(c.r0 + v / c.G) * c.nh + c.h * c.G + v % c.G) * D + ch * 8);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      *reinterpret_cast<uint4*>(q_s + ((tid + i * 32 * NW * NT) >> 4) * ROW_BYTES + (tid & 15) * 16) = x[i];
  }
  __syncthreads();
  TileState ts;
  tile_init(ts, smem_u32(q_s) + tile * BLOCK_BYTES, spos + 16 * tile, lane);
  for (int j = 0; j < count; ++j) {
    scales = next_scales;
    const long long next = j + 1 < count ? block_at(j + 1) : -1;
    stage(j + 1, next);
    cp_wait<1>();
    group_sync();
    if (blk >= 0) {
      const int kb = kb0 + group + NW * j;
      if (INT8) {  // (scale 1: the integers, exact in bf16; two warps convert a half each)
        const uint32_t raw = wbuf + (j & 1) * 4096, kv = wbuf + 8192;
        if (tile == 0) convert_half_int8(raw, kv, 0x3F80u, 0, lane);
        if (tile == NT - 1) convert_half_int8(raw + 2048, kv + BLOCK_BYTES, 0x3F80u, 16, lane);
        group_sync();
        own_block<true>(ts, kv, kv + BLOCK_BYTES, kb, scales, lane);
      } else {
        const uint32_t at = wbuf + (j & 1) * 2 * BLOCK_BYTES;
        own_block<false>(ts, at, at + BLOCK_BYTES, kb, 0u, lane);
      }
    }
    group_sync();
    blk = next;
  }
  cp_wait<0>();
  __syncthreads();
  float* mo = reinterpret_cast<float*>(buf);  // [NT][NW][16][128]
  float* mm = mo + NT * NW * 16 * D;          // [NT][NW][16]
  float* ml = mm + NT * NW * 16;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int at = warp * 16 + (lane >> 2) + 8 * r;
#pragma unroll
    for (int t = 0; t < 16; ++t)
      *reinterpret_cast<float2*>(&mo[at * D + 8 * t + 2 * (lane & 3)]) = make_float2(ts.o[t][2 * r], ts.o[t][2 * r + 1]);
    if ((lane & 3) == 0) {
      mm[at] = ts.m[r];
      ml[at] = ts.l[r];
    }
  }
  __syncthreads();
  // a warp per vector: four dimensions a lane
  for (int x = warp; x < v_end - v_base; x += NW * NT) {
    const int at = (x >> 4) * NW * 16 + (x & 15);
    float m = mm[at];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = max2(m, mm[at + 16 * w]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = mm[at + 16 * w], f = mw == NEG_INF ? 0.f : exp2f(mw - m);
      const float4 y = *reinterpret_cast<const float4*>(&mo[(at + 16 * w) * D + 4 * lane]);
      if (mw == NEG_INF) continue;  // (a group without blocks)
      l += f * ml[at + 16 * w];
      o = make_float4(o.x + f * y.x, o.y + f * y.y, o.z + f * y.z, o.w + f * y.w);
    }
    const int row = c.r0 + (v_base + x) / c.G, head = h * c.G + (v_base + x) % c.G;
    const long long to = ((long long)split * rows.max_rows + row) * nh + head;
    *reinterpret_cast<float4*>(parts.own_o + to * D + 4 * lane) = o;
    if (lane == 0) {
      parts.own_m[to] = m;
      parts.own_l[to] = l;
    }
  }
  pdl_wait();  // (no launch behind this one sees it complete before prefix_kernel is)
}

// ---------------------------------------------------------------- prefixes: the tensor-core kernel
// two softmax warpgroups; a load warp, two MMA warps, one idle; for an int8 pool four warps that load and
// convert (128 registers a thread then; other splits of the registers were measured and are slower)
constexpr int pre_threads(bool int8) { return int8 ? 512 : 384; }
constexpr int SLOT_BYTES = TILE * D * 2;   // one K or V tile: two halves of 64 dimensions, rows of 128 B
constexpr int RING = 4;
constexpr int HALF = TILE / 2;             // keys of a softmax step
constexpr int TMEM_COLS = 512;             // two halves of S (P in the same columns) and O for each query tile
constexpr int POLY_PAIRS = 3;              // of 8 pairs of weights, those whose 2^x runs on the FMA pipe
constexpr float RESCALE = 8.f;             // (log2) how far scores may pass the reference before it moves

struct alignas(16) PrePlan {
  uint32_t key[MAX_SEQS];                  // rows << 12 | group + 1 (0: none)
  int start[MAX_SEQS], at[MAX_SEQS];       // the entry's first row; its first row among its group's
  short member[MAX_SEQS];                  // the groups' entries in order, group by group
  int group_first[MAX_SEQS];               // the first of the group's members
  int work[MAX_SEQS + 1], vec[MAX_SEQS + 1];        // units, and vectors of one KV head, before the group
  int blocks[MAX_SEQS];                    // prefix_blocks
  int members;
};
struct alignas(16) PreShared {
  uint64_t full[RING], empty[RING], s_full[2][2], p_ready[2][2], o_done[2][2], q_ready[2];
  uint32_t tmem;
  volatile int abort_flag;
  uint32_t valid[RING];                    // valid blocks of the tile in a slot
  // int8: K scales (times log2(e) / sqrt(128)) and V scales of the tile whose V is in slot 1 or 3
  alignas(16) float scale[2][2][TILE];
};
constexpr size_t PRE_SMEM = 1024 + 2 * SLOT_BYTES + RING * SLOT_BYTES + sizeof(PrePlan) + sizeof(PreShared);
static_assert(PRE_SMEM <= 232448, "shared memory of one CTA");

// D[tmem] (+)= A[tmem] B[smem]: the weights (bf16 pairs, a row per lane) times a V tile.
__device__ __forceinline__ void tc_mma_bf16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// V as the B operand [keys][dimensions], dimensions contiguous: 64-dimension columns 16 KB apart, groups
// of eight keys 1024 B apart, 128-byte swizzle.
__device__ __forceinline__ uint64_t desc_v(uint32_t smem_addr) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)((SLOT_BYTES / 2) >> 4) << 16) |
         ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
constexpr uint32_t IDESC_QK = idesc_bf16_f32(TILE, HALF);
constexpr uint32_t IDESC_PV = idesc_bf16_f32(TILE, D) | (1u << 16);  // B with its N dimension contiguous

__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^t for two t up to 126 (0 below 2^-127, as the special-function one flushes), on the FMA pipe beside the special-function one:
// t = n + f, n = rint(t) read off the low bits of t + 1.5 x 2^23, and 2^f on [-1/2, 1/2] by the cubic
// whose largest relative error is least (7.5e-5, a fiftieth of the 2^-8 by which the rounding of the weight to
// bf16 may be off next).
__device__ __forceinline__ void ex2_poly(uint64_t t2, float& a, float& b) {
  unpack2(t2, a, b);
  t2 = pack2(fmaxf(a, -127.f), fmaxf(b, -127.f));
  constexpr float MAGIC = 12582912.f;
  constexpr float C0 = 0.99992806f, C1 = 0.69326097f, C2 = 0.24261113f, C3 = 0.05517165f;
  const uint64_t n2 = add2(t2, pack2(MAGIC, MAGIC));
  const uint64_t f2 = fma2(add2(n2, pack2(-MAGIC, -MAGIC)), pack2(-1.f, -1.f), t2);
  uint64_t y2 = fma2(f2, pack2(C3, C3), pack2(C2, C2));
  y2 = fma2(y2, f2, pack2(C1, C1));
  y2 = fma2(y2, f2, pack2(C0, C0));
  float na, nb;
  unpack2(n2, na, nb);
  unpack2(y2, a, b);
  // (an exponent below the smallest leaves the integer negative)
  a = __int_as_float(max(__float_as_int(a) + (__float_as_int(na) << 23), 0));
  b = __int_as_float(max(__float_as_int(b) + (__float_as_int(nb) << 23), 0));
}

// A CTA's part of one item: vectors [v0, v0 + nv) of (group, head), key tiles [t0, t1).
struct Segment {
  int group, h, item, v0, nv, t0, t1;
};

// Walks the segments of a CTA in order; every role walks them for itself.
struct Walk {
  const PrePlan* plan;
  int groups, nkv, G;
  int lo, hi;               // the CTA's units
  int g, h, item, at;       // the current item, and the units before it

  __device__ Walk(const PrePlan* p, const ne_prefix_groups& pg, int nkv_, int G_, int per)
      : plan(p), groups(pg.num_groups), nkv(nkv_), G(G_) {
    const int work = p->work[groups];
    lo = min(work, (int)blockIdx.x * per);
    hi = min(work, lo + per);
    int a = 0, b = groups;
    while (a < b) {  // the last group whose work starts at or before lo
      const int mid = (a + b + 1) >> 1;
      if (p->work[mid] <= lo) a = mid;
      else b = mid - 1;
    }
    g = min(a, max(groups - 1, 0));
    h = 0;
    item = 0;
    at = p->work[g];
    if (lo < hi) {
      const int vec = p->vec[g + 1] - p->vec[g], blocks = plan->blocks[g];
      const int hw = head_work(vec, blocks);
      h = (lo - at) / hw;
      at += h * hw;
      const int units = 4 * key_tiles(blocks);
      item = min((lo - at) / units, (vec - 1) / 256);
      at += item * units;
    }
  }
  __device__ bool next(Segment& s) {
    while (at < hi && lo < hi) {
      const int vec = plan->vec[g + 1] - plan->vec[g];
      if (vec == 0) {  // a group without rows has no work
        ++g;
        h = item = 0;
        if (g >= groups) return false;
        at = plan->work[g];
        continue;
      }
      const int tiles = key_tiles(plan->blocks[g]);
      const int nv = min(256, vec - 256 * item), u = item_units(nv);
      const int from = max(lo - at, 0), to = hi - at;
      const int t0 = (from + u - 1) / u, t1 = min(tiles, (to + u - 1) / u);
      s = Segment{g, h, item, 256 * item, nv, t0, t1};
      at += u * tiles;
      if (256 * (item + 1) < vec) {
        ++item;
      } else {
        item = 0;
        if (++h == nkv) {
          h = 0;
          ++g;
          if (g >= groups) at = hi;  // the end of all work
        }
      }
      if (t0 < t1) return true;
    }
    return false;
  }
};

// Two int8 values of ``word`` as bf16, exact: with its sign bit s and the seven others v, a value is
// (128 + v) - (s ? 256 : 128), both of which are bf16 numbers with the byte as their low bits.
__device__ __forceinline__ uint32_t exact_pair(uint32_t word, uint32_t sel) {
  const uint32_t p = __byte_perm(word, 0x43434343u, sel);
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(p & 0x437F437Fu), "r"(p & 0x43804380u));
  return d;
}

// Per segment, S = Q K^T (Q, K in shared memory, S in TMEM), P = 2^(S - ref) in S's columns, O += P V (P from
// TMEM), 64 keys a step so that the tensor cores work on one half's products while the other's weights
// are computed; O is rescaled only when the reference moves by more than 2^8. K and V tiles come through
// a ring of four slots by 3-D tensor loads of the 16-token pages (int8: loaded and converted by four
// warps). P is rounded to bf16 (the tensor cores take P and V in one type; l sums the unrounded weights): 2^-8
// of a weight at most, as the ordinary attention; int8: after the V scale, keys and values unrounded.
// Bound by the latency of the softmax's chain, one warp a scheduler and query tile: 16,384 shared tokens x 1,280
// vectors x 8 KV heads (85.9 GFLOP) take 103 us, 834 TFLOP/s, with the tensor pipe busy 47% of the time (a
// pair tile's products alone are 2,048 of its 4,000 cycles) and 1.8 of 4 issue slots used; 3 of 8 powers of two
// run on the FMA pipe. int8: 6,900 cycles a tile, of which a shorter softmax took 2,000 (steps of 32 keys, 9,100
// before), so that chain counts there too; how much the conversion beside it does was not measured. A CTA's
// fixed costs are about 15,000 cycles: plan 6,000, first query tile 2,700, epilogue 3,500 a segment. Spills, by
// ptxas: bf16 28 bytes stored and 44 loaded at 168 registers, int8 80 and 132 at 128.
template <bool INT8>
__global__ void __launch_bounds__(pre_threads(INT8), 1)
    prefix_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                  const int8_t* __restrict__ kc, const int8_t* __restrict__ vc, const __nv_bfloat16* __restrict__ ks,
                  const __nv_bfloat16* __restrict__ vs, const __nv_bfloat16* __restrict__ q, ne_rows rows,
                  ne_prefix_groups groups, int nh, int nkv, long long num_cache_slots, Parts parts, int* status) {
  constexpr int THREADS_P = pre_threads(INT8);
  pdl_wait();
  pdl_trigger();  // (after the wait: own_tokens_kernel relies on it)
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_s = smem;                              // [2 streams] query tiles
  uint8_t* ring = smem + 2 * SLOT_BYTES;            // [RING] K and V tiles
  PrePlan& plan = *reinterpret_cast<PrePlan*>(ring + RING * SLOT_BYTES);
  PreShared& sh = *reinterpret_cast<PreShared*>(reinterpret_cast<uint8_t*>(&plan) + sizeof(PrePlan));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = nh / nkv, n = rows.num_seqs, ng = groups.num_groups;

  // ---- barriers, tensor memory, and the plan
  if (tid == 0) {
    for (int i = 0; i < RING; ++i) {
      mbar_init(&sh.full[i], INT8 ? 64 : 1);  // (a tensor load's thread, or the two warps that convert)
      mbar_init(&sh.empty[i], 2);  // a release by each query tile's products
    }
    for (int s = 0; s < 2; ++s) {
      for (int half = 0; half < 2; ++half) {
        mbar_init(&sh.s_full[s][half], 1);
        mbar_init(&sh.p_ready[s][half], 128);
        mbar_init(&sh.o_done[s][half], 1);
      }
      mbar_init(&sh.q_ready[s], 128);
    }
    sh.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(&sh.tmem, TMEM_COLS);
    tmem_relinquish();
  }
  for (int g = tid; g < ng; g += THREADS_P) {
    plan.vec[g] = 0;          // (rows, until they are summed)
    plan.group_first[g] = 0;  // (members, until their offsets are known)
    plan.blocks[g] = groups.prefix_blocks[g];
  }
  for (int b = tid; b < (n + 3 & ~3); b += THREADS_P) {
    const Entry e = b < n ? entry_of(rows, groups, b, nullptr) : Entry{0, 0, -1};  // (own_tokens_kernel reports)
    plan.start[b] = e.start;
    plan.key[b] = e.group >= 0 ? (uint32_t)e.rows << 12 | (uint32_t)(e.group + 1) : 0u;
  }
  __syncthreads();
  int rank[(MAX_SEQS + THREADS_P - 1) / THREADS_P];  // members of the group before the entry
#pragma unroll
  for (int i = 0; i < (MAX_SEQS + THREADS_P - 1) / THREADS_P; ++i) {
    const int b = tid + i * THREADS_P;
    rank[i] = 0;
    const uint32_t key = b < n ? plan.key[b] : 0u;
    if (key == 0u) continue;
    int before = 0;
    auto count = [&](uint32_t other, int x) {
      if (x < b && ((other ^ key) & 0xFFFu) == 0u) {
        before += other >> 12;
        ++rank[i];
      }
    };
    for (int x = 0; x < b; x += 4) {
      const uint4 k4 = *reinterpret_cast<const uint4*>(&plan.key[x]);
      count(k4.x, x);
      count(k4.y, x + 1);
      count(k4.z, x + 2);
      count(k4.w, x + 3);
    }
    plan.at[b] = before;
    const int g = (int)(key & 0xFFFu) - 1;
    atomicAdd(&plan.vec[g], (int)(key >> 12));
    atomicAdd(&plan.group_first[g], 1);
    if (blockIdx.x == 0) parts.entry_at[b] = before;
  }
  __syncthreads();
  if (warp == 0) {
    // (rows below 2^30 in all, whatever the entries say; work and vectors count only if they pass the test)
    int work = 0, taken = 0, members = 0;
    for (int g0 = 0; g0 < ng; g0 += 32) {
      const int g = g0 + lane;
      const int mine = g < ng ? plan.vec[g] : 0, count = g < ng ? plan.group_first[g] : 0;
      const int w = mine ? nkv * head_work(mine * G, plan.blocks[g]) : 0;
      int wi = w, vi = mine, mi = count;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(ALL, wi, o), c = __shfl_up_sync(ALL, vi, o), d = __shfl_up_sync(ALL, mi, o);
        if (lane >= o) {
          wi += a;
          vi += c;
          mi += d;
        }
      }
      if (g < ng) {
        plan.work[g] = work + wi - w;
        plan.vec[g] = (taken + vi - mine) * G;
        plan.group_first[g] = members + mi - count;
      }
      work += __shfl_sync(ALL, wi, 31);
      taken += __shfl_sync(ALL, vi, 31);
      members += __shfl_sync(ALL, mi, 31);
    }
    __syncwarp();
    if (taken > rows.max_rows) {  // entries that share rows: more parts than there is room for
      if (lane == 0) report(status, NE_DEV_BAD_SLOT);
      for (int g = lane; g < ng; g += 32) plan.work[g] = 0;
      work = 0;
    }
    if (lane == 0) {
      plan.work[ng] = work;
      plan.vec[ng] = taken * G;
      plan.members = members;
    }
    __syncwarp();
    if (blockIdx.x == 0)
      for (int g = lane; g <= ng; g += 32) {
        parts.group_work[g] = plan.work[g];
        parts.group_vec[g] = plan.vec[g];
      }
  }
  tc_fence_before();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < (MAX_SEQS + THREADS_P - 1) / THREADS_P; ++i) {
    const int b = tid + i * THREADS_P;
    if (b < n && plan.key[b]) plan.member[plan.group_first[(plan.key[b] & 0xFFFu) - 1] + rank[i]] = (short)b;
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const int per = (plan.work[ng] + gridDim.x - 1) / gridDim.x;
  Walk walk(&plan, groups, nkv, G, per);
  Segment sg;

  if (warp < 8) {
    // ------------------------------------------------------------ softmax of query tile s, a row per thread
    const int s = warp >> 2, row = tid & 127;
    const uint32_t lane_base = (uint32_t)(warp & 3) << 21;  // 32 rows x (1 << 16)
    const uint32_t t_s = tmem + lane_base + s * TILE, t_o = tmem + lane_base + 256 + s * D;
    uint8_t* my_q = q_s + s * SLOT_BYTES;
    uint32_t tiles_before = 0, slots_before = 0;  // key tiles of earlier segments: this warpgroup's, all
    while (walk.next(sg)) {
      const int tiles = sg.t1 - sg.t0;
      if (s == 1 && sg.nv <= TILE) {  // one query tile: the second warpgroup sits this segment out
        slots_before += tiles;
        continue;
      }
      // the query tile: vector v of the group is head v % G of the group's row v / G
      const int v = sg.v0 + s * TILE + row;
      const bool live = v < sg.v0 + sg.nv;
      {
        int at = -1;  // the row of q, in units of vectors
        if (live) {
          const int r = v / G;
          int a = plan.group_first[sg.group];
          int z = (sg.group + 1 < ng ? plan.group_first[sg.group + 1] : plan.members) - 1;
          while (a < z) {  // the last member whose rows start at or before r
            const int mid = (a + z + 1) >> 1;
            if (plan.at[plan.member[mid]] <= r) a = mid;
            else z = mid - 1;
          }
          const int b = plan.member[a];
          at = (plan.start[b] + r - plan.at[b]) * nh + sg.h * G + v % G;
        }
        // half a warp a vector: 16 bytes a lane
        const int ch = lane & 15;
        uint4 x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int from = __shfl_sync(ALL, at, 2 * i + (lane >> 4));
          x[i] = from >= 0 ? *reinterpret_cast<const uint4*>(q + (long long)from * D + 8 * ch) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = (warp & 3) * 32 + 2 * i + (lane >> 4);
          *reinterpret_cast<uint4*>(my_q + (ch >> 3) * (SLOT_BYTES / 2) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = x[i];
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&sh.q_ready[s]);
      float ref = NEG_INF, l = 0.f;
      bool ok = true;
      for (int j = 0; j < 2 * tiles; ++j) {  // 64 keys a step, S in two buffers: the next half's scores
        const int t = j >> 1, half = j & 1;  // are computed while this one's weights are
        ok = mbar_wait(&sh.s_full[s][half], (tiles_before + t) & 1u, &sh.abort_flag, status);
        tc_fence_after();
        // int8: 32 keys at a time, the second 32 loaded twice (their maximum, then their weights), for the
        // scales take registers and what is spilled does not fit what shared memory leaves of the L1 (64 at
        // a time spilled inside the step; 9,100 cycles a tile instead of 6,900)
        constexpr int KEYS = INT8 ? HALF / 2 : HALF;
        float x[KEYS];
        tmem_ld32_start(t_s + HALF * half + (INT8 ? KEYS : 0), x);
        if (!INT8) tmem_ld32_start(t_s + HALF * half + 32, x + 32 % KEYS);
        // the mask comes with the V tile (K's slot may be refilled by now)
        const uint32_t v_at = 2 * (slots_before + t) + 1;
        ok = ok && mbar_wait(&sh.full[v_at % RING], (v_at / RING) & 1u, &sh.abort_flag, status);
        const uint32_t valid = sh.valid[v_at % RING] >> (4 * half) & 0xFu;
        const float* scale_k = sh.scale[(v_at % RING) >> 1][0] + HALF * half;
        const float* scale_v = sh.scale[(v_at % RING) >> 1][1] + HALF * half;
        auto finish = [&](int k0) {  // the scores of keys k0 .. of the half have been asked for
          tmem_ld_wait();
          if (INT8) {
#pragma unroll
            for (int c = 0; c < KEYS; c += 4) {
              const float4 k4 = *reinterpret_cast<const float4*>(scale_k + k0 + c);
              unpack2(mul2(pack2(x[c], x[c + 1]), pack2(k4.x, k4.y)), x[c], x[c + 1]);
              unpack2(mul2(pack2(x[c + 2], x[c + 3]), pack2(k4.z, k4.w)), x[c + 2], x[c + 3]);
            }
          }
          if (valid != 0xFu) {
#pragma unroll
            for (int c = 0; c < KEYS; ++c)
              if (!(valid >> ((k0 + c) >> 4) & 1u)) x[c] = NEG_INF;
          }
        };
        auto largest = [&] {
          float mx[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) mx[i] = max3(x[i], x[8 + i], x[16 + i]);
#pragma unroll
          for (int c = 24; c + 16 <= KEYS; c += 16)
#pragma unroll
            for (int i = 0; i < 8; ++i) mx[i] = max3(mx[i], x[c + i], x[c + 8 + i]);
#pragma unroll
          for (int i = 0; i < 8; ++i) mx[i] = max2(mx[i], x[KEYS - 8 + i]);
          return max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), max2(mx[6], mx[7]));
        };
        float top;
        if (INT8) {
          finish(KEYS);
          top = largest();
          tmem_ld32_start(t_s + HALF * half, x);
          finish(0);
          top = max2(top, largest());
        } else {
          finish(0);
          top = largest() * SCALE_LOG2;
        }
        const bool odd = __any_sync(ALL, !(fabsf(top) < INFINITY));  // NaN or infinite scores among them
        // the reference moves only when the scores pass it by 2^8 (the sums stay far inside fp32)
        if (__any_sync(ALL, !(top <= ref + RESCALE))) {
          const float next = max2(ref, top);
          const float f = ref == NEG_INF ? 0.f : ex2(ref - next);
          ref = next;
          l *= f;
          if (t + half > 0) {  // O must hold the product of the step before, which may still run
            ok = ok && mbar_wait(&sh.o_done[s][half ^ 1], (tiles_before + t - 1 + half) & 1u, &sh.abort_flag, status);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              float o[32];
              tmem_ld32_start(t_o + 32 * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= f;
              tmem_st32(t_o + 32 * c, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        const float base = ref == NEG_INF ? 0.f : ref;
        const uint64_t scale2 = pack2(SCALE_LOG2, SCALE_LOG2), base2 = pack2(-base, -base);
        uint64_t sum[2] = {0ull, 0ull};  // (pairs of fp32 zeros)
        uint32_t p[KEYS / 2];
        auto weigh = [&](bool all, int k0) {
#pragma unroll
          for (int i = 0; i < KEYS / 2; ++i) {
            float a, b;
            const uint64_t x2 = pack2(x[2 * i], x[2 * i + 1]);
            const uint64_t t2 = INT8 ? add2(x2, base2) : fma2(x2, scale2, base2);  // (int8: scaled already)
            if (all || i % 8 >= POLY_PAIRS) {
              unpack2(t2, a, b);
              a = ex2(a);
              b = ex2(b);
            } else {
              ex2_poly(t2, a, b);
            }
            sum[i & 1] = add2(sum[i & 1], pack2(a, b));
            if (INT8) {
              const float2 v2 = *reinterpret_cast<const float2*>(scale_v + k0 + 2 * i);
              unpack2(mul2(pack2(a, b), pack2(v2.x, v2.y)), a, b);
            }
            p[i] = pack_bf16(a, b);
          }
        };
        if (odd) weigh(true, 0);
        else weigh(false, 0);
        if constexpr (INT8) {  // (the first keys' weights lie where their scores did)
          tmem_st16(t_s + HALF * half, p);
          tmem_ld32_start(t_s + HALF * half + KEYS, x);
          finish(KEYS);
          if (odd) weigh(true, KEYS);
          else weigh(false, KEYS);
          tmem_st16(t_s + HALF * half + KEYS / 2, p);
        } else {
          tmem_st32(t_s + HALF * half, p);
        }
        float s0, s1;
        unpack2(add2(sum[0], sum[1]), s0, s1);
        l += s0 + s1;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sh.p_ready[s][half]);
        if (!__all_sync(ALL, ok)) {
          ok = false;
          break;
        }
      }
      if (!ok) break;
      tiles_before += tiles;
      slots_before += tiles;
      // the part: unnormalised sums, and the reference and sum of their weights
      const long long part = prefix_offset(plan.vec[sg.group], nkv, sg.h, plan.vec[sg.group + 1] - plan.vec[sg.group],
                                           sg.item, blockIdx.x) + s * TILE;
      const long long at = part + row;
      ok = mbar_wait(&sh.o_done[s][1], (tiles_before - 1) & 1u, &sh.abort_flag, status);
      if (!__all_sync(ALL, ok)) break;
      tc_fence_after();
      // O through shared memory (the warp's own rows of the query tile, whose products are done), 64
      // dimensions at a time, so that half a warp writes 256 consecutive bytes
      const int r0 = (warp & 3) * 32, rows_live = min(32, sg.nv - s * TILE - r0);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float o[64];
        tmem_ld32_start(t_o + 64 * c, o);
        tmem_ld32_start(t_o + 64 * c + 32, o + 32);
        tmem_ld_wait();
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          *reinterpret_cast<float4*>(my_q + (i >> 3) * (SLOT_BYTES / 2) + row * 128 + (((i & 7) ^ (row & 7)) << 4)) =
              make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        __syncwarp();
        const int ch = lane & 15;
        for (int r = lane >> 4; r < rows_live; r += 2) {
          const float4 y = *reinterpret_cast<const float4*>(my_q + (ch >> 3) * (SLOT_BYTES / 2) + (r0 + r) * 128 +
                                                            (((ch & 7) ^ (r & 7)) << 4));
          *reinterpret_cast<float4*>(parts.pre_o + (part + r0 + r) * D + 64 * c + 4 * ch) = y;
        }
      }
      tc_fence_before();
      if (live) {
        parts.pre_m[at] = ref;
        parts.pre_l[at] = l;
      }
    }
  } else if (!INT8 && warp == 8 && elect_one()) {
    // ------------------------------------------------------------ loads, issued by one thread
    uint32_t load = 0;  // ring slots filled
    bool ok = true;
    while (ok && walk.next(sg)) {
      const int blocks = plan.blocks[sg.group];
      const int32_t* table = table_of(rows, plan.member[plan.group_first[sg.group]]);
      int next[8];  // the next tile's block ids, loaded a tile ahead
      auto look = [&](int t) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int kb = t * 8 + x;
          next[x] = t < sg.t1 && kb < blocks ? table[kb] : -1;
        }
      };
      look(sg.t0);
      for (int t = sg.t0; ok && t < sg.t1; ++t) {  // K0 V0 K1 V1 ..
        int id[8];
        uint32_t mask = 0;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          id[x] = next[x];
          if (id[x] >= 0 && ((long long)id[x] + 1) * 16 <= num_cache_slots - 1) mask |= 1u << x;
          else if (t * 8 + x < blocks) report(status, NE_DEV_BAD_SLOT);
        }
        look(t + 1);
        for (int is_v = 0; is_v < 2; ++is_v, ++load) {
          const int slot = load % RING;
          if (load >= RING) {
            ok = mbar_wait(&sh.empty[slot], (load / RING - 1) & 1u, &sh.abort_flag, status);
            if (!ok) break;
          }
          sh.valid[slot] = mask;
          mbar_arrive_expect_tx(&sh.full[slot], __popc(mask) * 4096);
          uint8_t* dst = ring + slot * SLOT_BYTES;
          const CUtensorMap* map = is_v ? &vmap : &kmap;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            if (!(mask >> x & 1u)) continue;
            tma_load_3d(dst + x * 2048, map, &sh.full[slot], 0, sg.h, id[x] * 16);
            tma_load_3d(dst + SLOT_BYTES / 2 + x * 2048, map, &sh.full[slot], 64, sg.h, id[x] * 16);
          }
        }
      }
    }
    // (given up: the loads in flight land before the CTA leaves; the wait is bounded as all are)
    if (!ok)
      for (uint32_t i = load > RING ? load - RING : 0; i < load; ++i)
        mbar_wait(&sh.full[i % RING], (i / RING) & 1u, nullptr, status);
  } else if ((warp == 9 || warp == 10) && elect_one()) {
    // ------------------------------------------------------------ products of query tile s, issued by one thread
    const int s = warp - 9;
    uint32_t base = 0, tiles_before = 0, q_phase = 0;  // (descriptor offsets: 16-byte units)
    const uint64_t q_desc = smem_desc_sw128(smem_u32(q_s) + s * SLOT_BYTES), k_desc = smem_desc_sw128(smem_u32(ring)),
                   v_desc = desc_v(smem_u32(ring));
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t phase) {
      ok = ok && mbar_wait(bar, phase & 1u, &sh.abort_flag, status);
      return ok;
    };
    auto full = [&](uint32_t at) { return wait(&sh.full[(base + at) % RING], (base + at) / RING); };
    auto scores = [&](int t, int half) {  // S = Q K^T of 64 keys
      const uint64_t kd = k_desc + ((base + 2 * t) % RING * SLOT_BYTES + half * HALF * 128 >> 4);
      const uint32_t d = tmem + s * TILE + half * HALF;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const uint32_t off = ((kk >> 2) * (SLOT_BYTES / 2) + (kk & 3) * 32) >> 4;
        tc_mma_bf16(d, q_desc + off, kd + off, IDESC_QK, kk > 0);
      }
      tc_commit(&sh.s_full[s][half]);
    };
    bool begun = false;                   // O holds a product of this segment
    auto values = [&](int t, int half) {  // O (+)= P V, the valid blocks only
      const uint32_t slot = (base + 2 * t + 1) % RING;
      const uint64_t vd = v_desc + (slot * SLOT_BYTES + half * 4 * 2048 >> 4);
      const uint32_t mask = sh.valid[slot] >> (4 * half) & 0xFu;
      const uint32_t d = tmem + 256 + s * D, a = tmem + s * TILE + half * HALF;
      if (mask == 0xFu) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          tc_mma_bf16_ta(d, a + 8 * kk, vd + (kk * 2048 >> 4), IDESC_PV, kk > 0 || begun);
        begun = true;
      } else {
        for (int kk = 0; kk < 4; ++kk) {
          if (!(mask >> kk & 1u)) continue;
          tc_mma_bf16_ta(d, a + 8 * kk, vd + (kk * 2048 >> 4), IDESC_PV, begun);
          begun = true;
        }
      }
      tc_commit(&sh.o_done[s][half]);
    };
    while (ok && walk.next(sg)) {
      const int tiles = sg.t1 - sg.t0;
      const bool both = sg.nv > TILE;
      auto release = [&](uint32_t at) { tc_commit(&sh.empty[(base + at) % RING]); };
      if (both || s == 0) {
        begun = false;
        if (!wait(&sh.q_ready[s], q_phase++) || !full(0)) break;
        tc_fence_after();
        scores(0, 0);
        scores(0, 1);
        release(0);
        for (int t = 0; ok && t < tiles; ++t) {
          if (!full(2 * t + 1) || !wait(&sh.p_ready[s][0], tiles_before + t)) break;
          tc_fence_after();
          values(t, 0);
          if (t + 1 < tiles) {
            if (!full(2 * t + 2)) break;
            scores(t + 1, 0);
          }
          if (!wait(&sh.p_ready[s][1], tiles_before + t)) break;
          tc_fence_after();
          values(t, 1);
          release(2 * t + 1);
          if (t + 1 < tiles) {
            scores(t + 1, 1);
            release(2 * t + 2);
          }
        }
        tiles_before += tiles;
      } else {
        // no second query tile: its thread still takes part in every slot's turn. (Left to run ahead, it
        // would wait for a slot two turns on, whose parity the turn before it already shows.)
        for (int at = 0; at < 2 * tiles; ++at) {
          if (!full(at)) break;
          mbar_arrive(&sh.empty[(base + at) % RING]);
        }
      }
      base += 2 * tiles;
    }
  } else if (INT8 && warp >= 12) {
    // ------------------------------------------------------------ int8 loads: two warps for K, two for V
    // A tile is 1024 pieces of 16 integers: thread t takes pieces t + 64 i, all loads issued before the
    // slot is free, and writes each as bf16 (exact) where a tensor load would have put it.
    const int is_v = (warp - 12) >> 1, t64 = tid & 63, ch = t64 & 7;
    const int8_t* pool = is_v ? vc : kc;
    uint32_t tile = 0;
    bool ok = true;
    while (ok && walk.next(sg)) {
      const int blocks = plan.blocks[sg.group];
      const int32_t* table = table_of(rows, plan.member[plan.group_first[sg.group]]);
      int next[8];  // the next tile's block ids, loaded a tile ahead
      auto look = [&](int t) {
#pragma unroll
        for (int b = 0; b < 8; ++b) next[b] = t < sg.t1 && t * 8 + b < blocks ? table[t * 8 + b] : -1;
      };
      look(sg.t0);
      for (int t = sg.t0; ok && t < sg.t1; ++t, ++tile) {
        const uint32_t load = 2 * tile + is_v;
        const int slot = load % RING;
        uint32_t mask = 0, bad = 0;
        uint4 x[16];
        long long own = -1;  // the block of keys 2 t64 and 2 t64 + 1, whose scales this thread brings
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const long long id = next[b];
          const bool in = id >= 0 && (id + 1) * 16 <= num_cache_slots - 1;
          mask |= (in ? 1u : 0u) << b;
          bad |= !in && t * 8 + b < blocks;
          const long long at = ((in ? id * 16 : 0) + (t64 >> 3)) * nkv + sg.h;
#pragma unroll
          for (int i = 2 * b; i < 2 * b + 2; ++i) {
            x[i] = make_uint4(0, 0, 0, 0);
            if (in) x[i] = *reinterpret_cast<const uint4*>(pool + (at + 8 * (i & 1) * nkv) * D + 16 * ch);
          }
          if (in && t64 >> 3 == b) own = id;
        }
        __nv_bfloat16 scale[4] = {};
        if (is_v && own >= 0) {
          const long long key = (own * 16 + (2 * t64 & 15)) * nkv + sg.h;
          scale[0] = ks[key];
          scale[1] = ks[key + nkv];
          scale[2] = vs[key];
          scale[3] = vs[key + nkv];
        }
        look(t + 1);
        if (bad && t64 == 0) report(status, NE_DEV_BAD_SLOT);
        if (load >= RING) {
          ok = mbar_wait(&sh.empty[slot], (load / RING - 1) & 1u, &sh.abort_flag, status);
          ok = __all_sync(ALL, ok);
          if (!ok) break;
        }
        uint8_t* dst = ring + slot * SLOT_BYTES;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = 8 * i + (t64 >> 3);
          const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
          uint32_t o[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            o[2 * k] = exact_pair(w[k], 0x4140u);
            o[2 * k + 1] = exact_pair(w[k], 0x4342u);
          }
          uint8_t* row = dst + (ch >> 2) * (SLOT_BYTES / 2) + key * 128;
          *reinterpret_cast<uint4*>(row + (((2 * ch & 7) ^ (key & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(row + (((2 * ch + 1 & 7) ^ (key & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        if (is_v) {
          *reinterpret_cast<float2*>(&sh.scale[slot >> 1][0][2 * t64]) =
              make_float2(__bfloat162float(scale[0]) * SCALE_LOG2, __bfloat162float(scale[1]) * SCALE_LOG2);
          *reinterpret_cast<float2*>(&sh.scale[slot >> 1][1][2 * t64]) =
              make_float2(__bfloat162float(scale[2]), __bfloat162float(scale[3]));
        }
        if (t64 == 0) sh.valid[slot] = mask;
        fence_proxy_async_smem();
        mbar_arrive(&sh.full[slot]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, TMEM_COLS);
}

// ---------------------------------------------------------------- the join
constexpr int JOIN_WARPS = 8;

// A warp per vector. Bound by latency: three loads in a row behind the wait (where the parts are,
// their sums of weights, their values), the inputs before it. 20,480 vectors of two to three parts (31 MB,
// which lie in L2 behind the other two launches): 21 us alone and from DRAM.
__global__ void __launch_bounds__(32 * JOIN_WARPS)
    join_kernel(__nv_bfloat16* __restrict__ out, ne_rows rows, ne_prefix_groups groups, int nh, int nkv, Parts parts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.y;
  const Entry e = entry_of(rows, groups, b, nullptr);
  const int x = blockIdx.x * JOIN_WARPS + warp, blocks = e.group >= 0 ? groups.prefix_blocks[e.group] : 0;
  pdl_prologue();
  if (x >= e.rows * nh) return;
  const int j = x / nh, head = x % nh, G = nh / nkv;
  const long long at = ((long long)lane * rows.max_rows + e.start + j) * nh + head;
  const bool has = lane < parts.splits;  // (at most 16 splits)
  Sums sums;
  sums.add(parts.own_o, has ? parts.own_m[at] : NEG_INF, has ? parts.own_l[at] : 0.f, at, parts.splits);
  if (e.group >= 0)
    add_prefix(sums, parts, groups.num_groups, e.group, blocks, b, j, head / G, head % G, G, nkv);
  sums.store(out + ((long long)(e.start + j) * nh + head) * D);
}

int device_sms() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Chunks of an entry's query vectors: one of up to 32, or as many of 32 as it takes.
int own_chunks(int max_q_len, int G) { return (int)(((long long)max_q_len * G + 31) / 32); }

// Splits of the entries' own tokens: one, unless the launch leaves most SMs idle and contexts are long
// (32 blocks a split at least, as attention_plan_splits).
int own_splits(int num_seqs, int nkv, int chunks, int max_context, int sms) {
  const long long ctas = (long long)num_seqs * nkv * chunks;
  long long splits = (2LL * sms + ctas - 1) / ctas;
  splits = std::min<long long>(splits, max_context / 16 / 32);
  return (int)std::max<long long>(1, std::min<long long>(splits, 16));
}

template <typename K>
bool allow_smem(K kernel, size_t bytes, bool (&done)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (!done[dev])
    done[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess;
  return done[dev];
}

bool heads_ok(int nh, int nkv) { return nkv > 0 && nh > 0 && nh % nkv == 0 && nh / nkv <= MAX_GROUP; }

}  // namespace

// Whether a launch within these bounds can run: the entries and groups that the plan's arrays have places for,
// the grids' limits, rows of an entry in 20 bits and units of work in 31, and the workspace.
int prefix_attention_fits(const ne_rows& rows, const ne_prefix_groups& groups, int nh, int nkv, size_t ws_bytes) {
  if (rows.num_seqs < 1 || rows.num_seqs > MAX_SEQS || groups.num_groups < 0 || groups.num_groups > MAX_SEQS ||
      rows.max_rows < 1 || rows.max_q_len < 1 || rows.max_context < 0 || groups.max_prefix_blocks < 0 ||
      !heads_ok(nh, nkv))
    return NE_ERR_INVALID;
  const int sms = device_sms(), chunks = own_chunks(rows.max_q_len, nh / nkv);
  const int splits = own_splits(rows.num_seqs, nkv, chunks, rows.max_context, sms);
  if (ws_bytes < layout_of(rows.max_rows, rows.num_seqs, groups.num_groups, nh, splits, sms).total)
    return NE_ERR_WORKSPACE;
  if ((long long)chunks * splits > 65535 || nkv > 65535 || rows.max_q_len >= (1 << 20) ||
      (long long)rows.max_rows * nh >= (1 << 29) ||
      ((long long)rows.max_rows * nh / TILE + 2LL * groups.num_groups * nkv + 2) * (groups.max_prefix_blocks / 8 + 1) >=
          (1 << 28))
    return NE_ERR_UNSUPPORTED;
  return NE_OK;
}

int launch_prefix_attention(const __nv_bfloat16* q, __nv_bfloat16* out, const void* k_cache, const void* v_cache,
                            const __nv_bfloat16* k_scale, const __nv_bfloat16* v_scale, int kv_int8,
                            const ne_rows& rows, ne_prefix_groups groups, int nh, int nkv, long long slots,
                            uint8_t* ws, size_t ws_bytes, int* status, cudaStream_t stream) {
  const int fits = prefix_attention_fits(rows, groups, nh, nkv, ws_bytes);
  if (fits != NE_OK) return fits;
  const int sms = device_sms(), G = nh / nkv;
  const int chunks = own_chunks(rows.max_q_len, G);
  const int splits = own_splits(rows.num_seqs, nkv, chunks, rows.max_context, sms);
  const Layout l = layout_of(rows.max_rows, rows.num_seqs, groups.num_groups, nh, splits, sms);
  if (groups.max_prefix_blocks == 0) groups.num_groups = 0;
  auto f = [&](size_t at) { return reinterpret_cast<float*>(ws + at); };
  const Parts parts{f(l.own_o), f(l.own_m), f(l.own_l), f(l.pre_o), f(l.pre_m), f(l.pre_l),
                    reinterpret_cast<int32_t*>(ws + l.entry_at), reinterpret_cast<int32_t*>(ws + l.group_work),
                    reinterpret_cast<int32_t*>(ws + l.group_vec), splits, sms};
  static bool pre_done[2][64] = {};
  if (groups.num_groups > 0) {
    CUtensorMap kmap{}, vmap{};
    if (!kv_int8 && (!make_tmap_kv(&kmap, k_cache, nkv, slots) || !make_tmap_kv(&vmap, v_cache, nkv, slots)))
      return NE_ERR_CUDA;
    auto kernel = kv_int8 ? prefix_kernel<true> : prefix_kernel<false>;
    if (!allow_smem(kernel, PRE_SMEM, pre_done[kv_int8 ? 1 : 0])) return NE_ERR_CUDA;
    if (launch_kernel(kernel, dim3(sms), dim3(pre_threads(kv_int8 != 0)), PRE_SMEM, stream, kmap, vmap,
                      static_cast<const int8_t*>(k_cache), static_cast<const int8_t*>(v_cache), k_scale, v_scale, q, rows,
                      groups, nh, nkv, slots, parts, status) != cudaSuccess)
      return NE_ERR_CUDA;
  }
  // one query tile of up to 16 vectors: eight warps where that leaves at most a CTA an SM, two where
  // there are many short waves anyway (measured, the whole call: 512 CTAs of 10 blocks 41.3 us with two
  // warps, 38.3 with four; 2048 CTAs of 7 blocks 89.8 and 97.9); two tiles (up to 32, or chunks of 32):
  // four pairs of warps
  const long long ctas = (long long)rows.num_seqs * nkv * chunks * splits;
  const bool one = (long long)rows.max_q_len * G <= 16;
  const int late = groups.num_groups > 0 ? 1 : 0;
  auto launch = [&](auto kernel, size_t smem, int threads, bool (&done)[64]) {
    if (!allow_smem(kernel, smem, done)) return (int)NE_ERR_CUDA;
    return launch_kernel(kernel, dim3(rows.num_seqs, nkv, chunks * splits), dim3(threads), smem, stream, q, k_cache,
                         v_cache, k_scale, v_scale, rows, groups, nh, nkv, slots, parts, chunks, late,
                         status) == cudaSuccess ? (int)NE_OK : (int)NE_ERR_CUDA;
  };
  static bool done[8][64] = {};
  int rc;
  if (!one) {
    rc = kv_int8 ? launch(own_tokens_kernel<true, 4, 2>, own_smem<4, 2>(), 256, done[0])
                 : launch(own_tokens_kernel<false, 4, 2>, own_smem<4, 2>(), 256, done[1]);
  } else if (ctas <= sms) {
    rc = kv_int8 ? launch(own_tokens_kernel<true, 8, 1>, own_smem<8, 1>(), 256, done[2])
                 : launch(own_tokens_kernel<false, 8, 1>, own_smem<8, 1>(), 256, done[3]);
  } else if (ctas <= 6LL * sms) {
    rc = kv_int8 ? launch(own_tokens_kernel<true, 4, 1>, own_smem<4, 1>(), 128, done[4])
                 : launch(own_tokens_kernel<false, 4, 1>, own_smem<4, 1>(), 128, done[5]);
  } else {
    rc = kv_int8 ? launch(own_tokens_kernel<true, 2, 1>, own_smem<2, 1>(), 64, done[6])
                 : launch(own_tokens_kernel<false, 2, 1>, own_smem<2, 1>(), 64, done[7]);
  }
  if (rc != NE_OK) return rc;
  const long long vectors = (long long)rows.max_q_len * nh;
  return launch_kernel(join_kernel, dim3((unsigned)((vectors + JOIN_WARPS - 1) / JOIN_WARPS), rows.num_seqs),
                       dim3(32 * JOIN_WARPS), 0, stream, out, rows, groups, nh, nkv, parts) == cudaSuccess
             ? NE_OK
             : NE_ERR_CUDA;
}

}  // namespace ne

extern "C" NE_API size_t ne_prefix_attention_workspace_bytes(int max_rows, int num_seqs, int num_groups, int num_heads,
                                                             int num_kv_heads, int max_q_len, int max_context) {
  if (max_rows < 0 || num_seqs < 1 || num_seqs > ne::MAX_SEQS || num_groups < 0 || num_groups > ne::MAX_SEQS ||
      !ne::heads_ok(num_heads, num_kv_heads) || max_q_len < 1 || max_context < 0)
    return 0;
  const int sms = ne::device_sms();
  const int chunks = ne::own_chunks(max_q_len, num_heads / num_kv_heads);
  return ne::layout_of(max_rows, num_seqs, num_groups, num_heads,
                       ne::own_splits(num_seqs, num_kv_heads, chunks, max_context, sms), sms).total;
}

extern "C" NE_API int ne_prefix_attention(const void* q, void* out, const void* k_cache, const void* v_cache,
                                          const void* k_scale, const void* v_scale, int kv_int8, const ne_rows* rows,
                                          const ne_prefix_groups* groups, int num_heads, int num_kv_heads,
                                          int block_size, long long num_cache_slots, void* workspace,
                                          size_t workspace_bytes, int32_t* status, void* stream) {
  if (!q || !out || !k_cache || !v_cache || !rows || !groups || (kv_int8 && (!k_scale || !v_scale)) ||
      num_cache_slots < 17 || block_size != 16 || !ne::heads_ok(num_heads, num_kv_heads) || rows->num_seqs <= 0 ||
      rows->num_seqs > ne::MAX_SEQS || rows->max_rows <= 0 || rows->max_q_len <= 0 || rows->max_context < 0 ||
      rows->block_table_stride < 0 || !rows->positions || !rows->q_start || !rows->q_len || !rows->block_tables ||
      groups->num_groups < 0 || groups->num_groups > ne::MAX_SEQS || groups->max_prefix_blocks < 0 ||
      (groups->num_groups > 0 && (!groups->entry_group || !groups->prefix_blocks)))
    return NE_ERR_INVALID;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) ||
      ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 127u) || !workspace ||
      (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return NE_ERR_INVALID;
  return ne::launch_prefix_attention(
      static_cast<const __nv_bfloat16*>(q), static_cast<__nv_bfloat16*>(out), k_cache, v_cache,
      static_cast<const __nv_bfloat16*>(k_scale), static_cast<const __nv_bfloat16*>(v_scale), kv_int8, *rows, *groups,
      num_heads, num_kv_heads, num_cache_slots, static_cast<uint8_t*>(workspace), workspace_bytes, status,
      static_cast<cudaStream_t>(stream));
}
