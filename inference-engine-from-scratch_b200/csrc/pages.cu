// Pages of the KV cache: copying them within the pool, forking a sequence (its full pages shared,
// its last one copied), returning pages a sequence does not need, and compacting the pool.
//
// The pool is [layers][2][slots][kv heads][128] (bf16 or int8, with [layers][2][slots][kv heads]
// bf16 scales): a page (16 slots) is one contiguous piece of each (layer, K or V) plane. Every
// kernel here changes ids in place only where no other thread of the launch reads them, and every
// id is checked against the pool before it is used.
#include "kernels.cuh"

namespace ne {

namespace {

constexpr int BS = 16;  // tokens in a page
constexpr int COPY_THREADS = 256;

// One unit of work: page pair i in one (layer, K / V) plane, 16 bytes a thread and step, four loads
// in flight before the first store. Bound by memory: each page is read and written once (1.47 GB moved in
// 240 us: 6.1 TB/s, 95% of a plain copy's rate; four pairs in 28 layers, 9 MB, in 4 us from L2).
__global__ void __launch_bounds__(COPY_THREADS)
    copy_pages_kernel(uint8_t* kv, uint16_t* scales, int planes, int nkv, int elem_bytes,
                      long long slots, const int32_t* src, const int32_t* dst, const int32_t* count, int max_pairs,
                      int* status) {
  pdl_prologue();
  const int pairs = count ? min(max(*count, 0), max_pairs) : max_pairs;
  const long long units = (long long)pairs * planes;
  const int page_vec = BS * nkv * 128 * elem_bytes / 16;
  const long long plane_vec = slots * nkv * 128 * elem_bytes / 16;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int i = (int)(u / planes), plane = (int)(u % planes);
    const long long s = src[i], d = dst[i];
    if (s < 0 || s == d) continue;  // (a negative source: no copy is asked for)
    if ((s + 1) * BS > slots - 1 || d < 0 || (d + 1) * BS > slots - 1) {
      if (plane == 0 && threadIdx.x == 0) report(status, NE_DEV_BAD_SLOT);
      continue;
    }
    const uint4* from = reinterpret_cast<const uint4*>(kv) + plane * plane_vec + s * page_vec;
    uint4* to = reinterpret_cast<uint4*>(kv) + plane * plane_vec + d * page_vec;
    for (int v = threadIdx.x; v < page_vec; v += 4 * COPY_THREADS) {
      uint4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v + j * COPY_THREADS < page_vec) x[j] = from[v + j * COPY_THREADS];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v + j * COPY_THREADS < page_vec) to[v + j * COPY_THREADS] = x[j];
    }
    if (scales) {  // 2-byte pieces: a plane of an odd number of slots starts at no wider boundary
      const uint16_t* sf = scales + (plane * slots + s * BS) * nkv;
      uint16_t* st = scales + (plane * slots + d * BS) * nkv;
      for (int v = threadIdx.x; v < BS * nkv; v += COPY_THREADS) st[v] = sf[v];
    }
  }
}

// Which forks are made, and with which pages: thread i serves destination i. ``copy_src[i]``: the
// source's page to copy into copy_dst[i], -1 when the fork ends on a page boundary, -2 when the
// destination was refused (out of range, the source itself, listed before, or still holding pages).
__global__ void __launch_bounds__(1024)
    fork_plan_kernel(ne_batch_state st, int src, const int32_t* dst_slots, int num_dst, int at, const uint64_t* seeds,
                     int32_t* copy_src, int32_t* copy_dst, int* status) {
  pdl_prologue();
  __shared__ int s_dst[1024];
  __shared__ int s_rank[1024];
  __shared__ int fail;
  const int i = threadIdx.x;
  const int d = i < num_dst ? dst_slots[i] : -1;
  if (i < num_dst) s_dst[i] = d;
  if (i == 0) fail = 0;
  __syncthreads();
  bool ok = i < num_dst && d >= 0 && d < st.max_seqs && d != src && st.num_blocks_used[d] == 0;
  for (int j = 0; ok && j < i; ++j) ok = s_dst[j] != d;
  // the fork's tokens: the first ``at`` of the source's (0: all of them); the last one is always
  // left to be computed, as it is after every step
  const int len_src = st.seq_len[src];
  const int len = at > 0 ? at : len_src;
  const int cached = min(st.num_cached[src], len - 1);
  const int full = cached / BS, tail = cached % BS ? 1 : 0;
  if (len < 1 || len > len_src || cached < 0 || full + tail > st.num_blocks_used[src]) {
    if (i == 0) report(status, NE_DEV_HISTORY_FULL);
    ok = false;
  }
  const int valid = __syncthreads_count(ok);
  s_rank[i] = ok ? 1 : 0;
  __syncthreads();
  int rank = 0;  // valid destinations before this one
  for (int j = 0; j < i && j < num_dst; ++j) rank += s_rank[j];
  const long long head = st.ring_head_tail[0];
  if (i == 0 && tail && valid > st.ring_head_tail[1] - head) {
    report(status, NE_DEV_OUT_OF_BLOCKS);
    fail = 1;
  }
  __syncthreads();  // every thread has read the ring's head
  if (fail) ok = false;
  if (i < num_dst) {
    if (!ok && !fail) report(status, NE_DEV_BAD_SLOT);
    copy_src[i] = ok ? (tail ? st.block_tables[(long long)src * st.block_table_stride + full] : -1) : -2;
    copy_dst[i] = -1;
  }
  if (ok) {
    if (tail) {
      const int page = st.free_ring[(head + rank) % st.num_blocks];
      st.block_tables[(long long)d * st.block_table_stride + full] = page;
      copy_dst[i] = page;
    }
    st.num_blocks_used[d] = full + tail;
    st.num_shared_blocks[d] = full;
    st.seq_len[d] = len;
    st.num_cached[d] = cached;
    st.num_prompt[d] = min(st.num_prompt[src], len);
    st.max_new_tokens[d] = st.max_new_tokens[src];
    st.flags[d] = len < len_src ? st.flags[src] & ~NE_SEQ_FINISHED : st.flags[src];
    st.temperature[d] = st.temperature[src];
    st.top_p[d] = st.top_p[src];
    st.rng_seed[d] = seeds ? seeds[i] : st.rng_seed[src];
    st.rng_draws[d] = seeds ? 0 : st.rng_draws[src];
  }
  if (i == 0 && !fail && tail) st.ring_head_tail[0] = head + valid;
}

// The tokens and the shared table entries of every fork that was made (one CTA each).
__global__ void fork_rows_kernel(ne_batch_state st, int src, const int32_t* dst_slots, const int32_t* copy_src) {
  pdl_prologue();
  const int i = blockIdx.x;
  if (copy_src[i] == -2) return;
  const int d = dst_slots[i], len = st.seq_len[d], shared = st.num_shared_blocks[d];
  const int32_t* from = st.history + (long long)src * st.history_stride;
  int32_t* to = st.history + (long long)d * st.history_stride;
  for (int j = threadIdx.x; j < len; j += blockDim.x) to[j] = from[j];
  const int32_t* tf = st.block_tables + (long long)src * st.block_table_stride;
  int32_t* tt = st.block_tables + (long long)d * st.block_table_stride;
  for (int j = threadIdx.x; j < shared; j += blockDim.x) tt[j] = tf[j];
}

// Pages past the ones that hold cached tokens go back to the FIFO's tail in table order (one warp;
// the slots in turn, so that a slot listed twice is trimmed once).
__global__ void trim_slots_kernel(ne_batch_state st, const int32_t* slots, int num_slots, int* status) {
  pdl_prologue();
  const int lane = threadIdx.x;
  long long tail = st.ring_head_tail[1];
  for (int i = 0; i < num_slots; ++i) {
    const int s = slots[i];
    if (s < 0 || s >= st.max_seqs) {
      if (lane == 0) report(status, NE_DEV_BAD_SLOT);
      continue;
    }
    const int used = st.num_blocks_used[s];
    const int shared = st.num_shared_blocks ? min(st.num_shared_blocks[s], used) : 0;
    const int keep = max(shared, (st.num_cached[s] + BS - 1) / BS);
    __syncwarp();
    if (keep >= used) continue;
    int32_t* row = st.block_tables + (long long)s * st.block_table_stride;
    for (int j = keep + lane; j < used; j += 32) {
      st.free_ring[(tail + j - keep) % st.num_blocks] = row[j];
      row[j] = -1;
    }
    tail += used - keep;
    if (lane == 0) st.num_blocks_used[s] = keep;
    __syncwarp();
  }
  if (lane == 0) st.ring_head_tail[1] = tail;
}

// Exclusive scan over the CTA's 1024 threads; ``total`` gets the sum.
__device__ __forceinline__ int scan_1024(int v, int* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += t;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  *total = all;
  return before + incl - v;
}

// The pages in use move to ids 0 .. used - 1: page i >= used that is in use takes the place of an id
// below used that is not, both in ascending order, so no page is both read and written. ``map``
// [num_blocks]: each page's new id, -1 for a free one. The tables follow, the FIFO then holds the ids
// from used up in ascending order. One CTA: the work is a few reads per page and table entry.
__global__ void __launch_bounds__(1024)
    compact_kernel(ne_batch_state st, int32_t* map, int32_t* move_src, int32_t* move_dst, int32_t* move_count,
                   int32_t* copies, int* status) {
  pdl_prologue();
  __shared__ int sums[32];
  const int tid = threadIdx.x, n = st.num_blocks;
  for (int b = tid; b < n; b += 1024) map[b] = 0;
  __syncthreads();
  const int warp = tid >> 5, lane = tid & 31;
  for (int s = warp; s < st.max_seqs; s += 32) {
    const int used = min(st.num_blocks_used[s], st.block_table_stride);
    const int32_t* row = st.block_tables + (long long)s * st.block_table_stride;
    for (int j = lane; j < used; j += 32) {
      const int b = row[j];
      if (b < 0 || b >= n) report(status, NE_DEV_BAD_SLOT);
      else map[b] = 1;
    }
  }
  __syncthreads();
  int mine = 0;
  for (int b = tid; b < n; b += 1024) mine += map[b];
  int used;
  scan_1024(mine, sums, &used);
  // free ids below used, then used ids from used up: equally many, listed in ascending order
  int holes = 0, movers = 0;
  for (int base = 0; base < n; base += 1024) {
    const int b = base + tid;
    const int hole = b < used && map[b] == 0, mover = b >= used && b < n && map[b] == 1;
    int all_h, all_m;
    const int h = scan_1024(hole, sums, &all_h);
    const int m = scan_1024(mover, sums, &all_m);
    if (hole) move_dst[holes + h] = b;
    if (mover) move_src[movers + m] = b;
    holes += all_h;
    movers += all_m;
  }
  __syncthreads();
  for (int b = tid; b < n; b += 1024) map[b] = (b < used && map[b] == 1) ? b : -1;
  __syncthreads();
  for (int i = tid; i < movers; i += 1024) {
    const int from = move_src[i], to = move_dst[i];
    map[from] = to;
    if (copies) {  // a dequantised copy follows its page
      copies[to] = copies[from];
      copies[from] = -1;
    }
  }
  __syncthreads();
  for (int s = warp; s < st.max_seqs; s += 32) {
    const int len = min(st.num_blocks_used[s], st.block_table_stride);
    int32_t* row = st.block_tables + (long long)s * st.block_table_stride;
    for (int j = lane; j < len; j += 32) {
      const int b = row[j];
      if (b >= 0 && b < n) row[j] = map[b];
    }
  }
  for (int i = tid; i < n - used; i += 1024) st.free_ring[i] = used + i;
  if (tid == 0) {
    st.ring_head_tail[0] = 0;
    st.ring_head_tail[1] = n - used;
    *move_count = movers;
  }
}

int sm_count_of_device() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

bool state_ok(const ne_batch_state* st) {
  return st && st->max_seqs > 0 && st->history_stride > 0 && st->block_table_stride > 0 && st->num_blocks > 0 &&
         st->seq_len && st->num_cached && st->block_tables && st->num_blocks_used && st->free_ring && st->ring_head_tail;
}

}  // namespace

}  // namespace ne

extern "C" {

NE_API int ne_kv_copy_blocks(void* kv, void* scales, int kv_int8, int num_layers, int num_kv_heads,
                             long long num_cache_slots, const int32_t* src, const int32_t* dst, const int32_t* count,
                             int max_pairs, int32_t* status, void* stream) {
  if (!kv || (reinterpret_cast<uintptr_t>(kv) & 15u) || (kv_int8 ? !scales : scales != nullptr) || num_layers < 1 ||
      num_kv_heads < 1 || num_kv_heads > 1024 || num_cache_slots < 2 || max_pairs < 0 || (max_pairs > 0 && (!src || !dst)))
    return NE_ERR_INVALID;
  if (max_pairs == 0) return NE_OK;
  const long long units = (long long)max_pairs * 2 * num_layers;
  const long long most = 8LL * ne::sm_count_of_device();
  return ne::launch_kernel(ne::copy_pages_kernel, dim3((unsigned)(units < most ? units : most)), dim3(ne::COPY_THREADS),
                           0, static_cast<cudaStream_t>(stream), static_cast<uint8_t*>(kv),
                           static_cast<uint16_t*>(scales), 2 * num_layers, num_kv_heads, kv_int8 ? 1 : 2,
                           num_cache_slots, src, dst, count, max_pairs, status) == cudaSuccess
             ? NE_OK
             : NE_ERR_CUDA;
}

NE_API int ne_state_fork_slots(const ne_batch_state* st, int src_slot, const int32_t* dst_slots, int num_dst, int at,
                               const uint64_t* seeds, int32_t* copy_src, int32_t* copy_dst, int32_t* status,
                               void* stream) {
  if (!ne::state_ok(st) || !st->history || !st->num_shared_blocks || !st->num_prompt || !st->max_new_tokens ||
      !st->flags || !st->temperature || !st->top_p || !st->rng_seed || !st->rng_draws || src_slot < 0 ||
      src_slot >= st->max_seqs || at < 0 || at > st->history_stride || num_dst < 0 || num_dst > 1024 ||
      (num_dst > 0 && (!dst_slots || !copy_src || !copy_dst)))
    return NE_ERR_INVALID;
  if (num_dst == 0) return NE_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (ne::launch_kernel(ne::fork_plan_kernel, dim3(1), dim3(1024), 0, s, *st, src_slot, dst_slots, num_dst, at, seeds,
                        copy_src, copy_dst, status) != cudaSuccess)
    return NE_ERR_CUDA;
  return ne::launch_kernel(ne::fork_rows_kernel, dim3(num_dst), dim3(256), 0, s, *st, src_slot, dst_slots,
                           static_cast<const int32_t*>(copy_src)) == cudaSuccess
             ? NE_OK
             : NE_ERR_CUDA;
}

NE_API int ne_state_trim_slots(const ne_batch_state* st, const int32_t* slots, int num_slots, int32_t* status,
                               void* stream) {
  if (!ne::state_ok(st) || num_slots < 0 || (num_slots > 0 && !slots)) return NE_ERR_INVALID;
  if (num_slots == 0) return NE_OK;
  return ne::launch_kernel(ne::trim_slots_kernel, dim3(1), dim3(32), 0, static_cast<cudaStream_t>(stream), *st, slots,
                           num_slots, status) == cudaSuccess
             ? NE_OK
             : NE_ERR_CUDA;
}

NE_API int ne_state_compact(const ne_batch_state* st, int32_t* map, int32_t* move_src, int32_t* move_dst,
                            int32_t* move_count, int32_t* copy_map, int32_t* status, void* stream) {
  if (!ne::state_ok(st) || !map || !move_src || !move_dst || !move_count) return NE_ERR_INVALID;
  return ne::launch_kernel(ne::compact_kernel, dim3(1), dim3(1024), 0, static_cast<cudaStream_t>(stream), *st, map,
                           move_src, move_dst, move_count, copy_map, status) == cudaSuccess
             ? NE_OK
             : NE_ERR_CUDA;
}

}  // extern "C"
