// Paged attention for a batch whose sequences share prompt prefixes (include/nespec.h,
// ne_prefix_attention): the simplest kernel that is right for every case. A warp serves one query
// vector against its sequence's whole context, 32 keys at a time: a key per lane for the scores, four
// dimensions per lane for the values.
#include "attention.cuh"

namespace ne {

namespace {

constexpr int D = 128;
constexpr unsigned ALL = 0xFFFFFFFFu;

__global__ void __launch_bounds__(128)
    row_attention_kernel(const __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ out,
                         const void* __restrict__ kc, const void* __restrict__ vc, const __nv_bfloat16* __restrict__ ks,
                         const __nv_bfloat16* __restrict__ vs, int kv_int8, ne_rows rows, int nh, int nkv,
                         long long num_cache_slots, int* status) {
  pdl_prologue();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x;
  const int ql = rows.q_len[b];
  const int v = blockIdx.y * 4 + warp;  // vector of the entry: row v / nh, head v % nh
  if (v >= ql * nh) return;
  const int row = rows.q_start[b] + v / nh, head = v % nh, h = head / (nh / nkv);
  const int pos = rows.positions[row];
  const int32_t* table =
      rows.block_tables + (long long)(rows.table_index ? rows.table_index[b] : b) * rows.block_table_stride;
  const __nv_bfloat16* qr = q + ((long long)row * nh + head) * D;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 <= pos; k0 += 32) {
    const int key = k0 + lane;
    long long slot = -1;
    if (key <= pos) {
      const long long blk = key / 16 < rows.block_table_stride ? table[key / 16] : -1;
      if (blk < 0 || (blk + 1) * 16 > num_cache_slots - 1) report(status, NE_DEV_BAD_SLOT);
      else slot = blk * 16 + key % 16;
    }
    float s = -INFINITY;
    if (slot >= 0) {
      const long long at = (slot * nkv + h) * D;
      const float scale = kv_int8 ? ld_bf16(ks + slot * nkv + h) : 1.f;
      float dot = 0.f;
      for (int d = 0; d < D; ++d)
        dot += ld_bf16(qr + d) * (kv_int8 ? (float)static_cast<const int8_t*>(kc)[at + d]
                                          : ld_bf16(static_cast<const __nv_bfloat16*>(kc) + at + d));
      s = dot * scale * 0.08838834764831845f;  // 1 / sqrt(128)
    }
    float top = s;
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(ALL, top, x));
    const float mn = fmaxf(m, top);
    if (mn == -INFINITY) continue;
    const float c = expf(m - mn), p = slot >= 0 ? expf(s - mn) : 0.f;
    m = mn;
    float sum = p;
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(ALL, sum, x);
    l = l * c + sum;
    for (int j = 0; j < 4; ++j) o[j] *= c;
    for (int t = 0; t < 32; ++t) {
      const long long st = __shfl_sync(ALL, slot, t);
      if (st < 0) continue;
      const float pt = __shfl_sync(ALL, p, t) * (kv_int8 ? ld_bf16(vs + st * nkv + h) : 1.f);
      const long long at = (st * nkv + h) * D + 4 * lane;
      for (int j = 0; j < 4; ++j)
        o[j] += pt * (kv_int8 ? (float)static_cast<const int8_t*>(vc)[at + j]
                              : ld_bf16(static_cast<const __nv_bfloat16*>(vc) + at + j));
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
  for (int j = 0; j < 4; ++j)
    out[((long long)row * nh + head) * D + 4 * lane + j] = __float2bfloat16_rn(o[j] * inv);
}

}  // namespace

}  // namespace ne

extern "C" NE_API size_t ne_prefix_attention_workspace_bytes(int max_rows, int num_seqs, int num_groups, int num_heads,
                                                             int num_kv_heads, int max_q_len, int max_context) {
  if (max_rows < 0 || num_seqs < 0 || num_seqs > 1024 || num_groups < 0 || num_kv_heads < 1 || num_heads < 1 ||
      num_heads % num_kv_heads || num_heads / num_kv_heads > 32 || max_q_len < 0 || max_context < 0)
    return 0;
  return 256;
}

extern "C" NE_API int ne_prefix_attention(const void* q, void* out, const void* k_cache, const void* v_cache,
                                          const void* k_scale, const void* v_scale, int kv_int8, const ne_rows* rows,
                                          const ne_prefix_groups* groups, int num_heads, int num_kv_heads,
                                          int block_size, long long num_cache_slots, void* workspace,
                                          size_t workspace_bytes, int32_t* status, void* stream) {
  if (!q || !out || !k_cache || !v_cache || !rows || !groups || (kv_int8 && (!k_scale || !v_scale)) ||
      num_cache_slots < 2 || block_size != 16 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads ||
      num_heads / num_kv_heads > 32 || rows->num_seqs <= 0 || rows->num_seqs > 1024 || rows->max_rows <= 0 ||
      rows->max_q_len <= 0 || rows->max_context < 0 || rows->block_table_stride < 0 || !rows->positions ||
      !rows->q_start || !rows->q_len || !rows->block_tables || groups->num_groups < 0 ||
      groups->max_prefix_blocks < 0 || (groups->num_groups > 0 && (!groups->entry_group || !groups->prefix_blocks)))
    return NE_ERR_INVALID;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return NE_ERR_INVALID;
  const size_t need =
      ne_prefix_attention_workspace_bytes(rows->max_rows, rows->num_seqs, groups->num_groups, num_heads, num_kv_heads,
                                          rows->max_q_len, rows->max_context);
  if (need == 0) return NE_ERR_INVALID;
  if (workspace_bytes < need) return NE_ERR_WORKSPACE;
  return ne::launch_kernel(ne::row_attention_kernel,
                           dim3(rows->num_seqs, ((long long)rows->max_q_len * num_heads + 3) / 4), dim3(128), 0,
                           static_cast<cudaStream_t>(stream), static_cast<const __nv_bfloat16*>(q),
                           static_cast<__nv_bfloat16*>(out), k_cache, v_cache,
                           static_cast<const __nv_bfloat16*>(k_scale), static_cast<const __nv_bfloat16*>(v_scale),
                           kv_int8, *rows, num_heads, num_kv_heads, num_cache_slots, status) == cudaSuccess
             ? NE_OK
             : NE_ERR_CUDA;
}
