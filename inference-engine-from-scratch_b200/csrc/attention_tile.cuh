// Query tiles of 16 vectors against 16-token KV blocks on tensor cores (mma.sync m16n8k16): staging of
// K and V blocks, and one block's scores, online softmax and product. Shared by the attention kernels.
#pragma once

#include "attention.cuh"

namespace ne {

namespace {

constexpr int D = 128;
constexpr int ROW_BYTES = D * 2 + 16;            // padded smem row: conflict-free ldmatrix
constexpr int BLOCK_BYTES = 16 * ROW_BYTES;      // one 16-token K (or V) block in smem
constexpr float LOG2E = 1.4426950408889634f;
constexpr float SCALE_LOG2 = 0.08838834764831845f * LOG2E;  // 1/sqrt(128) folded into exp2
#define NEG_INF (-__int_as_float(0x7f800000))

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t saddr, const void* g) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(saddr), "l"(g) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

struct Ctx {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const void* kc;
  const void* vc;
  const __nv_bfloat16* ks;
  const __nv_bfloat16* vs;
  const int32_t* table;
  int nh, nkv, h, G, r0, nvec;
  long long num_cache_slots;
  int* status;
  KvShadow sh;
};

// Stage one 16-token K and V block (block id ``blk``) into smem at k_s / v_s, using ``nthr``
// threads numbered ``t`` (a warp: 32, the CTA: 128). bf16 pools go through cp.async.
template <bool INT8>
__device__ __forceinline__ void stage_block(const Ctx& c, long long blk, uint32_t k_s, uint32_t v_s, int t,
                                            int nthr) {
  if (!INT8) {
    for (int i = t; i < 16 * 16; i += nthr) {  // 16 tokens x 16 chunks of 16 B, K and V
      const int tok = i >> 4, ch = i & 15;
      const long long off = ((blk * 16 + tok) * c.nkv + c.h) * D + ch * 8;
      cp_async16(k_s + tok * ROW_BYTES + ch * 16, reinterpret_cast<const __nv_bfloat16*>(c.kc) + off);
      cp_async16(v_s + tok * ROW_BYTES + ch * 16, reinterpret_cast<const __nv_bfloat16*>(c.vc) + off);
    }
  } else {
    for (int i = t; i < 16 * 8; i += nthr) {  // 16 tokens x 8 chunks of 16 int8
      const int tok = i >> 3, ch = i & 7;
      const long long slot = blk * 16 + tok;
      const long long off = (slot * c.nkv + c.h) * D + ch * 16;
      const float ksc = __bfloat162float(c.ks[slot * c.nkv + c.h]);
      const float vsc = __bfloat162float(c.vs[slot * c.nkv + c.h]);
      const int4 kq = *reinterpret_cast<const int4*>(reinterpret_cast<const int8_t*>(c.kc) + off);
      const int4 vq = *reinterpret_cast<const int4*>(reinterpret_cast<const int8_t*>(c.vc) + off);
      const int8_t* kb = reinterpret_cast<const int8_t*>(&kq);
      const int8_t* vb = reinterpret_cast<const int8_t*>(&vq);
      uint32_t kw[8], vw[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        kw[j] = pack_bf16(bf16r((float)kb[2 * j] * ksc), bf16r((float)kb[2 * j + 1] * ksc));
        vw[j] = pack_bf16(bf16r((float)vb[2 * j] * vsc), bf16r((float)vb[2 * j + 1] * vsc));
      }
      const uint32_t ko = k_s + tok * ROW_BYTES + ch * 32, vo = v_s + tok * ROW_BYTES + ch * 32;
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(ko), "r"(kw[0]), "r"(kw[1]), "r"(kw[2]), "r"(kw[3]));
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(ko + 16), "r"(kw[4]), "r"(kw[5]), "r"(kw[6]),
                   "r"(kw[7]));
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(vo), "r"(vw[0]), "r"(vw[1]), "r"(vw[2]), "r"(vw[3]));
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(vo + 16), "r"(vw[4]), "r"(vw[5]), "r"(vw[6]),
                   "r"(vw[7]));
    }
  }
}

// Shared-memory address of (token, dimension col) in a staged K or V block: the padded row layout
// (cp.async and conversions), or (SW) the tensor-load layout: two 2 KB boxes of dimensions 0-63 and
// 64-127, rows of 128 B whose 16-byte chunk c sits at c ^ (token % 8) (the 128-byte swizzle).
template <bool SW>
__device__ __forceinline__ uint32_t kv_addr(uint32_t base, int tok, int col) {
  if (!SW) return base + tok * ROW_BYTES + col * 2;
  const int c = col >> 3;
  return base + (c >> 3) * 2048 + tok * 128 + (((c & 7) ^ (tok & 7)) << 4);
}

// Stage dequantised copy ``sh`` of a shared int8 block (bf16, the pool's row layout) by cp.async.
__device__ __forceinline__ void stage_shadow(const Ctx& c, int sh, uint32_t k_s, uint32_t v_s, int lane) {
  for (int i = lane; i < 16 * 16; i += 32) {
    const int tok = i >> 4, ch = i & 15;
    const long long off = (((long long)sh * 16 + tok) * c.nkv + c.h) * D + ch * 8;
    cp_async16(k_s + tok * ROW_BYTES + ch * 16, c.sh.k + off);
    cp_async16(v_s + tok * ROW_BYTES + ch * 16, c.sh.v + off);
  }
}

// int8 pool, per-warp path: issue one block's raw K and V rows (16 tokens x 128 int8 each) into
// smem at raw (K) and raw + 2048 (V) with cp.async (lane-strided 16-byte chunks).
__device__ __forceinline__ void stage_raw_int8(const Ctx& c, long long blk, uint32_t raw, int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = lane + 32 * j, tok = i >> 3, ch = i & 7;
    const long long off = ((blk * 16 + tok) * c.nkv + c.h) * D + ch * 16;
    cp_async16(raw + tok * 128 + ch * 16, reinterpret_cast<const int8_t*>(c.kc) + off);
    cp_async16(raw + 2048 + tok * 128 + ch * 16, reinterpret_cast<const int8_t*>(c.vc) + off);
  }
}
// The block's bf16 scales, one per lane: lanes 0-15 the K scale of token lane, 16-31 the V scale of
// token lane - 16 (plain loads, issued a block ahead of their use).
__device__ __forceinline__ uint32_t load_scales_int8(const Ctx& c, long long blk, int lane) {
  const long long slot = blk * 16 + (lane & 15);
  const __nv_bfloat16* src = lane < 16 ? c.ks : c.vs;
  return (uint32_t)__bfloat16_as_ushort(src[slot * c.nkv + c.h]);
}
// bf16(q * scale) for a pair of int8 values in the low 16 bits of ``word`` (selector 0x4140) or
// the high 16 bits (0x4342): q exact in bf16 from byte magic, then one bf16x2 multiply (the
// rounding of read_from_cache's int8.to(bf16) * scale).
__device__ __forceinline__ uint32_t dq_pair(uint32_t word, uint32_t sel, uint32_t scale2) {
  const uint32_t p = __byte_perm(word, 0x43434343u, sel);
  const uint32_t v = p & 0x437F437Fu, b = p & 0x43804380u;
  uint32_t q, r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(q) : "r"(v), "r"(b));
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(q), "r"(scale2));
  return r;
}
// 16 raw int8 rows (16 tokens x 128, at ``raw``) -> bf16 rows in the padded layout at ``dst``; the
// scale of token t is lane ``scale_lane + t``'s ``scales``. All four loads go out before the
// conversion (one shared-memory latency per block, not one per chunk).
__device__ __forceinline__ void convert_half_int8(uint32_t raw, uint32_t dst, uint32_t scales, int scale_lane,
                                                  int lane) {
  uint32_t w[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = lane + 32 * j, tok = i >> 3, ch = i & 7;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[j][0]), "=r"(w[j][1]), "=r"(w[j][2]), "=r"(w[j][3])
                 : "r"(raw + tok * 128 + ch * 16));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = lane + 32 * j, tok = i >> 3, ch = i & 7;
    const uint32_t sc = __shfl_sync(0xFFFFFFFFu, scales, scale_lane + tok);
    const uint32_t s2 = sc | (sc << 16);
    uint32_t o[8];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      o[2 * t] = dq_pair(w[j][t], 0x4140u, s2);
      o[2 * t + 1] = dq_pair(w[j][t], 0x4342u, s2);
    }
    const uint32_t d = dst + tok * ROW_BYTES + ch * 32;
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(d), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3])
                 : "memory");
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(d + 16), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                 : "memory");
  }
}
// Raw int8 block (staged by stage_raw_int8) -> bf16 K / V blocks in the padded row layout.
__device__ __forceinline__ void convert_raw_int8(uint32_t raw, uint32_t k_s, uint32_t v_s, uint32_t scales,
                                                 int lane) {
  convert_half_int8(raw, k_s, scales, 0, lane);
  convert_half_int8(raw + 2048, v_s, scales, 16, lane);
}
// The same from a raw block a tensor load wrote (16 rows of 128 int8, 16-byte chunk c of row t at
// c ^ (t % 8)) into the swizzled bf16 layout ``kv_addr<true>`` reads: chunk c of int8 becomes
// bf16 chunks 2c and 2c + 1. The same arithmetic as convert_half_int8.
__device__ __forceinline__ void convert_half_int8_sw(uint32_t raw, uint32_t dst, uint32_t scales, int scale_lane,
                                                     int lane) {
  uint32_t w[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = lane + 32 * j, tok = i >> 3, ch = i & 7;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[j][0]), "=r"(w[j][1]), "=r"(w[j][2]), "=r"(w[j][3])
                 : "r"(raw + tok * 128 + ((ch ^ (tok & 7)) << 4)));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = lane + 32 * j, tok = i >> 3, ch = i & 7;
    const uint32_t sc = __shfl_sync(0xFFFFFFFFu, scales, scale_lane + tok);
    const uint32_t s2 = sc | (sc << 16);
    uint32_t o[8];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      o[2 * t] = dq_pair(w[j][t], 0x4140u, s2);
      o[2 * t + 1] = dq_pair(w[j][t], 0x4342u, s2);
    }
    const uint32_t d0 = kv_addr<true>(dst, tok, 16 * ch), d1 = kv_addr<true>(dst, tok, 16 * ch + 8);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(d0), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3])
                 : "memory");
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(d1), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                 : "memory");
  }
}

// A block-table entry checked against the pool: the id, or -1 (reported) when it names no block.
__device__ __forceinline__ long long checked_block(const Ctx& c, long long blk) {
  if (blk < 0 || (blk + 1) * 16 > c.num_cache_slots - 1) {
    report(c.status, NE_DEV_BAD_SLOT);
    return -1;
  }
  return blk;
}

// Valid block id of logical block ``kb`` or -1 (reported) when the table names no pool block.
__device__ __forceinline__ long long block_id(const Ctx& c, int kb, int stride) {
  long long blk = kb < stride ? c.table[kb] : -1;
  if (blk < 0 || (blk + 1) * 16 > c.num_cache_slots - 1) {
    report(c.status, NE_DEV_BAD_SLOT);
    return -1;
  }
  return blk;
}

// Load the 16-vector query tile starting at vector ``v0`` (rows past nvec are zero) into smem.
__device__ __forceinline__ void load_q_tile(const Ctx& c, int v0, uint8_t* q_s, int t, int nthr) {
  for (int i = t; i < 16 * 16; i += nthr) {
    const int v = i >> 4, ch = i & 15;
    uint4 val = make_uint4(0, 0, 0, 0);
    if (v0 + v < c.nvec) {
      const int row = c.r0 + (v0 + v) / c.G;
      const int head = c.h * c.G + (v0 + v) % c.G;
      val = *reinterpret_cast<const uint4*>(c.q + ((long long)row * c.nh + head) * D + ch * 8);
    }
    *reinterpret_cast<uint4*>(q_s + v * ROW_BYTES + ch * 16) = val;
  }
}

struct TileState {
  uint32_t qa[8][4];  // Q A-fragments for the 8 k-steps of 16 dims
  float o[16][4];     // O accumulators: 16 tiles of 8 dims
  float m[2], l[2];   // running max (log2 domain) and sum for rows lane/4 and lane/4 + 8
  int pos[2];         // positions of those rows (-1: padding row)
};

__device__ __forceinline__ void tile_init(TileState& ts, uint32_t q_s, const int* spos, int lane) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
    const int row = (lane & 7) + 8 * ((lane >> 3) & 1);
    const int col = 16 * kk + 8 * (lane >> 4);
    ldsm_x4(ts.qa[kk], q_s + row * ROW_BYTES + col * 2);
  }
#pragma unroll
  for (int t = 0; t < 16; ++t) ts.o[t][0] = ts.o[t][1] = ts.o[t][2] = ts.o[t][3] = 0.f;
  ts.m[0] = ts.m[1] = NEG_INF;
  ts.l[0] = ts.l[1] = 0.f;
  ts.pos[0] = spos[lane >> 2];
  ts.pos[1] = spos[(lane >> 2) + 8];
}

// One 16-token block (logical index kb) staged at k_s / v_s against the tile.
template <bool SW = false>
__device__ __forceinline__ void tile_block(TileState& ts, uint32_t k_s, uint32_t v_s, int kb, int lane) {
  float s[2][4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; kk += 2) {
      uint32_t b[4];
      const int tok = 8 * j + (lane & 7);
      const int col = 16 * kk + 8 * (lane >> 3);
      ldsm_x4(b, kv_addr<SW>(k_s, tok, col));
      mma16816(s[j], ts.qa[kk], b[0], b[1]);
      mma16816(s[j], ts.qa[kk + 1], b[2], b[3]);
    }
  }
  // scale (log2 domain), causal mask, online softmax per row
  float mx[2] = {NEG_INF, NEG_INF};
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = e >> 1;
      const int key = kb * 16 + 8 * j + 2 * (lane & 3) + (e & 1);
      float v = s[j][e] * SCALE_LOG2;
      if (key > ts.pos[r]) v = NEG_INF;
      s[j][e] = v;
      mx[r] = fmaxf(mx[r], v);
    }
  float corr[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xFFFFFFFFu, mx[r], 1));
    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xFFFFFFFFu, mx[r], 2));
    const float m_new = fmaxf(ts.m[r], mx[r]);
    corr[r] = (m_new == NEG_INF || ts.m[r] == NEG_INF) ? (m_new == NEG_INF ? 1.f : 0.f) : exp2f(ts.m[r] - m_new);
    ts.m[r] = m_new;
  }
  float psum[2] = {0.f, 0.f};
  uint32_t pa[4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = e >> 1;
      p[e] = (s[j][e] == NEG_INF) ? 0.f : exp2f(s[j][e] - ts.m[r]);
      psum[r] += p[e];
    }
    pa[2 * j] = pack_bf16(p[0], p[1]);
    pa[2 * j + 1] = pack_bf16(p[2], p[3]);
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    psum[r] += __shfl_xor_sync(0xFFFFFFFFu, psum[r], 1);
    psum[r] += __shfl_xor_sync(0xFFFFFFFFu, psum[r], 2);
    ts.l[r] = ts.l[r] * corr[r] + psum[r];
  }
  // (a max that did not move leaves every factor at exactly 1: the products are skipped)
  if (__any_sync(0xFFFFFFFFu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      ts.o[t][0] *= corr[0];
      ts.o[t][1] *= corr[0];
      ts.o[t][2] *= corr[1];
      ts.o[t][3] *= corr[1];
    }
  }
#pragma unroll
  for (int t = 0; t < 16; t += 2) {
    uint32_t b[4];
    const int tok = (lane & 7) + 8 * ((lane >> 3) & 1);
    const int col = 8 * t + 8 * (lane >> 4);
    ldsm_x4_t(b, kv_addr<SW>(v_s, tok, col));
    mma16816(ts.o[t], pa, b[0], b[1]);
    mma16816(ts.o[t + 1], pa, b[2], b[3]);
  }
}

}  // namespace

}  // namespace ne
