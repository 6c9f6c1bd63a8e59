// KV cache held in 4 bits, in pages: geometry, argument blocks of the kernels
// and the launchers of kv4.cu / kv4_attn.cu / kv4_prompt.cu.
//
// A page holds page_size slots of every kv head:
//   [kv_heads][page_size / seg][K codes | K params | V codes | V params],
// seg = min(page_size, 64). Codes: seg rows of head_dim / 2 bytes, params:
// seg rows of head_dim / group words (f16 scale in the low half, f16 bias in
// the high half). A channel's value is scale * code + bias.
//
// A row is eight units of head_dim / 64 words; unit r, word w holds channels
// 64 w + 8 r .. + 7, low nibble first, so that one vector load of a unit
// gives a lane the same eight channels of every 64-channel block (the
// fragment order of the tensor-core kernels: kv4_attn.cu). Unit r of row t is
// stored at position r ^ kv4_swz(t): rows read together by a warp fall on
// different shared-memory banks.
#pragma once

#include "common.h"

namespace swl {

constexpr int KV4_BAD = 2;  // status bit 1: a page id or a length out of range

struct Kv4Geo {
  uint8_t* pages = nullptr;
  const int* table = nullptr;
  int64_t tstride = 0;
  int npages = 0, page = 0, pshift = 0, seg = 0, kvh = 0, hd = 0, group = 0, ng = 0;
  int blk = 0;           // bytes of one block: K codes, K params, V codes, V params
  int64_t page_bytes = 0;
};

struct Kv4Batch {
  const int* start = nullptr;  // [nseq + 1] first row of each sequence's new tokens
  const int* lens = nullptr;   // [nseq] slots, new tokens included
  int nseq = 0, total = 0, max_new = 0, max_len = 0;
  int* status = nullptr;
};

struct Kv4Rows {
  uint8_t* p = nullptr;
  int64_t ts = 0, hs = 0;  // elements between tokens and heads
};

struct Kv4IoArgs {  // append and read
  Kv4Geo g;
  Kv4Batch b;
  Kv4Rows k, v;
  float* weights = nullptr;
  int64_t wstride = 0;
};

struct Kv4AttnArgs {
  Kv4Geo g;
  Kv4Batch b;
  int dt = 0, heads = 0, rep = 0;
  float scale = 0.f;
  Kv4Rows q, out, gate;
  float* lse = nullptr;      // [total][heads]
  float* weights = nullptr;  // [nseq][kvh][wstride]
  int64_t wstride = 0;
  uint8_t* work = nullptr;
};

struct Kv4EvictArgs {
  Kv4Geo g;
  Kv4Batch b;
  int keep = 0, first = 0, recent = 0;
  const float* weights = nullptr;
  int64_t wstride = 0;
  const int* dst = nullptr;
  int64_t dstride = 0;
  int* new_lens = nullptr;
  float* new_weights = nullptr;
  int64_t nwstride = 0;
  int* kept = nullptr;  // [nseq][kvh][kstride]
  int64_t kstride = 0;
};

void launch_kv4_append(const Kv4IoArgs& a, int dt, cudaStream_t st);
void launch_kv4_read(const Kv4IoArgs& a, int dt, cudaStream_t st);
void launch_kv4_evict(const Kv4EvictArgs& a, cudaStream_t st);
int64_t kv4_attention_work(const Kv4Geo& g, const Kv4Batch& b, int heads);
void launch_kv4_attention(const Kv4AttnArgs& a, cudaStream_t st);
int64_t kv4_prompt_work(const Kv4Geo& g, const Kv4Batch& b, int heads);
void launch_kv4_prompt(const Kv4AttnArgs& a, cudaStream_t st);

#ifdef __CUDACC__
__device__ __forceinline__ int kv4_swz(int hd, int t) {
  return hd == 256 ? (t & 6) ^ ((t & 1) << 2) : hd == 128 ? (t & 2) << 1 : 0;
}

// Block that holds slot `slot` of head h, or null (and status bit 1) when the
// table names a page outside the pool.
__device__ __forceinline__ uint8_t* kv4_block(const Kv4Geo& g, const int* table, int64_t tstride, int seq, int h, int slot,
                                              int* status) {
  const int pg = __ldg(table + seq * tstride + (slot >> g.pshift));
  if (unsigned(pg) >= unsigned(g.npages)) {
    if (status) atomicOr(status, KV4_BAD);
    return nullptr;
  }
  const int nb = g.page / g.seg;
  return g.pages + pg * g.page_bytes + int64_t(h * nb + (slot & (g.page - 1)) / g.seg) * g.blk;
}

// Length of a sequence, held to [0, max_len] (status bit 1 outside).
__device__ __forceinline__ int kv4_len(const Kv4Batch& b, int seq) {
  const int n = __ldg(b.lens + seq);
  if (n >= 0 && n <= b.max_len) return n;
  if (b.status) atomicOr(b.status, KV4_BAD);
  return n < 0 ? 0 : b.max_len;
}

// New tokens of a sequence: first row and count, held to the rows [0, total).
__device__ __forceinline__ int kv4_new(const Kv4Batch& b, int seq, int& row0) {
  const int s0 = max(0, min(__ldg(b.start + seq), b.total)), s1 = max(0, min(__ldg(b.start + seq + 1), b.total));
  row0 = s0;
  return max(0, s1 - s0);
}

__device__ __forceinline__ float kv4_ld(const uint8_t* p, int dt, int64_t i) {
  if (dt == DT_F32) return reinterpret_cast<const float*>(p)[i];
  const uint16_t u = reinterpret_cast<const uint16_t*>(p)[i];
  return dt == DT_BF16 ? bf16_to_f32(u) : f16_bits_to_f32(u);
}
__device__ __forceinline__ void kv4_st(uint8_t* p, int dt, int64_t i, float v) {
  if (dt == DT_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dt == DT_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}
// Whether every 8 elements from a multiple of 8 on of r are 16-byte aligned.
__device__ __forceinline__ bool kv4_vec(const Kv4Rows& r, int dt) {
  const int64_t e = dt == DT_F32 ? 4 : 2;
  return ((reinterpret_cast<uintptr_t>(r.p) | uintptr_t(r.ts * e) | uintptr_t(r.hs * e)) & 15) == 0;
}
// Eight consecutive elements; `vec`: 16-byte aligned.
__device__ __forceinline__ void kv4_ld8(const uint8_t* p, int dt, int64_t i, bool vec, float (&x)[8]) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = kv4_ld(p, dt, i + e);
  } else if (dt == DT_F32) {
    const float4 a = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i)[0];
    const float4 b = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = dt == DT_BF16 ? bf16_to_f32(uint16_t(w[e])) : f16_bits_to_f32(uint16_t(w[e]));
      x[2 * e + 1] = dt == DT_BF16 ? bf16_to_f32(uint16_t(w[e] >> 16)) : f16_bits_to_f32(uint16_t(w[e] >> 16));
    }
  }
}
__device__ __forceinline__ void kv4_st8(uint8_t* p, int dt, int64_t i, bool vec, const float (&x)[8]) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) kv4_st(p, dt, i + e, x[e]);
  } else if (dt == DT_F32) {
    float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
    d[0] = make_float4(x[0], x[1], x[2], x[3]);
    d[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = dt == DT_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x[2 * e])) : __half_as_ushort(__float2half_rn(x[2 * e]));
      const uint32_t hi = dt == DT_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x[2 * e + 1])) : __half_as_ushort(__float2half_rn(x[2 * e + 1]));
      w[e] = lo | hi << 16;
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// Output gate, within a few units for any v above -87 (below, where the fast
// divide ends, 0 for less than 2^-125). The fast exponential would be off by 1.2
// |v| units; a correctly rounded divide costs prompts with a gate 4 % (2048
// tokens on 10000, bf16: 468 us instead of 455).
__device__ __forceinline__ float kv4_sigmoid(float v) { return __fdividef(1.f, 1.f + expf(-v)); }

// N consecutive words of shared or global memory as one vector load.
template <int N>
__device__ __forceinline__ void kv4_ldv(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
template <int N>
__device__ __forceinline__ void kv4_stv(uint8_t* p, const uint32_t (&w)[N]) {
  if constexpr (N == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (N == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(p) = w[0];
}
// Scale and bias of a group from its word.
__device__ __forceinline__ float2 kv4_param(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
#endif

}  // namespace swl
