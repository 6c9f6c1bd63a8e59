// Attention over the 4-bit KV cache (layout: kv4.h).
#include <algorithm>

#include "kcommon.cuh"
#include "kv4.h"
#include "launch.h"

namespace swl {

namespace {

// One warp per (row, head): the lane's head_dim / 32 channels of q, an online
// softmax over the slots the row sees, one slot at a time.
constexpr int SA_WARPS = 8;

template <int HD>
__device__ __forceinline__ void sa_slot(const Kv4Geo& g, const uint8_t* base, int t, int lane, float (&x)[HD / 32]) {
  constexpr int E = HD / 32;
  const int c0 = lane * E, unit = (c0 % 64) / 8;
  const uint8_t* p = base + t * (HD / 2) + (unit ^ kv4_swz(HD, t)) * (HD / 16) + c0 / 64 * 4 + c0 % 8 / 2;
  uint32_t w = 0;
  for (int b = 0; b < E / 2; ++b) w |= uint32_t(p[b]) << (8 * b);
  const float2 sb = kv4_param(reinterpret_cast<const uint32_t*>(base + g.seg * (HD / 2))[t * g.ng + c0 / g.group]);
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = fmaf(sb.x, float((w >> (4 * e)) & 15u), sb.y);
}

template <int HD>
__global__ void __launch_bounds__(SA_WARPS * 32) k_kv4_attn_rows(const Kv4AttnArgs a) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const int64_t wid = int64_t(blockIdx.x) * SA_WARPS + (threadIdx.x >> 5);
  const int j = int(wid / a.heads), hq = int(wid % a.heads), h = hq / a.rep;
  if (j >= a.b.total) return;
  const int seq = kv4_seq_of(a.b, j);
  if (seq < 0) return;
  int row0;
  const int n = kv4_new(a.b, seq, row0), len = kv4_len(a.b, seq);
  const int last = min(len - 1, len - n + (j - row0));
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = kv4_ld(a.q.p, a.dt, j * a.q.ts + hq * a.q.hs + lane * E + e);
    o[e] = 0.f;
  }
  for (int s = 0; s <= last; ++s) {
    const uint8_t* blk = kv4_block(a.g, a.g.table, a.g.tstride, seq, h, s, a.b.status);
    if (!blk) continue;
    float k[E], v[E], d = 0.f;
    sa_slot<HD>(a.g, blk, s & (a.g.seg - 1), lane, k);
    sa_slot<HD>(a.g, blk + a.g.blk / 2, s & (a.g.seg - 1), lane, v);
#pragma unroll
    for (int e = 0; e < E; ++e) d = fmaf(q[e], k[e], d);
    const float x = warp_sum(d) * a.scale, mn = fmaxf(m, x);
    const float al = expf(m - mn), p = expf(x - mn);
    l = l * al + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(p, v[e], o[e] * al);
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float r = l > 0.f || l != l ? o[e] / l : 0.f;
    if (a.gate.p) r *= sigmoid_ref(kv4_ld(a.gate.p, a.dt, j * a.gate.ts + hq * a.gate.hs + lane * E + e));
    kv4_st(a.out.p, a.dt, j * a.out.ts + hq * a.out.hs + lane * E + e, r);
  }
  if (lane == 0) {
    float* lse = a.lse ? a.lse : reinterpret_cast<float*>(a.work);
    lse[int64_t(j) * a.heads + hq] = m + logf(l);
  }
}

// Weights: one warp per (sequence, kv head, slot) adds exp(s - lse) over the
// rows that see the slot, in row order.
template <int HD>
__global__ void __launch_bounds__(SA_WARPS * 32) k_kv4_weights_rows(const Kv4AttnArgs a) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31, seq = blockIdx.z, h = blockIdx.y;
  const int s = blockIdx.x * SA_WARPS + (threadIdx.x >> 5);
  int row0;
  const int n = kv4_new(a.b, seq, row0), len = kv4_len(a.b, seq);
  if (s >= len) return;
  const uint8_t* blk = kv4_block(a.g, a.g.table, a.g.tstride, seq, h, s, a.b.status);
  if (!blk) return;
  float k[E], sum = 0.f;
  sa_slot<HD>(a.g, blk, s & (a.g.seg - 1), lane, k);
  const float* lse = a.lse ? a.lse : reinterpret_cast<const float*>(a.work);
  for (int i = max(0, s - (len - n)); i < n; ++i)
    for (int r = 0; r < a.rep; ++r) {
      const int j = row0 + i, hq = h * a.rep + r;
      float d = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) d = fmaf(kv4_ld(a.q.p, a.dt, j * a.q.ts + hq * a.q.hs + lane * E + e), k[e], d);
      sum += expf(warp_sum(d) * a.scale - lse[int64_t(j) * a.heads + hq]);
    }
  if (lane == 0) a.weights[(int64_t(seq) * a.g.kvh + h) * a.wstride + s] += sum;
}

template <int HD>
void run_rows(const Kv4AttnArgs& a, cudaStream_t st) {
  const int64_t warps = int64_t(a.b.total) * a.heads;
  launch(k_kv4_attn_rows<HD>, dim3(unsigned((warps + SA_WARPS - 1) / SA_WARPS)), dim3(SA_WARPS * 32), 0, st, false, a);
  if (a.weights && a.b.max_len > 0)
    launch(k_kv4_weights_rows<HD>, dim3((a.b.max_len + SA_WARPS - 1) / SA_WARPS, a.g.kvh, a.b.nseq), dim3(SA_WARPS * 32), 0, st,
           false, a);
}

}  // namespace

int64_t kv4_attention_work(const Kv4Geo& g, const Kv4Batch& b, int heads) { return std::max<int64_t>(16, int64_t(b.total) * heads * 4); }

void launch_kv4_attention(const Kv4AttnArgs& a, cudaStream_t st) {
  if (a.g.hd == 64) run_rows<64>(a, st);
  else if (a.g.hd == 128) run_rows<128>(a, st);
  else run_rows<256>(a, st);
}

}  // namespace swl
