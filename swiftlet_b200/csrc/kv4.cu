// The 4-bit KV cache: writing tokens into it, reading them back, eviction by
// accumulated attention weight, and the C entry points (attention itself is
// kv4_attn.cu and kv4_prompt.cu).
#include <algorithm>
#include <cmath>

#include "../../include/swiftlet_cuda.h"
#include "kcommon.cuh"
#include "kv4.h"
#include "launch.h"

namespace swl {

namespace {

// ------------------------------------------------------- append and read --
// A lane takes the eight consecutive channels of one code word, so a row of
// head_dim channels is head_dim / 8 lanes and a warp takes 256 / head_dim
// rows (keys or values of one token and head). Per group of `group` channels
// (8 or 16 lanes): b = f16(min), s = f16((max - min) * (1 / 15)), code =
// clamp(rint((x - b) * (1 / s)), 0, 15), every step rounded once to f32 (no
// contraction), so that the codes are the same wherever they are computed. A
// group with a non-finite value, or with b or s outside f16, gets NaN for
// both: it reads back as NaN instead of as something plausible.
constexpr int IO_THREADS = 256;

// Minimum and maximum that are NaN when either operand is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Smallest and largest of a group's values: eight a lane, GROUP / 8 lanes.
template <int GROUP>
__device__ __forceinline__ void group_range(const float (&x)[8], float& mn, float& mx) {
  mn = mx = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    mn = min_nan(mn, x[e]);
    mx = max_nan(mx, x[e]);
  }
#pragma unroll
  for (int o = 1; o < GROUP / 8; o <<= 1) {
    mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
}
// Two 16-bit values an instruction; min and -max travel as one word.
template <int DT>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if (DT == DT_BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int DT, int GROUP>
__device__ __forceinline__ void group_range(const uint4& w, float& mn, float& mx) {
  constexpr uint32_t NEG = 0x80008000u;
  const uint32_t lo = min2_nan<DT>(min2_nan<DT>(w.x, w.y), min2_nan<DT>(w.z, w.w));
  const uint32_t hi = min2_nan<DT>(min2_nan<DT>(w.x ^ NEG, w.y ^ NEG), min2_nan<DT>(w.z ^ NEG, w.w ^ NEG));
  uint32_t t = min2_nan<DT>(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
#pragma unroll
  for (int o = 1; o < GROUP / 8; o <<= 1) t = min2_nan<DT>(t, __shfl_xor_sync(0xffffffffu, t, o));
  t ^= 0x80000000u;
  mn = DT == DT_BF16 ? bf16_to_f32(uint16_t(t)) : f16_bits_to_f32(uint16_t(t));
  mx = DT == DT_BF16 ? bf16_to_f32(uint16_t(t >> 16)) : f16_bits_to_f32(uint16_t(t >> 16));
}

// Eight values as they come, and as f32.
template <int DT>
struct Row8 {
  uint4 w;
  __device__ __forceinline__ void zero() { w = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void load(const uint8_t* p, int64_t i, bool vec) {
    const uint16_t* f = reinterpret_cast<const uint16_t*>(p) + i;
    if (vec) {
      w = *reinterpret_cast<const uint4*>(f);
    } else {
      w.x = f[0] | uint32_t(f[1]) << 16, w.y = f[2] | uint32_t(f[3]) << 16, w.z = f[4] | uint32_t(f[5]) << 16, w.w = f[6] | uint32_t(f[7]) << 16;
    }
  }
  __device__ __forceinline__ float at(int e) const {
    const uint32_t u = e < 2 ? w.x : e < 4 ? w.y : e < 6 ? w.z : w.w;
    if (DT == DT_BF16) return __uint_as_float(e & 1 ? u & 0xffff0000u : u << 16);
    return f16_bits_to_f32(uint16_t(e & 1 ? u >> 16 : u));
  }
  template <int GROUP>
  __device__ __forceinline__ void range(float& mn, float& mx) const { group_range<DT, GROUP>(w, mn, mx); }
};
template <>
struct Row8<DT_F32> {
  float x[8];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
  }
  __device__ __forceinline__ void load(const uint8_t* p, int64_t i, bool vec) {
    const float* f = reinterpret_cast<const float*>(p) + i;
    if (vec) {
      const float4 a = reinterpret_cast<const float4*>(f)[0], b = reinterpret_cast<const float4*>(f)[1];
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = f[e];
    }
  }
  __device__ __forceinline__ float at(int e) const { return x[e]; }
  template <int GROUP>
  __device__ __forceinline__ void range(float& mn, float& mx) const { group_range<GROUP>(x, mn, mx); }
};
template <int DT>
__device__ __forceinline__ void store8(uint8_t* p, int64_t i, bool vec, const float (&x)[8]) {
  if (DT == DT_F32) {
    float* f = reinterpret_cast<float*>(p) + i;
    if (vec) {
      reinterpret_cast<float4*>(f)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(f)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = x[e];
    }
  } else {
    uint16_t u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      u[e] = DT == DT_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x[e])) : __half_as_ushort(__float2half_rn(x[e]));
    uint16_t* f = reinterpret_cast<uint16_t*>(p) + i;
    if (vec) {
      *reinterpret_cast<uint4*>(f) = *reinterpret_cast<const uint4*>(u);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = u[e];
    }
  }
}

// 16-byte accesses at every row of r (checked once per launch).
bool vec_rows(const Kv4Rows& r, int dt) {
  const int64_t e = dtype_bytes(dt);
  return reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.ts * e % 16 == 0 && r.hs * e % 16 == 0;
}

// A warp takes 1 << tshift consecutive tokens and, of each, IO_U rows at a time
// (K and V of some heads). The tokens' places (sequence, slot, page) are looked
// up by a lane each. Bound: the rows' bytes in and out, next to about 100
// instructions a row of quantising: nine prompts of 2500 to 9000 tokens (2 kv
// heads of 256 channels, bf16, 137 MB each way) are written in 45 us and read in
// 29 (3.0 and 4.7 TB/s).
constexpr int IO_TOKENS = 4;  // tokens of a warp at most
constexpr int IO_U = 4;       // rows a warp has in flight

template <int DT, bool READ, int HD, int GROUP>
__global__ void __launch_bounds__(IO_THREADS) k_kv4_io(const Kv4IoArgs a, bool vk, bool vv, int tshift) {
  constexpr int LPR = HD / 8, RPW = 32 / LPR, NG = HD / GROUP;  // lanes a row, rows a warp, groups a row
  pdl_wait();
  const Kv4Geo& g = a.g;
  const int lane = threadIdx.x & 31, sub = lane / LPR, l = lane % LPR;
  const int64_t j0 = (int64_t(blockIdx.x) * (IO_THREADS / 32) + (threadIdx.x >> 5)) << tshift;
  if (j0 >= a.b.total) return;
  const int n_tok = int(min(int64_t(1) << tshift, a.b.total - j0));
  // lane i: where token j0 + i goes
  uint8_t* blk = nullptr;
  int slot = 0, seq = 0;
  if (lane < n_tok) {
    // the last sequence that starts at or before the token
    int lo = 0, hi = a.b.nseq;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(a.b.start + mid + 1) <= j0 + lane) lo = mid + 1; else hi = mid;
    }
    seq = lo;
    int row0 = 0;
    if (seq < a.b.nseq) {
      const int n = kv4_new(a.b, seq, row0), len = kv4_len(a.b, seq);
      slot = len - n + int(j0 + lane - row0);
      // a negative slot: more new tokens than slots, the first of them have none
      if (j0 + lane >= row0 && slot >= 0 && slot < len) blk = kv4_block(g, g.table, g.tstride, seq, 0, slot, a.b.status);
    }
  }
  const int64_t hblk = int64_t(g.page / g.seg) * g.blk;
  for (int i = 0; i < n_tok; ++i) {
    uint8_t* const tb = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(blk), i));
    if (!tb) continue;
    const int s = __shfl_sync(0xffffffffu, slot, i), sq = __shfl_sync(0xffffffffu, seq, i), t = s & (g.seg - 1);
    const int wo = t * (HD / 2) + ((l & 7) ^ kv4_swz(HD, t)) * (HD / 16) + (l >> 3) * 4, po = g.seg * (HD / 2) + (t * NG + l * 8 / GROUP) * 4;
    const int64_t kj = (j0 + i) * a.k.ts + l * 8, vj = (j0 + i) * a.v.ts + l * 8;
    for (int h0 = sub; h0 - sub < g.kvh; h0 += IO_U / 2 * RPW) {
      Row8<DT> x[IO_U];
      uint32_t w[IO_U], pr[IO_U];
#pragma unroll
      for (int u = 0; u < IO_U; ++u) {
        const int h = h0 + (u >> 1) * RPW, kv = u & 1;
        w[u] = pr[u] = 0u;
        if (!READ) x[u].zero();
        if (h >= g.kvh) continue;
        if (READ) {
          const uint8_t* d = tb + h * hblk + (kv ? g.blk / 2 : 0);
          w[u] = *reinterpret_cast<const uint32_t*>(d + wo);
          pr[u] = *reinterpret_cast<const uint32_t*>(d + po);
        } else {
          x[u].load(kv ? a.v.p : a.k.p, kv ? vj + h * a.v.hs : kj + h * a.k.hs, kv ? vv : vk);
        }
      }
#pragma unroll
      for (int u = 0; u < IO_U; ++u) {
        const int h = h0 + (u >> 1) * RPW, kv = u & 1;
        if (READ) {
          if (h >= g.kvh) continue;
          const float2 sb = kv4_param(pr[u]);
          // a code at bit 4e of 2^23's mantissa is 2^23 + 16^e c; s c is exact, so
          // one rounding remains
          float y[8];
          const float s16[5] = {sb.x, sb.x * 0x1p-4f, sb.x * 0x1p-8f, sb.x * 0x1p-12f, sb.x * 0x1p-16f};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at4 = e < 5 ? e : e - 3;
            const uint32_t bits = (e < 5 ? w[u] : w[u] >> 12) & (15u << (4 * at4));
            y[e] = fmaf(__uint_as_float(bits | 0x4b000000u) - 8388608.f, s16[at4], sb.y);
          }
          store8<DT>(kv ? a.v.p : a.k.p, kv ? vj + h * a.v.hs : kj + h * a.k.hs, kv ? vv : vk, y);
          continue;
        }
        float mn, mx;
        x[u].template range<GROUP>(mn, mx);
        const __half hb = __float2half_rn(mn), hs = __float2half_rn(__fmul_rn(__fsub_rn(mx, mn), 1.f / 15.f));
        const float b = __half2float(hb), sc = __half2float(hs);
        const bool bad = !(fabsf(b) < INFINITY) || !(sc < INFINITY) || !(mx < INFINITY);
        const float inv = sc > 0.f ? __frcp_rn(sc) : 0.f;
        // held to [0, 15] first, a value is rounded by adding 1.5 * 2^23: the
        // code is the sum's last bits, over those of the constant
        uint32_t word = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float c = fminf(fmaxf(__fmul_rn(__fsub_rn(x[u].at(e), b), inv), 0.f), 15.f);
          word += __float_as_uint(__fadd_rn(c, 12582912.f)) << (4 * e);
        }
        word -= 0x3f400000u;  // the constant's bits, eight times
        if (h >= g.kvh) continue;
        uint8_t* d = tb + h * hblk + (kv ? g.blk / 2 : 0);
        *reinterpret_cast<uint32_t*>(d + wo) = bad ? 0u : word;
        if (l % (GROUP / 8) == 0)
          *reinterpret_cast<uint32_t*>(d + po) = bad ? 0x7e007e00u : uint32_t(__half_as_ushort(hs)) | uint32_t(__half_as_ushort(hb)) << 16;
        if (a.weights && l == 0 && kv == 0) a.weights[(int64_t(sq) * g.kvh + h) * a.wstride + s] = 0.f;
      }
    }
  }
}

template <int DT, bool READ>
void launch_io_dt(const Kv4IoArgs& a, cudaStream_t st) {
  // tokens a warp: as many as leave sixteen warps an SM, so that a step of a
  // few tokens still spreads over the GPU (64 tokens: 8 us with one a warp, 26
  // with eight; nine prompts of 2500 to 9000, written and read: 91 us with
  // one, 74 with four, 79 with eight)
  int tshift = 0;
  while ((2 << tshift) <= IO_TOKENS && (a.b.total >> (tshift + 1)) >= 148 * 16) ++tshift;
  const int per = IO_THREADS / 32 << tshift;
  const bool vk = vec_rows(a.k, DT), vv = vec_rows(a.v, DT);
  const dim3 grid((a.b.total + per - 1) / per), block(IO_THREADS);
  if (a.g.hd == 64) launch(k_kv4_io<DT, READ, 64, 64>, grid, block, 0, st, true, a, vk, vv, tshift);
  else if (a.g.hd == 128 && a.g.group == 64) launch(k_kv4_io<DT, READ, 128, 64>, grid, block, 0, st, true, a, vk, vv, tshift);
  else if (a.g.hd == 128) launch(k_kv4_io<DT, READ, 128, 128>, grid, block, 0, st, true, a, vk, vv, tshift);
  else if (a.g.group == 64) launch(k_kv4_io<DT, READ, 256, 64>, grid, block, 0, st, true, a, vk, vv, tshift);
  else launch(k_kv4_io<DT, READ, 256, 128>, grid, block, 0, st, true, a, vk, vv, tshift);
}

template <bool READ>
void launch_io(const Kv4IoArgs& a, int dt, cudaStream_t st) {
  if (dt == DT_F32) launch_io_dt<DT_F32, READ>(a, st);
  else if (dt == DT_BF16) launch_io_dt<DT_BF16, READ>(a, st);
  else launch_io_dt<DT_F16, READ>(a, st);
}

// ---------------------------------------------------------------- evict --
// Which slots survive, per (sequence, kv head): the first `first`, the last
// `recent`, and of the others the largest weights up to `keep` in all (ties to
// the lowest slot, NaN as -infinity). A cluster of EV_CL CTAs shares the slots
// in contiguous parts; each keeps the order-preserving 32-bit keys of its part
// in shared memory (as far as they fit) and they select by radix, 11, 11 and 10
// bits, adding up their histograms through distributed shared memory. Each CTA
// then writes the survivors of its part in order, behind those of the CTAs
// before it. Bound: the latency of the passes (reads of `len` words): two heads
// of 65536 slots cut to 32768, with the copy, 31 us (1.2 TB/s); with one CTA for
// each head the selection alone took 130.
constexpr int EV_THREADS = 1024;
constexpr int EV_CL = 8;       // CTAs a cluster at most
constexpr int EV_BINS = 2048;
constexpr int EV_KEYS = 16384;  // keys a CTA holds
constexpr size_t EV_SMEM = EV_KEYS * 4;

__device__ __forceinline__ uint32_t ev_key(float w) {
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 ties with 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ void ev_ld2(uint32_t addr, int& a, int& b) {
  asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr) : "memory");
}
__device__ __forceinline__ int ev_ld(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Exclusive scan of one int a thread; returns the total.
__device__ int ev_scan(int v, int* ex, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int w = warp_sums[lane];
    int wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, wi, o);
      if (lane >= o) wi += y;
    }
    warp_sums[lane] = wi - w;
    if (lane == 31) warp_sums[32] = wi;
  }
  __syncthreads();
  *ex = warp_sums[warp] + inc - v;
  const int total = warp_sums[32];
  __syncthreads();
  return total;
}

__global__ void __launch_bounds__(EV_THREADS, 1) k_kv4_evict_select(const Kv4EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ __align__(8) int hist[2][EV_BINS];
  __shared__ int warp_sums[33], s_bin, s_above, s_cnt[2];
  pdl_wait();
  const int seq = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  const int rank = int(cluster_rank()), ncl = gridDim.x;  // one cluster in x
  const int len = kv4_len(a.b, seq), nl = min(len, a.keep);
  if (h == 0 && rank == 0 && tid == 0) a.new_lens[seq] = nl;
  const float* w = a.weights + (int64_t(seq) * a.g.kvh + h) * a.wstride;
  int* kept = a.kept + (int64_t(seq) * a.g.kvh + h) * a.kstride;
  const int part = (len + ncl - 1) / ncl, p0 = min(len, rank * part), p1 = min(len, p0 + part);
  if (nl == len) {  // the whole cluster takes this way
    for (int i = p0 + tid; i < p1; i += EV_THREADS) kept[i] = i;
    return;
  }
  // candidates: [first, len - recent); first + recent <= keep < len
  const int c0 = max(p0, a.first), c1 = min(p1, len - a.recent);
  const int held = min(c1, c0 + EV_KEYS);
  for (int i = c0 + tid; i < held; i += EV_THREADS) keys[i - c0] = ev_key(w[i]);
  auto key_of = [&](int i) { return i < held ? keys[i - c0] : ev_key(w[i]); };
  int rem = a.keep - a.first - a.recent;  // still to be found among the keys with the prefix
  uint32_t prefix = 0u, mask = 0u;
  const bool none = rem == 0;
  if (!none)
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      int* hs = hist[pass & 1];
      for (int b = tid; b < EV_BINS; b += EV_THREADS) hs[b] = 0;
      __syncthreads();
      for (int i = c0 + tid; i < c1; i += EV_THREADS) {
        const uint32_t key = key_of(i);
        if ((key & mask) == prefix) atomicAdd(&hs[(key >> shift) & ((1u << bits) - 1u)], 1);
      }
      cluster_sync();
      // two bins a thread, the largest first
      int n[2], ex;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        n[k] = 0;
      }
      for (int c = 0; c < ncl; ++c) {
        int lo, hi;
        ev_ld2(dsmem_map(&hs[EV_BINS - 2 - 2 * tid], c), lo, hi);
        n[0] += hi;
        n[1] += lo;
      }
      ev_scan(n[0] + n[1], &ex, warp_sums);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int above = ex + (k ? n[0] : 0);
        if (above < rem && above + n[k] >= rem) {
          s_bin = EV_BINS - 1 - (2 * tid + k);
          s_above = above;
        }
      }
      __syncthreads();
      prefix |= uint32_t(s_bin) << shift;
      rem -= s_above;
      mask |= ((1u << bits) - 1u) << shift;
      __syncthreads();
    }
  const uint32_t thr = prefix;
  // survivors and ties at the threshold of the parts before this one
  int gt = 0, eq = 0;
  for (int i = p0 + tid; i < p1; i += EV_THREADS) {
    const bool cand = i >= c0 && i < c1;
    const uint32_t key = cand ? key_of(i) : 0u;
    gt += !cand || (!none && key > thr);
    eq += cand && !none && key == thr;
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (tid < 2) s_cnt[tid] = 0;
  __syncthreads();
  if ((tid & 31) == 0) {
    atomicAdd(&s_cnt[0], gt);
    atomicAdd(&s_cnt[1], eq);
  }
  cluster_sync();
  int gt0 = 0, eq0 = 0;
  for (int c = 0; c < rank; ++c) {
    gt0 += ev_ld(dsmem_map(&s_cnt[0], c));
    eq0 += ev_ld(dsmem_map(&s_cnt[1], c));
  }
  cluster_arrive();  // done with the others' shared memory; theirs with this one's before the exit
  int need = max(0, rem - eq0), out = gt0 + min(rem, eq0);
  for (int i0 = p0; i0 < p1; i0 += EV_THREADS) {
    const int i = i0 + tid;
    const bool in = i < p1, cand = in && i >= c0 && i < c1;
    const uint32_t key = cand ? key_of(i) : 0u;
    const bool tie = cand && !none && key == thr, sure = in && (!cand || (!none && key > thr));
    // one scan of both: ties in the high half
    int at;
    const int tot = ev_scan(int(sure) | int(tie) << 16, &at, warp_sums);
    const int ties = at >> 16, place = out + (at & 0xffff) + min(ties, need);
    if (sure || (tie && ties < need)) kept[place] = i;
    out += (tot & 0xffff) + min(tot >> 16, need);
    need -= min(need, tot >> 16);
  }
  cluster_wait();
}

// Copies survivors to slots 0, 1, ... of the destination: eight lanes a row (a
// unit each; a row's units are stored in another order in another slot), keys
// and values, two rows a lane group.
constexpr int EC_ROWS = 64;  // survivors a block
template <int HD>
__global__ void __launch_bounds__(256) k_kv4_evict_copy(const Kv4EvictArgs a) {
  constexpr int NW = HD / 64;
  pdl_wait();
  const Kv4Geo& g = a.g;
  const int seq = blockIdx.z, h = blockIdx.y, u = threadIdx.x & 7;
  const int len = kv4_len(a.b, seq), nl = min(len, a.keep);
  const int i0 = blockIdx.x * EC_ROWS + (threadIdx.x >> 3);
  const int64_t pair = int64_t(seq) * g.kvh + h;
  int src[2], slot[2];
  const uint8_t* from[2];
  uint8_t* to[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    slot[k] = i0 + 32 * k;
    src[k] = slot[k] < nl ? a.kept[pair * a.kstride + slot[k]] : -1;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    from[k] = src[k] >= 0 ? kv4_block(g, g.table, g.tstride, seq, h, src[k], a.b.status) : nullptr;
    to[k] = src[k] >= 0 ? kv4_block(g, a.dst, a.dstride, seq, h, slot[k], a.b.status) : nullptr;
  }
  uint32_t c[2][2][NW], p[2][2];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
      if (from[k] && to[k]) {
        const int t = src[k] & (g.seg - 1);
        const uint8_t* f = from[k] + kv * (g.blk / 2);
        kv4_ldv(f + t * (HD / 2) + (u ^ kv4_swz(HD, t)) * (HD / 16), c[k][kv]);
        if (u < g.ng) p[k][kv] = reinterpret_cast<const uint32_t*>(f + g.seg * (HD / 2))[t * g.ng + u];
      }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (from[k] && to[k])
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int t = slot[k] & (g.seg - 1);
        uint8_t* d = to[k] + kv * (g.blk / 2);
        kv4_stv(d + t * (HD / 2) + (u ^ kv4_swz(HD, t)) * (HD / 16), c[k][kv]);
        if (u < g.ng) reinterpret_cast<uint32_t*>(d + g.seg * (HD / 2))[t * g.ng + u] = p[k][kv];
      }
    if (a.new_weights && u == 0 && src[k] >= 0) a.new_weights[pair * a.nwstride + slot[k]] = a.weights[pair * a.wstride + src[k]];
  }
}

// ------------------------------------------------------------- arguments --
Kv4Geo geo_of(const swl_kv4_cache* c) {
  if (!c || !c->pages || !c->page_table) throw Error(ERR_INVALID, "kv4: null cache, pages or page table");
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    throw Error(ERR_UNSUPPORTED, "kv4: head_dim must be 64, 128 or 256");
  if ((c->group != 64 && c->group != 128) || c->group > c->head_dim)
    throw Error(ERR_UNSUPPORTED, "kv4: group must be 64 or 128 and at most head_dim");
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    throw Error(ERR_UNSUPPORTED, "kv4: page_size must be 16, 32, 64 or 128");
  if (c->kv_heads < 1 || c->kv_heads > 1024 || c->num_pages < 1 || c->table_stride < 1)
    throw Error(ERR_INVALID, "kv4: kv_heads (1..1024), num_pages and table_stride must be positive");
  if (reinterpret_cast<uintptr_t>(c->pages) % 16) throw Error(ERR_INVALID, "kv4: pages must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(c->page_table) % 4) throw Error(ERR_INVALID, "kv4: page table must be 4-byte aligned");
  Kv4Geo g;
  g.pages = static_cast<uint8_t*>(c->pages);
  g.table = c->page_table;
  g.tstride = c->table_stride;
  g.npages = c->num_pages;
  g.page = c->page_size;
  g.pshift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  g.seg = std::min(g.page, 64);
  g.kvh = c->kv_heads;
  g.hd = c->head_dim;
  g.group = c->group;
  g.ng = g.hd / g.group;
  g.blk = 2 * g.seg * (g.hd / 2 + 4 * g.ng);
  g.page_bytes = int64_t(g.kvh) * (g.page / g.seg) * g.blk;
  return g;
}

Kv4Batch batch_of(const swl_kv4_batch* b, const Kv4Geo& g, bool tokens) {
  if (!b) throw Error(ERR_INVALID, "kv4: null batch");
  if (b->nseq < 0 || b->nseq > 65535 || b->total < 0 || b->max_new < 0 || b->max_len < 0)
    throw Error(ERR_INVALID, "kv4: nseq (0..65535), total, max_new and max_len must not be negative");
  // counts of tiles, units and rows are rounded up in 32 bits
  if (b->total > 0x7fffffff - 4095 || b->max_len > 0x7fffffff - 4095)
    throw Error(ERR_UNSUPPORTED, "kv4: total and max_len must be at most 2^31 - 4096");
  if (b->nseq > 0 && (!b->lens || (tokens && !b->start))) throw Error(ERR_INVALID, "kv4: null lens or start");
  if (reinterpret_cast<uintptr_t>(b->lens) % 4 || reinterpret_cast<uintptr_t>(b->start) % 4 ||
      reinterpret_cast<uintptr_t>(b->status) % 4)
    throw Error(ERR_INVALID, "kv4: lens, start and status must be 4-byte aligned");
  if (b->max_len > g.tstride * g.page)
    throw Error(ERR_CAPACITY, "kv4: max_len " + std::to_string(b->max_len) + " above the page table's " +
                                  std::to_string(g.tstride * g.page) + " slots");
  Kv4Batch r;
  r.start = b->start; r.lens = b->lens; r.nseq = b->nseq; r.total = b->total; r.max_new = b->max_new; r.max_len = b->max_len;
  r.status = b->status;
  return r;
}

Kv4Rows rows_of(const swl_kv4_rows* r, int dt, int hd, const char* what) {
  if (!r || !r->data) throw Error(ERR_INVALID, std::string("kv4: null ") + what);
  if (reinterpret_cast<uintptr_t>(r->data) % dtype_bytes(dt)) throw Error(ERR_INVALID, std::string("kv4: misaligned ") + what);
  if (r->token_stride < 0 || r->head_stride < 0) throw Error(ERR_INVALID, std::string("kv4: negative stride of ") + what);
  Kv4Rows o;
  o.p = static_cast<uint8_t*>(const_cast<void*>(r->data));
  o.ts = r->token_stride;
  o.hs = r->head_stride;
  return o;
}

void check_dtype(int dt) {
  if (dt < 0 || dt > 2) throw Error(ERR_UNSUPPORTED, "kv4: dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
}

// Runs the launches on the device that holds the pages.
struct OnDevice {
  int before = -1;
  explicit OnDevice(const void* p) {
    cudaPointerAttributes at;
    SWL_CUDA(cudaPointerGetAttributes(&at, p));
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
      throw Error(ERR_INVALID, "kv4: pages are not device memory");
    int cur = 0;
    SWL_CUDA(cudaGetDevice(&cur));
    if (cur != at.device) {
      SWL_CUDA(cudaSetDevice(at.device));
      before = cur;
    }
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

template <typename F>
int guarded(F f) {
  try {
    f();
    return SWL_OK;
  } catch (const Error& e) {
    set_last_error(e.what());
    return e.code;
  } catch (const std::exception& e) {
    set_last_error(e.what());
    return SWL_ERR_INVALID;
  }
}

void io_call(bool read, const swl_kv4_cache* cache, const swl_kv4_batch* batch, int dt, const swl_kv4_rows* k,
             const swl_kv4_rows* v, float* weights, int64_t wstride, void* stream) {
  Kv4IoArgs a;
  a.g = geo_of(cache);
  a.b = batch_of(batch, a.g, true);
  check_dtype(dt);
  if (weights && wstride < a.b.max_len) throw Error(ERR_INVALID, "kv4: weights_stride below max_len");
  if (reinterpret_cast<uintptr_t>(weights) % 4) throw Error(ERR_INVALID, "kv4: weights must be 4-byte aligned");
  if (a.b.nseq == 0 || a.b.total == 0) return;
  a.k = rows_of(k, dt, a.g.hd, "k rows");
  a.v = rows_of(v, dt, a.g.hd, "v rows");
  a.weights = weights;
  a.wstride = wstride;
  OnDevice dev(a.g.pages);
  if (read) launch_kv4_read(a, dt, static_cast<cudaStream_t>(stream));
  else launch_kv4_append(a, dt, static_cast<cudaStream_t>(stream));
}

}  // namespace

void launch_kv4_append(const Kv4IoArgs& a, int dt, cudaStream_t st) { launch_io<false>(a, dt, st); }
void launch_kv4_read(const Kv4IoArgs& a, int dt, cudaStream_t st) { launch_io<true>(a, dt, st); }

void launch_kv4_evict(const Kv4EvictArgs& a, cudaStream_t st) {
  // as many CTAs a (sequence, head) as one wave of the GPU has for them: 64
  // x 2 of at most 4608 slots took 52 us with eight each (seven waves), two
  // of 65536 took 33 us with eight, 130 us with one
  int cl = EV_CL;
  while (cl > 1 && int64_t(cl) * a.g.kvh * a.b.nseq > 148) cl >>= 1;
  launch_cluster(k_kv4_evict_select, dim3(cl, a.g.kvh, a.b.nseq), dim3(EV_THREADS), dim3(cl, 1, 1), EV_SMEM, st, true, a);
  const int most = std::min(a.keep, a.b.max_len);
  if (most < 1) return;
  const dim3 grid((most + EC_ROWS - 1) / EC_ROWS, a.g.kvh, a.b.nseq), block(256);
  if (a.g.hd == 64) launch(k_kv4_evict_copy<64>, grid, block, 0, st, true, a);
  else if (a.g.hd == 128) launch(k_kv4_evict_copy<128>, grid, block, 0, st, true, a);
  else launch(k_kv4_evict_copy<256>, grid, block, 0, st, true, a);
}

}  // namespace swl

using namespace swl;

extern "C" {

int64_t swl_kv4_page_bytes(int32_t kv_heads, int32_t head_dim, int32_t group, int32_t page_size) {
  int64_t n = 0;
  const int rc = guarded([&] {
    swl_kv4_cache c = {reinterpret_cast<void*>(16), reinterpret_cast<const int32_t*>(16), 1, 1, page_size, kv_heads, head_dim, group};
    n = geo_of(&c).page_bytes;
  });
  return rc == SWL_OK ? n : rc;
}

int swl_kv4_append_device(const swl_kv4_cache* cache, const swl_kv4_batch* batch, int32_t dtype, const swl_kv4_rows* k,
                          const swl_kv4_rows* v, float* d_weights, int64_t weights_stride, void* cuda_stream) {
  return guarded([&] { io_call(false, cache, batch, dtype, k, v, d_weights, weights_stride, cuda_stream); });
}

int swl_kv4_read_device(const swl_kv4_cache* cache, const swl_kv4_batch* batch, int32_t dtype, const swl_kv4_rows* k,
                        const swl_kv4_rows* v, void* cuda_stream) {
  return guarded([&] { io_call(true, cache, batch, dtype, k, v, nullptr, 0, cuda_stream); });
}

int64_t swl_kv4_attention_workspace(const swl_kv4_cache* cache, const swl_kv4_batch* batch, int32_t heads) {
  int64_t n = 0;
  const int rc = guarded([&] {
    const Kv4Geo g = geo_of(cache);
    const Kv4Batch b = batch_of(batch, g, true);
    if (heads < 1 || heads % g.kvh) throw Error(ERR_INVALID, "kv4: heads must be a positive multiple of kv_heads");
    n = kv4_attention_work(g, b, heads);
  });
  return rc == SWL_OK ? n : rc;
}

int swl_kv4_attention_device(const swl_kv4_cache* cache, const swl_kv4_batch* batch, const swl_kv4_attention* attention,
                             void* cuda_stream) {
  return guarded([&] {
    Kv4AttnArgs a;
    a.g = geo_of(cache);
    a.b = batch_of(batch, a.g, true);
    const swl_kv4_attention* t = attention;
    if (!t) throw Error(ERR_INVALID, "kv4: null attention arguments");
    check_dtype(t->dtype);
    if (t->heads < 1 || t->heads % a.g.kvh) throw Error(ERR_INVALID, "kv4: heads must be a positive multiple of kv_heads");
    if (t->heads / a.g.kvh > 64) throw Error(ERR_UNSUPPORTED, "kv4: more than 64 query heads a kv head");
    if (!std::isfinite(t->scale)) throw Error(ERR_INVALID, "kv4: scale must be finite");
    if (t->weights && t->weights_stride < a.b.max_len) throw Error(ERR_INVALID, "kv4: weights_stride below max_len");
    if (reinterpret_cast<uintptr_t>(t->weights) % 4 || reinterpret_cast<uintptr_t>(t->lse) % 4)
      throw Error(ERR_INVALID, "kv4: weights and lse must be 4-byte aligned");
    if (a.b.nseq == 0 || a.b.total == 0) return;
    a.dt = t->dtype; a.heads = t->heads; a.rep = t->heads / a.g.kvh; a.scale = t->scale;
    a.q = rows_of(&t->q, a.dt, a.g.hd, "q rows");
    a.out = rows_of(&t->out, a.dt, a.g.hd, "out rows");
    if (t->gate.data) a.gate = rows_of(&t->gate, a.dt, a.g.hd, "gate rows");
    if (a.out.p == a.q.p || a.out.p == a.gate.p) throw Error(ERR_INVALID, "kv4: out must not be q or gate");
    a.lse = t->lse; a.weights = t->weights; a.wstride = t->weights_stride;
    const int64_t need = kv4_attention_work(a.g, a.b, a.heads);
    if (!t->work || t->work_bytes < need)
      throw Error(ERR_CAPACITY, "kv4: workspace of " + std::to_string(t->work ? t->work_bytes : 0) + " bytes, " +
                                    std::to_string(need) + " needed");
    if (reinterpret_cast<uintptr_t>(t->work) % 16) throw Error(ERR_INVALID, "kv4: workspace must be 16-byte aligned");
    a.work = static_cast<uint8_t*>(t->work);
    OnDevice dev(a.g.pages);
    launch_kv4_attention(a, static_cast<cudaStream_t>(cuda_stream));
  });
}

int64_t swl_kv4_evict_workspace(const swl_kv4_cache* cache, const swl_kv4_batch* batch, int32_t keep) {
  int64_t n = 0;
  const int rc = guarded([&] {
    const Kv4Geo g = geo_of(cache);
    const Kv4Batch b = batch_of(batch, g, false);
    if (keep < 0) throw Error(ERR_INVALID, "kv4: keep must not be negative");
    n = int64_t(b.nseq) * g.kvh * std::min(keep, b.max_len) * 4;
  });
  return rc == SWL_OK ? n : rc;
}

int swl_kv4_evict_device(const swl_kv4_cache* cache, const swl_kv4_batch* batch, const swl_kv4_evict* evict,
                         void* cuda_stream) {
  return guarded([&] {
    Kv4EvictArgs a;
    a.g = geo_of(cache);
    a.b = batch_of(batch, a.g, false);
    const swl_kv4_evict* t = evict;
    if (!t) throw Error(ERR_INVALID, "kv4: null evict arguments");
    if (t->keep < 0 || t->first < 0 || t->recent < 0 || int64_t(t->first) + t->recent > t->keep)
      throw Error(ERR_INVALID, "kv4: first and recent must not be negative and together at most keep");
    if (a.b.nseq == 0) return;
    const int64_t most = std::min(t->keep, a.b.max_len);
    if (!t->weights || !t->dst_table || !t->new_lens) throw Error(ERR_INVALID, "kv4: null weights, dst_table or new_lens");
    if (t->weights_stride < a.b.max_len) throw Error(ERR_INVALID, "kv4: weights_stride below max_len");
    if (t->new_weights && t->new_weights_stride < most) throw Error(ERR_INVALID, "kv4: new_weights_stride below the survivors");
    if (t->kept && t->kept_stride < most) throw Error(ERR_INVALID, "kv4: kept_stride below the survivors");
    if (t->dst_stride < 1 || t->dst_stride * a.g.page < most)
      throw Error(ERR_CAPACITY, "kv4: destination table too short for the survivors");
    if (t->dst_table == a.g.table) throw Error(ERR_INVALID, "kv4: destination table is the source's");
    if (t->new_weights == t->weights || t->new_lens == a.b.lens) throw Error(ERR_INVALID, "kv4: new weights and lens must not be the old ones");
    for (const void* p : {static_cast<const void*>(t->weights), static_cast<const void*>(t->dst_table),
                          static_cast<const void*>(t->new_lens), static_cast<const void*>(t->new_weights),
                          static_cast<const void*>(t->kept), static_cast<const void*>(t->work)})
      if (reinterpret_cast<uintptr_t>(p) % 4) throw Error(ERR_INVALID, "kv4: buffers must be 4-byte aligned");
    a.keep = t->keep; a.first = t->first; a.recent = t->recent; a.weights = t->weights; a.wstride = t->weights_stride;
    a.dst = t->dst_table; a.dstride = t->dst_stride; a.new_lens = t->new_lens; a.new_weights = t->new_weights;
    a.nwstride = t->new_weights_stride;
    if (t->kept) {
      a.kept = t->kept;
      a.kstride = t->kept_stride;
    } else {
      const int64_t need = int64_t(a.b.nseq) * a.g.kvh * most * 4;
      if (need && (!t->work || t->work_bytes < need))
        throw Error(ERR_CAPACITY, "kv4: workspace of " + std::to_string(t->work ? t->work_bytes : 0) + " bytes, " +
                                      std::to_string(need) + " needed");
      a.kept = static_cast<int*>(t->work);
      a.kstride = most;
    }
    OnDevice dev(a.g.pages);
    launch_kv4_evict(a, static_cast<cudaStream_t>(cuda_stream));
  });
}

}  // extern "C"
