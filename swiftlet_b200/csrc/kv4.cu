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

template <int DT>
__device__ __forceinline__ void load8(const uint8_t* p, int64_t i, bool vec, float (&x)[8]) {
  if (DT == DT_F32) {
    const float* f = reinterpret_cast<const float*>(p) + i;
    if (vec) {
      const float4 a = reinterpret_cast<const float4*>(f)[0], b = reinterpret_cast<const float4*>(f)[1];
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = f[e];
    }
  } else {
    const uint16_t* f = reinterpret_cast<const uint16_t*>(p) + i;
    uint16_t u[8];
    if (vec) {
      *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(f);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = f[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = DT == DT_BF16 ? bf16_to_f32(u[e]) : f16_bits_to_f32(u[e]);
  }
}

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

template <int DT, bool READ>
__global__ void __launch_bounds__(IO_THREADS) k_kv4_io(const Kv4IoArgs a, bool vk, bool vv) {
  const Kv4Geo& g = a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lpr = g.hd / 8, rpw = 32 / lpr;       // lanes a row, rows a warp
  const int per = (g.kvh * 2 + rpw - 1) / rpw;    // warps a token
  const int64_t wid = int64_t(blockIdx.x) * (IO_THREADS / 32) + warp;
  const int j = int(wid / per);
  if (j >= a.b.total) return;
  const int seq = kv4_seq_of(a.b, j);
  if (seq < 0) return;
  int row0;
  const int n = kv4_new(a.b, seq, row0);
  const int len = kv4_len(a.b, seq);
  const int slot = len - n + (j - row0);
  if (slot < 0 || slot >= len) return;  // more new tokens than slots: the first of them have none
  const int row = int(wid % per) * rpw + lane / lpr, l = lane % lpr;
  const bool on = row < g.kvh * 2;
  const int h = on ? row >> 1 : 0, kv = row & 1;
  uint8_t* blk = kv4_block(g, g.table, g.tstride, seq, h, slot, a.b.status);
  if (!blk) return;  // the same page for the whole warp
  const int t = slot & (g.seg - 1);
  uint8_t* base = blk + (kv ? g.blk / 2 : 0);
  uint32_t* word = reinterpret_cast<uint32_t*>(base + t * (g.hd / 2) + ((l & 7) ^ kv4_swz(g.hd, t)) * (g.hd / 16) + (l >> 3) * 4);
  uint32_t* par = reinterpret_cast<uint32_t*>(base + g.seg * (g.hd / 2)) + t * g.ng + l * 8 / g.group;
  const Kv4Rows& r = kv ? a.v : a.k;
  const int64_t at = j * r.ts + h * r.hs + l * 8;
  const bool vec = kv ? vv : vk;
  float x[8];
  if (READ) {
    if (!on) return;
    const float2 sb = kv4_param(*par);
    const uint32_t w = *word;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(__fmul_rn(sb.x, float((w >> (4 * e)) & 15u)), sb.y);
    store8<DT>(r.p, at, vec, x);
  } else {
    if (on) load8<DT>(r.p, at, vec, x);
    else
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
    float mn = x[0], mx = x[0];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mn = fminf(mn, x[e]);
      mx = fmaxf(mx, x[e]);
      bad |= !(fabsf(x[e]) < INFINITY);
    }
    for (int o = 1; o < g.group / 8; o <<= 1) {
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      bad |= __shfl_xor_sync(0xffffffffu, int(bad), o) != 0;
    }
    const __half hb = __float2half_rn(mn), hs = __float2half_rn(__fmul_rn(__fsub_rn(mx, mn), 1.f / 15.f));
    const float b = __half2float(hb), s = __half2float(hs);
    bad |= !(fabsf(b) < INFINITY) || !(s < INFINITY);
    const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
    uint32_t w = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[e], b), inv)), 0.f), 15.f);
      w |= uint32_t(int(c)) << (4 * e);
    }
    if (!on) return;
    *word = bad ? 0u : w;
    if (l * 8 % g.group == 0)
      *par = bad ? 0x7e007e00u : uint32_t(__half_as_ushort(hs)) | uint32_t(__half_as_ushort(hb)) << 16;
    if (a.weights && l == 0 && kv == 0) a.weights[(int64_t(seq) * g.kvh + h) * a.wstride + slot] = 0.f;
  }
}

template <bool READ>
void launch_io(const Kv4IoArgs& a, int dt, cudaStream_t st) {
  const int rpw = 256 / a.g.hd, per = (a.g.kvh * 2 + rpw - 1) / rpw;
  const int64_t warps = int64_t(a.b.total) * per, blocks = (warps + IO_THREADS / 32 - 1) / (IO_THREADS / 32);
  if (blocks > 0x7fffffff) throw Error(ERR_UNSUPPORTED, "kv4: too many rows for one launch");
  const bool vk = vec_rows(a.k, dt), vv = vec_rows(a.v, dt);
  const dim3 grid = dim3(unsigned(blocks)), block(IO_THREADS);
  if (dt == DT_F32) launch(k_kv4_io<DT_F32, READ>, grid, block, 0, st, false, a, vk, vv);
  else if (dt == DT_BF16) launch(k_kv4_io<DT_BF16, READ>, grid, block, 0, st, false, a, vk, vv);
  else launch(k_kv4_io<DT_F16, READ>, grid, block, 0, st, false, a, vk, vv);
}

// ---------------------------------------------------------------- evict --
// Which slots survive, per (sequence, kv head): the first `first`, the last
// `recent`, and of the others the largest weights up to `keep` in all (ties to
// the lowest slot, NaN as -infinity). Radix select over order-preserving
// 32-bit keys, then the survivors' slots in ascending order.
constexpr int EV_THREADS = 1024;

__device__ __forceinline__ uint32_t ev_key(float w) {
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 ties with 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

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

__global__ void __launch_bounds__(EV_THREADS) k_kv4_evict_select(const Kv4EvictArgs a) {
  __shared__ unsigned hist[256];
  __shared__ int warp_sums[33];
  __shared__ uint32_t s_prefix;
  __shared__ int s_rem;
  const int seq = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
  const int len = kv4_len(a.b, seq), nl = min(len, a.keep);
  if (h == 0 && tid == 0) a.new_lens[seq] = nl;
  const float* w = a.weights + (int64_t(seq) * a.g.kvh + h) * a.wstride;
  int* kept = a.kept + (int64_t(seq) * a.g.kvh + h) * a.kstride;
  if (nl == len) {
    for (int i = tid; i < len; i += EV_THREADS) kept[i] = i;
    return;
  }
  const int lo = a.first, hi = len - a.recent;  // candidates [lo, hi); first + recent <= keep < len
  uint32_t mask = 0u;
  if (tid == 0) { s_prefix = 0u; s_rem = a.keep - a.first - a.recent; }
  __syncthreads();
  const bool none = s_rem == 0;
  if (!none)
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int b = tid; b < 256; b += EV_THREADS) hist[b] = 0u;
      __syncthreads();
      const uint32_t prefix = s_prefix;
      for (int i = lo + tid; i < hi; i += EV_THREADS) {
        const uint32_t key = ev_key(w[i]);
        if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        int rem = s_rem, b = 255;
        for (; b > 0; --b) {
          if (int(hist[b]) >= rem) break;
          rem -= int(hist[b]);
        }
        s_prefix = prefix | (uint32_t(b) << shift);
        s_rem = rem;
      }
      mask |= 255u << shift;
      __syncthreads();
    }
  const uint32_t thr = none ? 0xffffffffu : s_prefix;
  int need_eq = none ? 0 : s_rem, out = 0;
  for (int i0 = 0; i0 < len; i0 += EV_THREADS) {
    const int i = i0 + tid;
    const bool cand = i >= lo && i < hi;
    const uint32_t key = cand ? ev_key(w[i]) : 0u;
    int eq_at, at;
    const int n_eq = ev_scan(cand && key == thr, &eq_at, warp_sums);
    const bool take = i < len && (!cand || (key > thr && !none) || (key == thr && eq_at < need_eq));
    const int n = ev_scan(take, &at, warp_sums);
    if (take) kept[out + at] = i;
    out += n;
    need_eq -= min(need_eq, n_eq);
  }
}

// Copies survivor i of a (sequence, kv head) to slot i of the destination: one
// warp a row, keys then values; a row's units are stored in another order in
// another slot.
__global__ void __launch_bounds__(256) k_kv4_evict_copy(const Kv4EvictArgs a) {
  const Kv4Geo& g = a.g;
  const int seq = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31;
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int len = kv4_len(a.b, seq), nl = min(len, a.keep);
  if (i >= nl) return;
  const int64_t pair = int64_t(seq) * g.kvh + h;
  const int src = a.kept[pair * a.kstride + i];
  const uint8_t* from = kv4_block(g, g.table, g.tstride, seq, h, src, a.b.status);
  uint8_t* to = kv4_block(g, a.dst, a.dstride, seq, h, i, a.b.status);
  if (!from || !to) return;
  const int ts = src & (g.seg - 1), td = i & (g.seg - 1), wpu = g.hd / 64, mix = kv4_swz(g.hd, ts) ^ kv4_swz(g.hd, td);
  for (int kv = 0; kv < 2; ++kv, from += g.blk / 2, to += g.blk / 2) {
    const uint32_t* s = reinterpret_cast<const uint32_t*>(from + ts * (g.hd / 2));
    uint32_t* d = reinterpret_cast<uint32_t*>(to + td * (g.hd / 2));
    if (lane < 8 * wpu) d[(((lane / wpu) ^ mix) * wpu) + lane % wpu] = s[lane];
    const uint32_t* sp = reinterpret_cast<const uint32_t*>(from + g.seg * (g.hd / 2)) + ts * g.ng;
    uint32_t* dp = reinterpret_cast<uint32_t*>(to + g.seg * (g.hd / 2)) + td * g.ng;
    if (lane < g.ng) dp[lane] = sp[lane];
  }
  if (a.new_weights && lane == 0) a.new_weights[pair * a.nwstride + i] = a.weights[pair * a.wstride + src];
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
  launch(k_kv4_evict_select, dim3(a.g.kvh, a.b.nseq), dim3(EV_THREADS), 0, st, false, a);
  const int most = std::min(a.keep, a.b.max_len);
  if (most > 0) launch(k_kv4_evict_copy, dim3((most + 7) / 8, a.g.kvh, a.b.nseq), dim3(256), 0, st, false, a);
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
