// Attention over the 4-bit KV cache for few query rows a sequence (single
// tokens above all), and the accumulation of attention weights.
//
// With codes c, group scales s and biases b of a slot t (kv4.h), e = c - 7.5
// and b' = b + 7.5 s (the group's middle, so that neither part carries a
// large common term):
//   q.k_t = sum_g s_tg (sum_{i in g} q_i e_ti) + b'_tg (sum_{i in g} q_i)
//   out_i = sum_t (p_t s_tg) e_ti + sum_t p_t b'_tg          (i in group g)
// Codes are exact in f16, so both inner sums are matrix products of exact
// 4-bit operands: mma.m16n8k16 (f16, f32 accumulators) with 16 slots x 16
// channels of codes against the 8 query columns of a kv head, per group, and
// 16 channels x 16 slots against the weights p s. For f32 inputs q and p s go
// in as two f16 terms each (22 bits); for 16-bit inputs q is exact (bf16) or
// itself (f16) and p s is rounded to 11 bits. Softmax statistics, group sums
// and outputs are f32. Columns are scaled by powers of two on their way into
// f16 (q by its largest element, p by the largest group scale seen), which
// changes no bit of the result but keeps both terms in range.
// The accumulators truncate, so a sum is off by its largest partial sums, and
// with codes of one sign those are twice the score's (its error then measured
// 7.6e-6 on scores of 1.5) and 150 times the output's (at 128k equal weights:
// outputs 1e-2 off, all to one side). f32 inputs: codes are centred (10
// instructions per 8 codes) and a unit's outputs added apart. 16-bit inputs: keys
// go in as plain codes (one LOP3 a pair, 5 instructions per 8), and so do the
// values of a unit's first 8 slots; its last 8 go in as 15 - c against -p s, at
// the same cost, which keeps every partial sum small. With h the f16 weights as
// they go in (signed), sum |h| e = (sum h c') - 7.5 sum h, whose last sum is one
// more product a group, with -7.5 in every place: the rounding of p s counts
// against e, not c (f16 outputs 6e-4 -> 3.0e-4 off, where their own rounding is
// 2.1e-4; centring the values' codes instead cost 64 long contexts 244 us, not 226).
//
// Bound: the cache's bytes (2 (D / 2 + 4 D / g) a slot and kv head), next to
// the instructions of unpacking and weighting (f32: some 1050 a unit of 16
// slots at 256 channels and 2.1 a cycle and SM, which is what f32 waits for),
// which is why codes go to the tensor cores unscaled and the scales are applied
// to the 16 x 8 results. 2 kv heads of 256 channels, 16 query heads: one
// sequence of 131072 slots in f32 50 us (1.5 TB/s), 64 of 61 to
// 8192 slots in f32 80 us (1.9 TB/s), 64 of 20000 to 32768 in bf16 226 us (4.3
// TB/s).
#include <algorithm>

#include "kcommon.cuh"
#include "kv4.h"
#include "launch.h"

namespace swl {

namespace {

constexpr int AT_WARPS = 12;                // three per scheduler at 168 registers (8 and 16 were no faster)
constexpr int AT_THREADS = AT_WARPS * 32;
constexpr int AT_UNIT = 16;                 // slots a warp takes at a time: the MMA's M (keys) and K (values)
constexpr int AT_TILE = 128;                // slots of a tile, the grain in which work is shared out
constexpr int AT_HEAD = 4;                  // what an item costs beside its tiles, in tiles
constexpr int AT_COLS = 8;                  // query columns (token, head) of an item: the MMA's N
constexpr int AT_GRID = 148;                // one CTA per SM
// The reference point of a column moves when its maximum has outgrown it by
// 2^AT_SLACK; p carries 2^K with K = AT_UP - the exponent of the largest value
// scale s, so that p s (s < 2^(exponent + 1)) stays below 2^15, and f16's
// smallest step, 2^-24, is 2^-34 of the reference's p s: with a slack of 2^8 (and
// 2^6) f32 outputs of 2000 slots 18 nats behind the first were 5e-5 off, with
// this one 7e-6. It costs nothing (64 sequences of 61 to 8192 slots 80 us).
constexpr float AT_SLACK = 4.f;
constexpr int AT_UP = 10;
constexpr int WT_WARPS = 8;                 // warps of the weight kernel: one tile
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// ------------------------------------------------------------ primitives --
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8 x 8 matrix of 16-bit elements spread over the warp.
__device__ __forceinline__ uint32_t movm(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// Nibbles 0 and 1 of both halves of a word as two f16 pairs. Plain: the bits
// themselves, subnormals 2^-24 c and 2^-20 c. Centred: c - 7.5; a code at bits
// 1..4 of 0x6000 (512, step 0.5) is 512 + c, at bits 5..8 512 + 16 c, and both
// results are exact (x is the word shifted left by one).
__device__ __forceinline__ void unpack_plain(uint32_t x, uint32_t& n0, uint32_t& n1) {
  n0 = x & 0x000f000fu;
  n1 = x & 0x00f000f0u;
}
// Of the complements, 15 - c.
__device__ __forceinline__ void unpack_rest(uint32_t x, uint32_t& n0, uint32_t& n1) {
  n0 = ~x & 0x000f000fu;
  n1 = ~x & 0x00f000f0u;
}
__device__ __forceinline__ void unpack_centred(uint32_t x, uint32_t& n0, uint32_t& n1) {
  const __half2 m0 = u2h(0xe00fe00fu);                    // -519.5
  const __half2 m1 = u2h(0xd0f0d0f0u), r = u2h(0x2c002c00u);  // -39.5, 1 / 16
  n0 = h2u(__hadd2(u2h((x & 0x001e001eu) | 0x60006000u), m0));
  n1 = h2u(__hfma2(u2h((x & 0x01e001e0u) | 0x60006000u), r, m1));
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
// ------------------------------------------------------------------ work --
// The work is the list of all (sequence, column block, kv head) items, each of
// ceil(len / 128) tiles (one at least); a CTA takes an equal, contiguous share
// of all tiles, so ragged batches and single long sequences spread alike. An
// item counts AT_HEAD tiles more, in front of its own, for its beginning and
// end (queries, first copies, combination of the warps): 64 sequences of 61
// to 8192 slots took 97 us with one, 81 with four.
// Every warp finds its place from the lengths in device memory: nothing of the
// split is known to the host.
struct Place {
  int seq, item;   // item within the sequence: column block * kvh + kv head
  int tile;        // first tile of this share within the item, AT_HEAD tiles of overhead in front counted
  int row0, n, len, tiles, items;  // tiles: with AT_HEAD
};

__device__ __forceinline__ void load_seq(const Kv4AttnArgs& a, int seq, Place& p) {
  p.seq = seq;
  p.n = kv4_new(a.b, seq, p.row0);
  p.len = kv4_len(a.b, seq);
  p.tiles = AT_HEAD + max(1, (p.len + AT_TILE - 1) / AT_TILE);
  p.items = (int)(((int64_t)p.n * a.rep + AT_COLS - 1) / AT_COLS) * a.g.kvh;
}

__device__ __forceinline__ int64_t warp_incl(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

__device__ __forceinline__ int64_t total_tiles(const Kv4AttnArgs& a) {
  const int lane = threadIdx.x & 31;
  int64_t sum = 0;
  for (int i = lane; i < a.b.nseq; i += 32) {
    Place p;
    load_seq(a, i, p);
    sum += int64_t(p.tiles) * p.items;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// Place of tile number `flat` (0 <= flat < total).
__device__ __forceinline__ Place find_place(const Kv4AttnArgs& a, int64_t flat) {
  const int lane = threadIdx.x & 31;
  int64_t base = 0;
  Place p;
  for (int i0 = 0; i0 < a.b.nseq; i0 += 32) {
    int64_t cnt = 0;
    if (i0 + lane < a.b.nseq) {
      load_seq(a, i0 + lane, p);
      cnt = int64_t(p.tiles) * p.items;
    }
    const int64_t incl = warp_incl(cnt, lane);
    const unsigned hit = __ballot_sync(0xffffffffu, base + incl > flat);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int64_t before = base + __shfl_sync(0xffffffffu, incl - cnt, src);
      load_seq(a, i0 + src, p);
      const int64_t rem = flat - before;
      p.item = rem >> 32 ? int(rem / p.tiles) : int(unsigned(rem) / unsigned(p.tiles));
      p.tile = int(rem - int64_t(p.item) * p.tiles);
      return p;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  p = Place{0, 0, 0, 0, 0, 0, 1, 0};
  return p;
}

__device__ __forceinline__ void next_item(const Kv4AttnArgs& a, Place& p) {
  p.tile = 0;
  if (++p.item < p.items) return;
  p.item = 0;
  int s = p.seq + 1;
  for (; s < a.b.nseq; ++s) {
    load_seq(a, s, p);
    if (p.items) return;
  }
}

// ------------------------------------------------------- query columns ----
// Column c of block cb of a sequence's new rows: token (8 cb + c) / rep, query
// head h * rep + (8 cb + c) % rep.
template <int HD, bool SPLIT>
struct QStage {
  static constexpr int KS = HD / 16;  // k steps
  static constexpr int W = SPLIT ? 4 : 2;
  uint32_t frag[KS * 32 * W];        // B fragments: {hi b0, hi b1[, lo b0, lo b1]} per k step and lane
  float sum[AT_COLS][HD / 64];       // sums of the scaled column over each 64 channels, in the codes' unit
  float mul[AT_COLS];                // score = mul * (scaled sum), in units of log2
  int lim[AT_COLS];                  // last slot the column sees (INT_MAX: unused column)
};

// Warp w stages column w. Word l of the row (8 channels) is lane l's.
template <int HD, bool SPLIT>
__device__ __forceinline__ void stage_q(const Kv4AttnArgs& a, const Place& p, int h, int cb, int col, int lane, QStage<HD, SPLIT>* qs) {
  const int ci = cb * AT_COLS + col, t = ci / a.rep, hq = h * a.rep + ci % a.rep;
  const bool on = t < p.n;
  const bool act = lane < HD / 8;
  float x[8];
  float am = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = on && act ? kv4_ld(a.q.p, a.dt, (p.row0 + t) * a.q.ts + hq * a.q.hs + lane * 8 + e) : 0.f;
    am = fmaxf(am, fabsf(x[e]));
  }
  am = warp_max(am);
  // largest element to [2^12, 2^13); a column of zeros or infinities as it is
  int ex = am > 0.f && am < INFINITY ? 12 - (int(__float_as_uint(am) >> 23) - 127) : 0;
  ex = max(-100, min(100, ex));
  const float up = __int_as_float((127 + ex) << 23);
  float s = 0.f;
  uint32_t hi[8], lo[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] *= up;
    s += x[e];
    const float y = !SPLIT && (e & 1) ? x[e] * 0.0625f : x[e];  // odd nibbles come unpacked as 16 c
    const __half hh = __float2half_rn(y);
    hi[e] = __half_as_ushort(hh);
    if (SPLIT) lo[e] = __half_as_ushort(__float2half_rn(y - __half2float(hh)));
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (act) {
    if ((lane & 7) == 0) qs->sum[col][lane >> 3] = SPLIT ? s : s * 0x1p-24f;
    const int wi = lane >> 3, u = lane & 7;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int ks = (wi * 2 + (u >> 2)) * 2 + st;
      uint32_t* f = qs->frag + (ks * 32 + col * 4 + (u & 3)) * QStage<HD, SPLIT>::W;
      const uint32_t h0 = hi[2 * st] | hi[2 * st + 4] << 16, h1 = hi[2 * st + 1] | hi[2 * st + 5] << 16;
      if (SPLIT)
        *reinterpret_cast<uint4*>(f) = make_uint4(h0, h1, lo[2 * st] | lo[2 * st + 4] << 16, lo[2 * st + 1] | lo[2 * st + 5] << 16);
      else
        *reinterpret_cast<uint2*>(f) = make_uint2(h0, h1);
    }
  }
  if (lane == 0) {
    qs->mul[col] = a.scale * LOG2E * __int_as_float((127 - ex) << 23) * (SPLIT ? 1.f : 0x1p24f);
    qs->lim[col] = on ? p.len - p.n + t : 0x7fffffff;
  }
}

// The scores of 16 slots (rows r = lane / 4 and r + 8 of the fragment) against
// the 8 columns, before the column factor: kw = the rows' words of units c and
// c + 4 (c = lane % 4), kp = their params.
template <int HD, int GROUP, bool SPLIT, typename QF>
__device__ __forceinline__ void scores(const uint32_t (&kw)[2][2][HD / 64], const uint32_t (&kp)[2][HD / GROUP],
                                       const float (&qsum)[2][HD / GROUP], QF qf, float (&sc)[4]) {
  // the groups' sums side by side: one chain of products each, so that a
  // product does not wait for the one before it
  constexpr int NG = HD / GROUP;
  float acc[NG][4];
#pragma unroll
  for (int g = 0; g < NG; ++g) acc[g][0] = acc[g][1] = acc[g][2] = acc[g][3] = 0.f;
#pragma unroll
  for (int w = 0; w < GROUP / 64; ++w)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        uint32_t a0[NG], a1[NG], a2[NG], a3[NG], b[NG][SPLIT ? 4 : 2];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const int wi = g * (GROUP / 64) + w;
          if (SPLIT) {
            unpack_centred(st ? kw[hf][0][wi] >> 7 : kw[hf][0][wi] << 1, a0[g], a2[g]);
            unpack_centred(st ? kw[hf][1][wi] >> 7 : kw[hf][1][wi] << 1, a1[g], a3[g]);
          } else {
            unpack_plain(st ? kw[hf][0][wi] >> 8 : kw[hf][0][wi], a0[g], a2[g]);
            unpack_plain(st ? kw[hf][1][wi] >> 8 : kw[hf][1][wi], a1[g], a3[g]);
          }
          qf((wi * 2 + hf) * 2 + st, b[g]);
          mma16816(acc[g], a0[g], a1[g], a2[g], a3[g], b[g][0], b[g][1]);
        }
        if constexpr (SPLIT)
#pragma unroll
          for (int g = 0; g < NG; ++g) mma16816(acc[g], a0[g], a1[g], a2[g], a3[g], b[g][2], b[g][3]);
      }
  sc[0] = sc[1] = sc[2] = sc[3] = 0.f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float2 s0 = kv4_param(kp[0][g]), s1 = kv4_param(kp[1][g]);
    if (SPLIT) {  // the middle of the group
      s0.y = fmaf(7.5f, s0.x, s0.y);
      s1.y = fmaf(7.5f, s1.x, s1.y);
    }
    sc[0] = fmaf(s0.x, acc[g][0], fmaf(s0.y, qsum[0][g], sc[0]));
    sc[1] = fmaf(s0.x, acc[g][1], fmaf(s0.y, qsum[1][g], sc[1]));
    sc[2] = fmaf(s1.x, acc[g][2], fmaf(s1.y, qsum[0][g], sc[2]));
    sc[3] = fmaf(s1.x, acc[g][3], fmaf(s1.y, qsum[1][g], sc[3]));
  }
}

template <int HD, int GROUP, bool SPLIT>
struct AttnShared {
  static constexpr int CODES = AT_UNIT * HD / 2, PARAMS = AT_UNIT * 4 * (HD / GROUP);  // bytes of a unit's keys (values)
  static constexpr int UNIT_BYTES = 2 * (CODES + PARAMS);
  static constexpr int STAGES = HD == 256 ? 4 : 8;                  // units in flight a warp (18 KB at 256 channels)
  static constexpr int SLICE = STAGES * UNIT_BYTES;                 // one warp's ring, its outputs at the end of an item
  static_assert(SLICE >= AT_COLS * HD * 4, "a warp's outputs fit its ring");
  alignas(128) uint8_t ring[AT_WARPS][SLICE];
  QStage<HD, SPLIT> q;
  float m[AT_WARPS][AT_COLS], l[AT_WARPS][AT_COLS], f[AT_WARPS];  // maxima, sums, factors 2^-K of the warps
};

// Floats of one partial result: max, sum, outputs.
__host__ __device__ constexpr int part_floats(int hd) { return 2 * AT_COLS + AT_COLS * hd; }

__device__ __forceinline__ float* attn_lse(const Kv4AttnArgs& a) { return a.lse ? a.lse : reinterpret_cast<float*>(a.work); }
// The item that begins in a share and goes on: shares first .. last hold its
// parts (first < 0: none).
struct AtJoin {
  int first, last, row0, n, cb, h;
  int64_t total;  // of the launch
};
__device__ __forceinline__ AtJoin* attn_joins(const Kv4AttnArgs& a) {
  return reinterpret_cast<AtJoin*>(a.work + (int64_t(a.b.total) * a.heads * 4 + 15) / 16 * 16);
}
__device__ __forceinline__ float* attn_parts(const Kv4AttnArgs& a) { return reinterpret_cast<float*>(attn_joins(a) + AT_GRID); }
// First tile of a share, and the share that a tile is in.
__device__ __forceinline__ int64_t share_begin(int64_t total, int x) { return total * x / AT_GRID; }
__device__ __forceinline__ int share_of(int64_t total, int64_t tile) { return int(((tile + 1) * AT_GRID + total - 1) / total) - 1; }

// One output of a row, gated.
__device__ __forceinline__ void write_out(const Kv4AttnArgs& a, int64_t row, int hq, int ch, float v) {
  if (a.gate.p) v *= kv4_sigmoid(kv4_ld(a.gate.p, a.dt, row * a.gate.ts + hq * a.gate.hs + ch));
  kv4_st(a.out.p, a.dt, row * a.out.ts + hq * a.out.hs + ch, v);
}

template <int HD, int GROUP, bool SPLIT>
__global__ void __launch_bounds__(AT_THREADS, 1) k_kv4_attn(const Kv4AttnArgs a) {
  using Sh = AttnShared<HD, GROUP, SPLIT>;
  constexpr int NG = HD / GROUP, NW = HD / 64, S = Sh::STAGES;
  extern __shared__ __align__(128) uint8_t at_raw[];
  Sh& sh = *reinterpret_cast<Sh*>(at_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch();
  const int64_t total = total_tiles(a);
  const int64_t r0 = share_begin(total, blockIdx.x), r1 = share_begin(total, blockIdx.x + 1);
  if (threadIdx.x == 0) attn_joins(a)[blockIdx.x].first = -1;
  if (r0 == r1) return;
  Place p = find_place(a, r0);
  const Kv4Geo& g = a.g;
  const int r = lane >> 2, c = lane & 3;
  uint8_t* ring = sh.ring[warp];
  // this lane's vectors within a unit's keys and values
  const int koff0 = r * (HD / 2) + (c ^ kv4_swz(HD, r)) * (HD / 16), koff1 = r * (HD / 2) + ((c + 4) ^ kv4_swz(HD, r)) * (HD / 16);
  const int voff0 = 2 * c * (HD / 2) + (r ^ kv4_swz(HD, 2 * c)) * (HD / 16);
  const int voff1 = (2 * c + 1) * (HD / 2) + (r ^ kv4_swz(HD, 2 * c + 1)) * (HD / 16);
  const int nblk = g.page / g.seg;

  for (int64_t f = r0; f < r1; next_item(a, p)) {
    const int h = p.item % g.kvh, cb = p.item / g.kvh;
    const int v1 = int(min(int64_t(p.tiles), p.tile + (r1 - f)));
    // real tiles tb .. t1 - 1; the item's first part of several goes to slot 1, a later one (the share's first) to slot 0
    const int tb = max(0, p.tile - AT_HEAD), t1 = v1 - AT_HEAD, slot = p.tile == 0 ? 1 : 0;
    if (threadIdx.x == 0 && p.tile == 0 && v1 < p.tiles) {
      const int first = share_of(total, f + AT_HEAD), last = share_of(total, f + p.tiles - 1);
      if (first < last) attn_joins(a)[blockIdx.x] = AtJoin{first, last, p.row0, p.n, cb, h, total};
    }
    f += v1 - p.tile;
    if (t1 <= 0) continue;  // only overhead of the next share's item
    // units u0, u0 + 16, ... < u1 are this warp's
    const int u0 = tb * (AT_TILE / AT_UNIT) + warp, u1 = min(t1 * (AT_TILE / AT_UNIT), (p.len + AT_UNIT - 1) / AT_UNIT);
    const int* tab = g.table + p.seq * g.tstride;
    auto page_of = [&](int u) { return u < u1 ? __ldg(tab + ((u * AT_UNIT) >> g.pshift)) : 0; };
    unsigned lost = 0u;  // bit s: the page of stage s is outside the pool
    // the unit's keys, their params, values and theirs by 16-byte copies into this warp's own stage
    auto issue = [&](int u, int pg, int s) {
      lost &= ~(1u << s);
      if (u < u1) {
        if (unsigned(pg) < unsigned(g.npages)) {
          const int slot = u * AT_UNIT, t = slot & (g.seg - 1);
          const uint8_t* blk = g.pages + pg * g.page_bytes + int64_t(h * nblk + (slot & (g.page - 1)) / g.seg) * g.blk;
          const uint8_t* kc = blk + t * (HD / 2) + lane * 16;
          uint8_t* d = ring + s * Sh::UNIT_BYTES;
          constexpr int NC = Sh::CODES / 512, NP = Sh::PARAMS / 16;
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            cp_async16(d + i * 512 + lane * 16, kc + i * 512);
            cp_async16(d + Sh::CODES + Sh::PARAMS + i * 512 + lane * 16, kc + g.blk / 2 + i * 512);
          }
          const int hv = lane >> 4, lp = lane & 15;
          if (lp < NP)
            cp_async16(d + Sh::CODES + hv * (Sh::CODES + Sh::PARAMS) + lp * 16,
                       blk + hv * (g.blk / 2) + g.seg * (HD / 2) + t * NG * 4 + lp * 16);
        } else {
          lost |= 1u << s;
          if (lane == 0 && a.b.status) atomicOr(a.b.status, KV4_BAD);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < S; ++s) issue(u0 + s * AT_WARPS, page_of(u0 + s * AT_WARPS), s);
    int pg = page_of(u0 + S * AT_WARPS);
    if (warp < AT_COLS) stage_q<HD, SPLIT>(a, p, h, cb, warp, lane, &sh.q);
    __syncthreads();
    float qsum[2][NG], mul[2];
    int lim[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      mul[q] = sh.q.mul[2 * c + q];
      lim[q] = sh.q.lim[2 * c + q];
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        qsum[q][i] = 0.f;
#pragma unroll
        for (int w = 0; w < GROUP / 64; ++w) qsum[q][i] += sh.q.sum[2 * c + q][i * (GROUP / 64) + w];
      }
    }
    const int free_to = __reduce_min_sync(0xffffffffu, min(lim[0], lim[1]));  // every column sees slots up to here
    float o[NW * 4][4];
    float hs[NG][2];       // 16-bit inputs: -7.5 sum of the f16 weights as they go in
    float pb[NG][2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int K = 0;             // p carries a factor 2^K (AT_UP)
    unsigned smax = 0u;    // that scale's bits
#pragma unroll
    for (int i = 0; i < NW * 4; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int i = 0; i < NG; ++i) pb[i][0] = pb[i][1] = hs[i][0] = hs[i][1] = 0.f;

    int s = 0;
    for (int u = u0; u < u1; u += AT_WARPS) {
      cp_async_wait_group<S - 1>();
      __syncwarp();
      const int s0 = u * AT_UNIT;
      const uint8_t* st = ring + s * Sh::UNIT_BYTES;
      const uint8_t* sv = st + Sh::CODES + Sh::PARAMS;
      const bool gone = (lost >> s) & 1;
      const bool edge = gone || s0 + 15 > free_to || s0 + 15 >= p.len;
      float x[4];
      {
        uint32_t kw[2][2][NW], kp[2][NG];
        kv4_ldv(st + koff0, kw[0][0]);
        kv4_ldv(st + koff0 + 8 * (HD / 2), kw[0][1]);
        kv4_ldv(st + koff1, kw[1][0]);
        kv4_ldv(st + koff1 + 8 * (HD / 2), kw[1][1]);
        kv4_ldv(st + Sh::CODES + r * NG * 4, kp[0]);
        kv4_ldv(st + Sh::CODES + (r + 8) * NG * 4, kp[1]);
        scores<HD, GROUP, SPLIT>(kw, kp, qsum, [&](int k, uint32_t (&b)[SPLIT ? 4 : 2]) {
          kv4_ldv(reinterpret_cast<const uint8_t*>(sh.q.frag + (k * 32 + lane) * QStage<HD, SPLIT>::W), b);
        }, x);
      }
      uint32_t vp[2][NG], vw[4][NW];
      kv4_ldv(sv + Sh::CODES + r * NG * 4, vp[0]);
      kv4_ldv(sv + Sh::CODES + (r + 8) * NG * 4, vp[1]);
      kv4_ldv(sv + voff0, vw[0]);
      kv4_ldv(sv + voff1, vw[1]);
      kv4_ldv(sv + voff0 + 8 * (HD / 2), vw[2]);
      kv4_ldv(sv + voff1 + 8 * (HD / 2), vw[3]);
      unsigned see = 15u;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] *= mul[i & 1];
      if (edge) {
        // what a column does not see: no weight, whatever the memory holds
        const bool live0 = !gone && s0 + r < p.len, live1 = !gone && s0 + r + 8 < p.len;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!((i < 2 ? live0 : live1) && s0 + r + (i < 2 ? 0 : 8) <= lim[i & 1])) {
            see &= ~(1u << i);
            x[i] = -INFINITY;
          }
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          if (!live0) vp[0][i] = 0u;
          if (!live1) vp[1][i] = 0u;
        }
      }
      // running maximum of each column, and of the value scales
      float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], d));
        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], d));
      }
      unsigned sb = __vmaxu2(vp[0][0], vp[1][0]);  // scales are the low halves, and positive
#pragma unroll
      for (int i = 1; i < NG; ++i) sb = __vmaxu2(sb, __vmaxu2(vp[0][i], vp[1][i]));
      sb = __reduce_max_sync(0xffffffffu, sb & 0xffffu);
      if (sb >= 0x7c00u) {  // groups that read as NaN have no say: a column that sees none of them keeps its bits
        sb = 0u;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if ((vp[k][i] & 0x7c00u) != 0x7c00u) sb = max(sb, vp[k][i] & 0xffffu);
        sb = __reduce_max_sync(0xffffffffu, sb);
      }
      if (__any_sync(0xffffffffu, mx[0] > m[0] + AT_SLACK || mx[1] > m[1] + AT_SLACK) || sb > smax) {
        int dk = 0;
        if (sb > smax) {
          smax = sb | 0x3ffu;  // the whole binade: K goes by the exponent (s < 2^(e + 1))
          const int e = int(sb >> 10) - 15;
          dk = AT_UP - e - K;
          K = AT_UP - e;
        }
        const float up = ex2(float(dk));
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float mn = mx[q] > m[q] + AT_SLACK ? mx[q] : m[q];
          const float al = m[q] == -INFINITY ? 0.f : ex2(m[q] - mn) * up;
          m[q] = mn;
          l[q] *= al;
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            pb[i][q] *= al;
            if constexpr (!SPLIT) hs[i][q] *= al;
          }
#pragma unroll
          for (int i = 0; i < NW * 4; ++i) {
            o[i][q] *= al;
            o[i][q + 2] *= al;
          }
        }
      }
      float pr[4];
      {
        const float mk0 = m[0] == -INFINITY ? 0.f : m[0] - float(K), mk1 = m[1] == -INFINITY ? 0.f : m[1] - float(K);
        pr[0] = ex2(x[0] - mk0);
        pr[1] = ex2(x[1] - mk1);
        pr[2] = ex2(x[2] - mk0);
        pr[3] = ex2(x[3] - mk1);
      }
      l[0] += pr[0] + pr[2];
      l[1] += pr[1] + pr[3];
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        float2 v0 = kv4_param(vp[0][gi]), v1 = kv4_param(vp[1][gi]);
        v0.y = fmaf(7.5f, v0.x, v0.y);  // the middle of the group
        v1.y = fmaf(7.5f, v1.x, v1.y);
        const float s1 = SPLIT ? v1.x : -v1.x;
        float ps[4] = {pr[0] * v0.x, pr[1] * v0.x, pr[2] * s1, pr[3] * s1};
        if (edge) {
          float pm[4] = {pr[0] * v0.y, pr[1] * v0.y, pr[2] * v1.y, pr[3] * v1.y};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!((see >> i) & 1)) ps[i] = pm[i] = 0.f;
          pb[gi][0] += pm[0] + pm[2];
          pb[gi][1] += pm[1] + pm[3];
        } else {
          pb[gi][0] = fmaf(pr[2], v1.y, fmaf(pr[0], v0.y, pb[gi][0]));
          pb[gi][1] = fmaf(pr[3], v1.y, fmaf(pr[1], v0.y, pb[gi][1]));
        }
        const __half2 h0 = __floats2half2_rn(ps[0], ps[1]), h1 = __floats2half2_rn(ps[2], ps[3]);
        const uint32_t bh0 = movm(h2u(h0)), bh1 = movm(h2u(h1));
        uint32_t bl0 = 0, bl1 = 0;
        if (SPLIT) {
          const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
          bl0 = movm(h2u(__floats2half2_rn(ps[0] - f0.x, ps[1] - f0.y)));
          bl1 = movm(h2u(__floats2half2_rn(ps[2] - f1.x, ps[3] - f1.y)));
        }
        if constexpr (!SPLIT) {
          float d[4] = {hs[gi][0], hs[gi][1], 0.f, 0.f};  // rows are alike
          mma16816(d, 0xc780c780u, 0xc780c780u, 0xc780c780u, 0xc780c780u, bh0, bh1);
          hs[gi][0] = d[0];
          hs[gi][1] = d[1];
        }
#pragma unroll
        for (int w = 0; w < GROUP / 64; ++w) {
          const int wi = gi * (GROUP / 64) + w;
          uint32_t av[4][4];
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            const uint32_t sel = pt ? 0x7632u : 0x5410u;
            const uint32_t ab = prmt(vw[0][wi], vw[1][wi], sel), cd = prmt(vw[2][wi], vw[3][wi], sel);
#pragma unroll
            for (int st2 = 0; st2 < 2; ++st2) {
              uint32_t(&f)[4] = av[pt * 2 + st2];
              if (SPLIT) {
                unpack_centred(st2 ? ab >> 7 : ab << 1, f[0], f[1]);
                unpack_centred(st2 ? cd >> 7 : cd << 1, f[2], f[3]);
              } else {
                unpack_plain(st2 ? ab >> 8 : ab, f[0], f[1]);
                unpack_rest(st2 ? cd >> 8 : cd, f[2], f[3]);
              }
              if (!SPLIT) mma16816(o[wi * 4 + pt * 2 + st2], f[0], f[1], f[2], f[3], bh0, bh1);
            }
          }
          if (SPLIT) {
            // the accumulators truncate: a unit's sums (the small products
            // first) are made apart and added with correct rounding
            float d[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              d[k][0] = d[k][1] = d[k][2] = d[k][3] = 0.f;
              mma16816(d[k], av[k][0], av[k][1], av[k][2], av[k][3], bl0, bl1);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) mma16816(d[k], av[k][0], av[k][1], av[k][2], av[k][3], bh0, bh1);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[wi * 4 + k][e] += d[k][e];
          }
        }
      }
      __syncwarp();
      issue(u + S * AT_WARPS, pg, s);
      pg = page_of(u + (S + 1) * AT_WARPS);
      s = s + 1 == S ? 0 : s + 1;
    }
    cp_async_wait_all();
    __syncwarp();

    // ---- the item's share is done: combine the warps. A warp leaves its
    // outputs in its own ring: [word][column parity][k][lane], the k-th of the
    // 8 channels of a 64-channel block that the lane holds for a column ----
#pragma unroll
    for (int d = 4; d < 32; d <<= 1)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        l[q] += __shfl_xor_sync(0xffffffffu, l[q], d);
#pragma unroll
        for (int i = 0; i < NG; ++i) pb[i][q] += __shfl_xor_sync(0xffffffffu, pb[i][q], d);
      }
#pragma unroll
    for (int i = 0; i < NG; ++i)
      if constexpr (!SPLIT) {  // these are whole in every lane
        pb[i][0] += hs[i][0];
        pb[i][1] += hs[i][1];
      }
    if (r == 0) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        // a NaN score leaves the maximum alone, but not the sum: infinity makes
        // the column NaN when it is joined
        sh.m[warp][2 * c + q] = l[q] != l[q] ? INFINITY : m[q];
        sh.l[warp][2 * c + q] = l[q];
      }
    }
    if (lane == 0) sh.f[warp] = ex2(float(-K));
    float* red = reinterpret_cast<float*>(ring);
    // codes as they stand carry 2^-24, and 16 where the nibble is odd
    constexpr float E0 = SPLIT ? 1.f : 0x1p24f, E1 = SPLIT ? 1.f : 0x1p20f;
    if (u0 < u1)
#pragma unroll
      for (int wi = 0; wi < NW; ++wi)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int k = 0; k < 8; ++k)
            red[((wi * 2 + q) * 8 + k) * 32 + lane] = fmaf(o[wi * 4 + k / 2][q + 2 * (k & 1)], k & 1 ? E1 : E0, pb[wi / (GROUP / 64)][q]);
    __syncthreads();
    // four outputs of a column at a time
    for (int i = warp; i < NW * 4; i += AT_WARPS) {
      const int e = i >> 2, q = (i >> 1) & 1, hf = i & 1;
      const int col = 2 * c + q;
      float v[4] = {0.f, 0.f, 0.f, 0.f}, M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < AT_WARPS; ++w) M = fmaxf(M, sh.m[w][col]);
#pragma unroll
      for (int w = 0; w < AT_WARPS; ++w) {
        const float mw = sh.m[w][col];
        if (mw == -INFINITY) continue;  // nothing seen by this warp
        const float fw = ex2(mw - M) * sh.f[w];
        L = fmaf(sh.l[w][col], fw, L);
        const float* rw = reinterpret_cast<const float*>(sh.ring[w]);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = fmaf(rw[((e * 2 + q) * 8 + hf * 4 + k) * 32 + lane], fw, v[k]);
      }
      const int ch = e * 64 + r * 8 + hf * 4;
      if (tb == 0 && v1 == p.tiles) {
        const int ci = cb * AT_COLS + col, tok = ci / a.rep, hq = h * a.rep + ci % a.rep;
        if (tok < p.n) {
          const float inv = M == -INFINITY ? 0.f : 1.f / L;
#pragma unroll
          for (int k = 0; k < 4; ++k) write_out(a, p.row0 + tok, hq, ch + k, v[k] * inv);
          if (ch == 0) attn_lse(a)[int64_t(p.row0 + tok) * a.heads + hq] = M == -INFINITY ? -INFINITY : (M + log2f(L)) * LN2;
        }
      } else {
        float* part = attn_parts(a) + (int64_t(blockIdx.x) * 2 + slot) * part_floats(HD);
        if (ch == 0) {
          part[col] = M;
          part[AT_COLS + col] = L;
        }
        *reinterpret_cast<float4*>(part + 2 * AT_COLS + col * HD + ch) = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    __syncthreads();  // the rings are free again
  }
}

// Joins the parts of the item that begins in share x and goes on: one block per
// (share, column), a thread four channels of every G-th part. Bound: latency,
// so that the first parts' outputs are under way before their factors are known.
// One long sequence (two items of 74 parts) takes 49 us with 512 threads a block
// and 50 with 256, but 128 items of two parts 84 and 79.
constexpr int AJ_THREADS = 256;
template <int HD>
__global__ void __launch_bounds__(AJ_THREADS) k_kv4_attn_join(const Kv4AttnArgs a) {
  constexpr int C4 = HD / 4, G = AJ_THREADS / C4, PRE = 4;
  static_assert(AT_GRID <= AJ_THREADS, "a thread a part");
  __shared__ float wt[AT_GRID];
  __shared__ float red[32];
  __shared__ float4 acc[AJ_THREADS];
  pdl_wait();
  const int x = blockIdx.x, col = blockIdx.y, tid = threadIdx.x, c4 = tid % C4, gi = tid / C4;
  const AtJoin d = attn_joins(a)[x];
  if (d.first < 0) return;
  const int ci = d.cb * AT_COLS + col, tok = ci / a.rep, hq = d.h * a.rep + ci % a.rep;
  if (tok >= d.n) return;
  const float* parts = attn_parts(a);
  auto part = [&](int i) { return parts + (int64_t(d.first + i) * 2 + (d.first + i == x ? 1 : 0)) * part_floats(HD); };
  const int np = d.last - d.first + 1;
  // with fewer tiles than shares some are empty, and have no part
  auto has = [&](int i) {
    return i < np && (d.total >= AT_GRID || share_begin(d.total, d.first + i) < share_begin(d.total, d.first + i + 1));
  };
  auto vec = [&](int i) { return __ldcg(reinterpret_cast<const float4*>(part(i) + 2 * AT_COLS + col * HD) + c4); };
  float4 pre[PRE];
#pragma unroll
  for (int k = 0; k < PRE; ++k) pre[k] = has(gi + k * G) ? vec(gi + k * G) : make_float4(0.f, 0.f, 0.f, 0.f);
  float mi = -INFINITY, li = 0.f;
  if (has(tid)) {
    mi = __ldcg(part(tid) + col);
    li = __ldcg(part(tid) + AT_COLS + col);
  }
  float M = warp_max(mi);
  if ((tid & 31) == 0) red[tid >> 5] = M;
  __syncthreads();
  M = red[0];
#pragma unroll
  for (int w = 1; w < AJ_THREADS / 32; ++w) M = fmaxf(M, red[w]);
  __syncthreads();
  const float fi = mi == -INFINITY ? 0.f : ex2(mi - M);
  if (tid < np) wt[tid] = fi;
  const float L = block_sum(mi == -INFINITY ? 0.f : li * fi, red);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float f, const float4& o) {
    if (f == 0.f) return;
    v.x = fmaf(f, o.x, v.x), v.y = fmaf(f, o.y, v.y), v.z = fmaf(f, o.z, v.z), v.w = fmaf(f, o.w, v.w);
  };
#pragma unroll
  for (int k = 0; k < PRE; ++k)
    if (gi + k * G < np) add(wt[gi + k * G], pre[k]);
#pragma unroll 4
  for (int i = gi + PRE * G; i < np; i += G) add(wt[i], has(i) ? vec(i) : make_float4(0.f, 0.f, 0.f, 0.f));
  acc[tid] = v;
  __syncthreads();
  if (gi) return;
#pragma unroll
  for (int k = 1; k < G; ++k) add(1.f, acc[k * C4 + c4]);
  const int64_t row = d.row0 + tok;
  const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) write_out(a, row, hq, c4 * 4 + k, M == -INFINITY ? 0.f : o[k] / L);
  if (tid == 0) attn_lse(a)[row * a.heads + hq] = M == -INFINITY ? -INFINITY : (M + log2f(L)) * LN2;
}

// ------------------------------------------------------- accumulated weight --
// weights[t] += sum over the columns that see slot t of exp(score - lse), the
// scores computed again from the keys alone: 144 bytes a slot and kv head at 256
// channels, 72 at 128, and no space of rows x slots. (Scores written out and
// read back would be 64 bytes for the 8 query heads of a single token.) A CTA
// owns 128 slots of a kv head and walks all the sequence's columns, so every sum
// has one order. Bound: latency (a single token, 16 sequences of 3000 to 8200
// slots in f32: 62 us with the attention, of which this is some 20, 28 alone).
template <int HD, int GROUP, bool SPLIT>
__global__ void __launch_bounds__(WT_WARPS * 32) k_kv4_weights(const Kv4AttnArgs a) {
  constexpr int NG = HD / GROUP, NW = HD / 64;
  __shared__ __align__(16) QStage<HD, SPLIT> sq[2];
  __shared__ float slse[2][AT_COLS];
  pdl_wait();
  const Kv4Geo& g = a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int h = blockIdx.y;
  Place p;
  load_seq(a, blockIdx.z, p);
  const int tile0 = blockIdx.x * AT_TILE;
  if (tile0 >= p.len || p.n == 0) return;
  const int s0 = tile0 + warp * 16;
  const uint8_t* blk = s0 < p.len ? kv4_block(g, g.table, g.tstride, p.seq, h, s0, a.b.status) : nullptr;
  uint32_t kw[2][2][NW], kp[2][NG];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = (s0 & (g.seg - 1)) + r + 8 * i;
#pragma unroll
    for (int w = 0; w < NW; ++w) kw[0][i][w] = kw[1][i][w] = 0u;
#pragma unroll
    for (int w = 0; w < NG; ++w) kp[i][w] = 0u;
    if (blk) {
      kv4_ldv(blk + t * (HD / 2) + (c ^ kv4_swz(HD, t)) * (HD / 16), kw[0][i]);
      kv4_ldv(blk + t * (HD / 2) + ((c + 4) ^ kv4_swz(HD, t)) * (HD / 16), kw[1][i]);
      kv4_ldv(blk + g.seg * (HD / 2) + t * NG * 4, kp[i]);
    }
  }
  const float* lse = attn_lse(a);
  const int ncb = (p.n * a.rep + AT_COLS - 1) / AT_COLS;
  // the first column block with a token that sees the tile's first slot
  const int first = int(max(int64_t(0), int64_t(tile0) - (p.len - p.n)) * a.rep / AT_COLS);
  float w0 = 0.f, w1 = 0.f;
  for (int cb = first; cb < ncb; ++cb) {
    QStage<HD, SPLIT>& q = sq[cb & 1];
    stage_q<HD, SPLIT>(a, p, h, cb, warp, lane, &q);
    if (lane == 0) {
      const int ci = cb * AT_COLS + warp, tok = ci / a.rep;
      slse[cb & 1][warp] = tok < p.n ? lse[int64_t(p.row0 + tok) * a.heads + h * a.rep + ci % a.rep] * LOG2E : INFINITY;
    }
    __syncthreads();
    float qsum[2][NG], x[4];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        qsum[k][i] = 0.f;
#pragma unroll
        for (int w = 0; w < GROUP / 64; ++w) qsum[k][i] += q.sum[2 * c + k][i * (GROUP / 64) + w];
      }
    scores<HD, GROUP, SPLIT>(kw, kp, qsum, [&](int k, uint32_t (&b)[SPLIT ? 4 : 2]) {
      kv4_ldv(reinterpret_cast<const uint8_t*>(q.frag + (k * 32 + lane) * QStage<HD, SPLIT>::W), b);
    }, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = i & 1, slot = s0 + r + (i < 2 ? 0 : 8);
      const bool see = slot <= q.lim[2 * c + k] && cb * AT_COLS + 2 * c + k < p.n * a.rep;
      const float e = see ? ex2(fmaf(x[i], q.mul[2 * c + k], -slse[cb & 1][2 * c + k])) : 0.f;
      if (i < 2) w0 += e; else w1 += e;
    }
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    w0 += __shfl_xor_sync(0xffffffffu, w0, d);
    w1 += __shfl_xor_sync(0xffffffffu, w1, d);
  }
  if (c == 0 && blk) {
    float* w = a.weights + (int64_t(p.seq) * g.kvh + h) * a.wstride;
    if (s0 + r < p.len) w[s0 + r] += w0;
    if (s0 + r + 8 < p.len) w[s0 + r + 8] += w1;
  }
}

// Query rows a kv head up to which these kernels are used. A tile of the prompt
// kernel costs the same for 1 to 128 rows, here every 8 rows take the item's
// tiles once more. 32 sequences of 2000 slots (2 kv heads of 256 channels,
// bf16): 32 rows 55 us here and 95 there, 64 rows 96 and 97, 96 rows 137 and 99
// (f32: 64 rows 138 and 139, 96 rows 198 and 143). One of 30000 slots: 64 rows
// 43 and 76, 96 rows 57 and 76.
constexpr int64_t AT_FEW = 64;
bool few_rows(const Kv4Batch& b, int rep) { return int64_t(b.max_new) * rep <= AT_FEW; }

template <int HD, int GROUP, bool SPLIT>
void run(const Kv4AttnArgs& a, cudaStream_t st) {
  if (few_rows(a.b, a.rep)) {
    launch(k_kv4_attn<HD, GROUP, SPLIT>, dim3(AT_GRID), dim3(AT_THREADS), sizeof(AttnShared<HD, GROUP, SPLIT>), st, true, a);
    if (a.b.max_len > AT_TILE)  // or every item is one tile, and written at once
      launch(k_kv4_attn_join<HD>, dim3(AT_GRID, AT_COLS), dim3(AJ_THREADS), 0, st, true, a);
  } else {
    launch_kv4_prompt(a, st);
    return;
  }
  if (a.weights && a.b.max_len > 0)
    launch(k_kv4_weights<HD, GROUP, SPLIT>, dim3((a.b.max_len + AT_TILE - 1) / AT_TILE, a.g.kvh, a.b.nseq), dim3(WT_WARPS * 32), 0, st,
           true, a);
}

template <int HD, int GROUP>
void run_dt(const Kv4AttnArgs& a, cudaStream_t st) {
  if (a.dt == DT_F32) run<HD, GROUP, true>(a, st);
  else run<HD, GROUP, false>(a, st);
}

}  // namespace

int64_t kv4_attention_work(const Kv4Geo& g, const Kv4Batch& b, int heads) {
  if (!few_rows(b, heads / g.kvh)) return kv4_prompt_work(g, b, heads);
  return (int64_t(b.total) * heads * 4 + 15) / 16 * 16 + AT_GRID * int64_t(sizeof(AtJoin)) + int64_t(AT_GRID) * 2 * part_floats(g.hd) * 4;
}

void launch_kv4_attention(const Kv4AttnArgs& a, cudaStream_t st) {
  if (a.g.hd == 64) run_dt<64, 64>(a, st);
  else if (a.g.hd == 128) a.g.group == 64 ? run_dt<128, 64>(a, st) : run_dt<128, 128>(a, st);
  else a.g.group == 64 ? run_dt<256, 64>(a, st) : run_dt<256, 128>(a, st);
}

}  // namespace swl
