// Attention over the 4-bit KV cache for many query rows a sequence (prompts,
// chunks of them, long turns) on the 5th-generation tensor cores.
//
// An item is 128 query rows (token-major, the heads of one kv head adjacent)
// of one sequence and kv head; the context is walked in tiles of BN slots:
//   S = Q K^T (tcgen05.mma, M 128, N BN, K head_dim; accumulator in TMEM),
//   online softmax by two threads a row, P to TMEM as f16,
//   O += P V (M 128, N head_dim, K BN; A from TMEM, V as an N-major operand).
// Keys and values are unpacked to f16 on their way into shared memory, scaled
// by a power of two so that the largest value of the sequence and head is
// just below 2^14 (k_kv4_range reads the params for it). Keys are two f16
// terms, for scores, lse and the weights are f32 whatever the inputs' type.
// 16-bit inputs: keys are taken about their group's middle and exact, the
// middles are a product of 16 columns; queries and values are one term (values
// rounded to 11 bits like the inputs themselves), so two products and the
// small one make S and one O; for f16 the weights are two terms and O takes two
// (with one, outputs were off by 1.6 times their own rounding, with two 1.2 times). f32
// inputs: all operands are two terms (22 bits) and three products each make S
// and O (hi lo, lo hi, hi hi).
// The tensor cores' f32 accumulators truncate: every product added takes up to
// 2^-24 off the size of what it is added to. S is built from its small terms up;
// for f32 inputs O is taken out of TMEM every PT_FLUSH tiles and added up with
// correct rounding (without that, outputs were off by 1.5e-5 after some 30 tiles).
//
// Warps: 0-7 softmax and output (two threads a row, half of the tile's slots
// each), 8-15 unpacking of keys, 16-23 of values, 24 MMA issue and TMEM, 25 and
// 26 bulk copies of the cache's bytes (a tile's keys, a tile's values). Q stands in TMEM (its low terms in shared memory), S and
// P share columns and are double-buffered, so Q K^T of the next tile runs
// during the softmax of this one; the running maximum moves only when it has
// grown by 2^8 (f32: 2^4), so O in TMEM is rarely touched. Bound: the chain of copy,
// unpack, product, softmax, product. A tile of 64 slots at 256 channels is some
// 1560 cycles of MMA for bf16 (3070 for f32), and takes some 3200 (6000), with every
// role busy for two thirds of it or more (2.7 instructions a cycle and SM, the
// tensor pipe 47 % of the time): leaving out the exponentials, the
// maxima, the keys' low terms or a third of the products changed it by 3 % at
// most, the values' unpacking by 5, a second warp for the issue of products by
// nothing. Shared memory holds two buffers of unpacked tiles at most (one for
// f32), TMEM no second item.
// 2048 tokens on a context of 10000 (2 kv heads of 256 channels, 16 query heads,
// bf16): 455 to 500 us, 0.60 to 0.66 PFLOP/s; 8192 tokens from the first (4 kv
// heads of 128, 16 query heads, f16, four products): 695 to 710 us, 0.39; 8 chunks
// of 33 to 200 tokens on 900 to 4100 (2 of 256, f32, six products): 226 us, 0.18.
//
// The work is shared out like that of kv4_attn.cu: equal contiguous shares of
// all tiles of all items over 148 CTAs, parts of an item that several CTAs
// work on joined by a second kernel.
#include <algorithm>

#include "kcommon.cuh"
#include "kv4.h"
#include "launch.h"
#include "tc.cuh"

namespace swl {

namespace {

constexpr int PT_ROWS = 128;
constexpr int PT_BN = 64;                               // slots of a tile
constexpr int PT_GRID = 148;
constexpr int PT_SOFT = 256, PT_UNPACK = 512;           // threads of the softmax and unpack roles
constexpr int PT_THREADS = PT_SOFT + PT_UNPACK + 128;   // and a warpgroup that issues MMAs and copies
constexpr int PT_MMA = (PT_SOFT + PT_UNPACK) / 32, PT_COPY = PT_MMA + 1;  // warps
// Registers a thread: 72 at launch, then 256 x 96 + 512 x 64 + 128 x 56 (= 896 x 72).
constexpr int PT_REGS_SOFT = 96, PT_REGS_UNPACK = 64, PT_REGS_ISSUE = 56;
// Cost of an item beside its tiles, in tiles (queries, filling the pipeline, output): 8192 tokens
// from the first, whose early items are short, took 1565 us with one, 700 with twelve; chunks on long contexts 263 and 227.
constexpr int PT_HEAD = 12;
constexpr int PT_FLUSH = 4;                             // tiles that O of f32 inputs stays in TMEM
// The running maximum moves when it has grown by 2^pt_slack; the weights carry
// 2^pt_up, so that they stay below 2^15, and sums of them and outputs with them.
// f16's smallest step, 2^-24, is then 2^-31 of the maximum or less (f32 inputs
// 2^-35): weights that many slots share behind a dominant one are still there
// (unscaled, those below 2^-25 were lost to the outputs: 2000 slots 18 nats
// behind the first, f32, 2 % of the output). A slack of 2^4 costs f32 inputs 4 % (8
// chunks 219 and 228 us) and 16-bit inputs, which gain nothing from it, 9 to 18 %.
constexpr int pt_slack(bool split) { return split ? 4 : 8; }
constexpr int pt_up(bool split) { return 15 - pt_slack(split); }
constexpr int RG_SPLIT = 16;                            // blocks a (sequence, head) of the range kernel
constexpr float P_LOG2E = 1.4426950408889634f, P_LN2 = 0.6931471805599453f;

template <int HD, int GROUP, bool SPLIT>
struct PtShape {
  static constexpr int T = SPLIT ? 2 : 1;                  // f16 terms of queries, weights and values
  static constexpr int KT = 2;                             // and of keys
  static constexpr int KST = HD == 256 && SPLIT ? 1 : 2;   // buffers of unpacked keys, and of values
  // Copied stages, of the keys and of the values: a stage is read into registers
  // before the wait for the unpacked buffer, so that the next copy is under way
  // meanwhile, and more of them gain nothing (8192 tokens at 128 channels: two of
  // keys 728 us, one 694). Each kind has its own, for a wait by parity tells two
  // neighbouring phases apart and no more.
  static constexpr int RK = 1, RV = 1, RST = RK + RV;
  static constexpr int QB = PT_ROWS * HD * 2;              // bytes of one term of Q
  static constexpr int KB = PT_BN * HD * 2;                // of one term of a tile's keys (values)
  static constexpr int RAW = PT_BN * (HD / 2 + 4 * (HD / GROUP));  // bytes of a tile's keys (values) as they are held
  // low terms of Q, keys (first the high terms of Q, on their way to TMEM), values, copied stages
  static constexpr int SCR = 8 * 32 * 33 * 4;              // the output's scratch, over the key buffers
  // 16-bit inputs: 16 more columns of Q and of every tile of keys, for the groups' middles (pt_middles)
  static constexpr int XQB = SPLIT ? 0 : PT_ROWS * 32, XKB = SPLIT ? 0 : PT_BN * 32;
  static constexpr int KS = KST * KT * KB > SCR ? KST * KT * KB : (SCR + 1023) / 1024 * 1024;
  static constexpr int Q_OFF = 0, K_OFF = SPLIT ? QB : 0, V_OFF = K_OFF + KS, R_OFF = V_OFF + KST * T * KB;
  static constexpr int XQ_OFF = R_OFF + RST * RAW, XK_OFF = XQ_OFF + XQB;
  static constexpr int M_OFF = XK_OFF + KST * XKB;         // the rows' factors and limits, exchange of the halves
  static constexpr int BAR_OFF = M_OFF + PT_ROWS * 16;
  static constexpr int NBAR = 4 * KST + 2 * RST + 7;       // k, v full / empty, raw full / empty, s full, p full, o done, drain
  static constexpr int TOTAL = BAR_OFF + NBAR * 8 + 16 + RST * 4 + 1024;  // 1024: base alignment
  static_assert(KS >= QB, "Q fits the key buffers");
  static_assert(TOTAL <= 232448, "shared memory");
  // TMEM columns: O, S (two tiles; P over it), Q
  static constexpr int O_COL = 0, S_COL = HD, Q_COL = HD + 2 * PT_BN;
  static_assert(Q_COL + HD / 2 <= 512, "TMEM columns");
};

// D f32, A and B f16; N, transposed (N-major) B
constexpr uint32_t pt_idesc(int n, bool bt) {
  return (1u << 4) | (uint32_t(bt) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(PT_ROWS >> 4) << 24);
}
// N-major operand, 128-byte swizzle: rows of 64 elements (one K index each),
// eight to an atom of 1024 bytes (SBO, along K); the next 64 elements of N lie
// lbo bytes on.
__device__ __forceinline__ uint64_t pt_desc_n(uint32_t saddr, uint32_t lbo) {
  return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(lbo >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
// K-major operand of 16 columns, no swizzle: blocks of eight rows x 16 bytes,
// the two of a row's 32 bytes 128 bytes apart (LBO), the next eight rows 256 (SBO).
__device__ __forceinline__ uint64_t pt_desc_x(uint32_t saddr) {
  return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(128 >> 4) << 16) | (uint64_t(256 >> 4) << 32) | (uint64_t(1) << 46);
}
// Byte of column c of row r in such an operand.
__device__ __forceinline__ constexpr int pt_x(int r, int c) { return (r >> 3) * 256 + (c >> 3) * 128 + (r & 7) * 16 + (c & 7) * 2; }
__device__ __forceinline__ void pt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc))
      : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc))
      : "memory");
}
__device__ __forceinline__ void pt_ld32(uint32_t t, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(t));
}
__device__ __forceinline__ void pt_st32(uint32_t t, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(t)
      : "memory");
}
__device__ __forceinline__ void pt_st16(uint32_t t, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]),
      "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(t)
      : "memory");
}
__device__ __forceinline__ void pt_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Pipeline wait: polls (hand-offs come within a tile's time), and gives up
// after 2^32 cycles, over two seconds. The bound goes by the SM's clock: a read
// of the global timer costs more than most waits.
__device__ __forceinline__ bool pt_wait(uint64_t* b, unsigned parity) {
  if (mbar_try(b, parity)) return true;
  const long long t0 = clock64();
  do {
    for (int i = 0; i < 256; ++i)
      if (mbar_try(b, parity)) return true;
  } while (clock64() - t0 < (1ll << 32));
  return false;
}
// One lane of a converged warp.
__device__ __forceinline__ bool pt_elect() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
  return ok != 0;
}
// Channel of a column within eight: the order in which codes come unpacked.
__device__ __forceinline__ constexpr int pt_channel(int col) { return (col >> 1) + 4 * (col & 1); }
// Adds O's columns of a row (HD / 2 of them at TMEM address t) to p, [by
// four][rows], which holds f times as much (nothing yet: on false).
template <int HD>
__device__ __forceinline__ void pt_add_out(uint32_t t, float4* p, bool on, float f) {
#pragma unroll 1
  for (int q = 0; q < HD / 64; ++q) {
    uint32_t o[32];
    pt_ld32(t + q * 32, o);
    tg_ld_wait();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float4* at = p + (q * 8 + e) * PT_ROWS;
      float4 v = on ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
      v.x = fmaf(v.x, f, __uint_as_float(o[4 * e]));
      v.y = fmaf(v.y, f, __uint_as_float(o[4 * e + 1]));
      v.z = fmaf(v.z, f, __uint_as_float(o[4 * e + 2]));
      v.w = fmaf(v.w, f, __uint_as_float(o[4 * e + 3]));
      *at = v;
    }
  }
}
// Barrier `id` of N threads; true when `v` is true for any of them.
template <int N = 64>
__device__ __forceinline__ bool pt_bar_any(int id, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %2, 0;\n\tbarrier.cta.red.or.pred.aligned q, %1, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(uint32_t(v)), "n"(N)
      : "memory");
  return r != 0;
}
template <int N>
__device__ __forceinline__ void pt_regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void pt_regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ float pt_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pt_h2(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 pt_u2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// ------------------------------------------------------------------ work --
struct PtPlace {
  int seq, qt, h;              // item: query tile qt, kv head h
  int tile, tiles;             // first tile of the share and tiles of the item, PT_HEAD counted in front
  int row0, n, len, nq;        // the sequence: first row, new tokens, slots, query tiles
};

// Tiles of query tile qt: up to the last slot its last row sees.
__device__ __forceinline__ int pt_tiles(int n, int len, int rep, int bn, int qt) {
  const int last = int(min(unsigned(n) - 1u, (unsigned(qt + 1) * PT_ROWS - 1u) / unsigned(rep)));
  const int seen = max(0, min(len, len - n + last + 1));
  return PT_HEAD + max(1, (seen + bn - 1) / bn);
}
__device__ __forceinline__ void pt_seq(const Kv4AttnArgs& a, int seq, PtPlace& p) {
  p.seq = seq;
  p.n = kv4_new(a.b, seq, p.row0);
  p.len = kv4_len(a.b, seq);
  p.nq = (p.n * a.rep + PT_ROWS - 1) / PT_ROWS;
}
__device__ __forceinline__ int64_t pt_total(const Kv4AttnArgs& a, int bn) {
  int64_t sum = 0;
  PtPlace p;
  for (int s = 0; s < a.b.nseq; ++s) {
    pt_seq(a, s, p);
    for (int q = threadIdx.x & 31; q < p.nq; q += 32) sum += pt_tiles(p.n, p.len, a.rep, bn, q);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum * a.g.kvh;
}
// Place of tile number `flat` (0 <= flat < total).
__device__ __forceinline__ PtPlace pt_find(const Kv4AttnArgs& a, int bn, int64_t flat) {
  const int lane = threadIdx.x & 31;
  int64_t base = 0;
  PtPlace p = {};
  for (int s = 0; s < a.b.nseq; ++s) {
    pt_seq(a, s, p);
    for (int q0 = 0; q0 < p.nq; q0 += 32) {
      const int64_t cnt = q0 + lane < p.nq ? int64_t(pt_tiles(p.n, p.len, a.rep, bn, q0 + lane)) * a.g.kvh : 0;
      int64_t incl = cnt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, base + incl > flat);
      if (hit) {
        const int src = __ffs(hit) - 1;
        const unsigned rem = unsigned(flat - base - __shfl_sync(0xffffffffu, incl - cnt, src));
        p.qt = q0 + src;
        p.tiles = pt_tiles(p.n, p.len, a.rep, bn, p.qt);
        p.h = int(rem / unsigned(p.tiles));
        p.tile = int(rem % unsigned(p.tiles));
        return p;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  return p;
}
__device__ __forceinline__ void pt_next(const Kv4AttnArgs& a, int bn, PtPlace& p) {
  p.tile = 0;
  if (++p.h < a.g.kvh) return;
  p.h = 0;
  if (++p.qt < p.nq) {
    p.tiles = pt_tiles(p.n, p.len, a.rep, bn, p.qt);
    return;
  }
  p.qt = 0;
  for (int s = p.seq + 1; s < a.b.nseq; ++s) {
    pt_seq(a, s, p);
    if (p.nq) {
      p.tiles = pt_tiles(p.n, p.len, a.rep, bn, 0);
      return;
    }
  }
}

// The item that begins in a share and goes on: shares first .. last hold its
// parts (first < 0: none).
struct PtJoin {
  int first, last, row0, n, qt, h;
  int64_t total;  // of the launch
};

// Workspace: lse rows, ranges, joins, parts.
__host__ __device__ inline int64_t pt_lse_bytes(int64_t total, int heads) { return (total * heads * 4 + 15) / 16 * 16; }
__host__ __device__ inline int64_t pt_range_bytes(int64_t nseq, int kvh) { return nseq * kvh * RG_SPLIT * 16; }
__host__ __device__ constexpr int pt_part_floats(int hd) { return PT_ROWS * (hd + 2); }
__device__ __forceinline__ float* pt_lse(const Kv4AttnArgs& a) { return a.lse ? a.lse : reinterpret_cast<float*>(a.work); }
__device__ __forceinline__ int4* pt_ranges(const Kv4AttnArgs& a) { return reinterpret_cast<int4*>(a.work + pt_lse_bytes(a.b.total, a.heads)); }
__device__ __forceinline__ PtJoin* pt_joins(const Kv4AttnArgs& a) {
  return reinterpret_cast<PtJoin*>(a.work + pt_lse_bytes(a.b.total, a.heads) + pt_range_bytes(a.b.nseq, a.g.kvh));
}
__device__ __forceinline__ float* pt_parts(const Kv4AttnArgs& a) { return reinterpret_cast<float*>(pt_joins(a) + PT_GRID); }

// Largest |value| of the keys and of the values of each (sequence, kv head),
// as f32 bits, and flags (bit 0: a value group is NaN, bit 1: a page outside the
// pool), over one of RG_SPLIT shares of the slots a block.
__global__ void __launch_bounds__(256) k_kv4_range(const Kv4AttnArgs a) {
  pdl_wait();
  pdl_launch();
  const int pair = blockIdx.x, seq = pair / a.g.kvh, h = pair % a.g.kvh;
  int row0;
  const int n = kv4_new(a.b, seq, row0), len = n ? kv4_len(a.b, seq) : 0;
  unsigned mk = 0u, mv = 0u, nan = 0u;
  for (int s = blockIdx.y * 256 + threadIdx.x; s < len; s += 256 * RG_SPLIT) {
    const uint8_t* blk = kv4_block(a.g, a.g.table, a.g.tstride, seq, h, s, a.b.status);
    if (!blk) {
      nan |= 2u;
      continue;
    }
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(blk + a.g.seg * (a.g.hd / 2)) + (s & (a.g.seg - 1)) * a.g.ng;
    const uint32_t* vp = kp + a.g.blk / 8;
    for (int i = 0; i < a.g.ng; ++i) {
      const float2 k = kv4_param(kp[i]), v = kv4_param(vp[i]);
      const float ka = fmaxf(fabsf(k.y), fabsf(fmaf(15.f, k.x, k.y))), va = fmaxf(fabsf(v.y), fabsf(fmaf(15.f, v.x, v.y)));
      if (ka < INFINITY) mk = max(mk, __float_as_uint(ka));
      if (va < INFINITY) mv = max(mv, __float_as_uint(va));
      nan |= unsigned(!(va < INFINITY));
    }
  }
  __shared__ unsigned red[3][8];
  mk = __reduce_max_sync(0xffffffffu, mk);
  mv = __reduce_max_sync(0xffffffffu, mv);
  nan = __reduce_or_sync(0xffffffffu, nan);
  if ((threadIdx.x & 31) == 0) red[0][threadIdx.x >> 5] = mk, red[1][threadIdx.x >> 5] = mv, red[2][threadIdx.x >> 5] = nan;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) mk = max(mk, red[0][w]), mv = max(mv, red[1][w]), nan |= red[2][w];
    pt_ranges(a)[int64_t(pair) * RG_SPLIT + blockIdx.y] = make_int4(int(mk), int(mv), int(nan), 0);
  }
}

// Exponent that takes a largest |value| (f32 bits) to [2^13, 2^14), as far as
// an f16 factor goes. Params times it are exact, but where they leave f16's
// normal range (below 2^-28 of the largest value).
__device__ __forceinline__ int pt_exp(unsigned bits) { return bits ? max(-14, min(14, 13 - (int(bits >> 23) - 127))) : 0; }
__device__ __forceinline__ float pt_pow2(int e) { return __int_as_float((127 + e) << 23); }

// Eight codes of a word as f16 pairs (0 4)(1 5)(2 6)(3 7), the codes exact.
__device__ __forceinline__ void pt_codes(uint32_t w, __half2 (&c)[4]) {
  const __half2 m0 = pt_u2(0xe400e400u);                          // 1024 + c less 1024
  const __half2 r = pt_u2(0x2c002c00u), m1 = pt_u2(0xd400d400u);  // (1024 + 16 c) / 16 less 64
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = i ? w >> 8 : w;
    c[2 * i] = __hadd2(pt_u2((x & 0x000f000fu) | 0x64006400u), m0);
    c[2 * i + 1] = __hfma2(pt_u2((x & 0x00f000f0u) | 0x64006400u), r, m1);
  }
}
// Their scaled values s c + b: rounded once, or two terms of them (22 bits).
template <bool SPLIT>
__device__ __forceinline__ void pt_unpack(uint32_t w, __half2 sb, uint4& hi, uint4& lo) {
  uint32_t* H = &hi.x;
  uint32_t* L = &lo.x;
  __half2 c[4];
  pt_codes(w, c);
  if (!SPLIT) {
    const __half2 s = __low2half2(sb), b = __high2half2(sb);
#pragma unroll
    for (int i = 0; i < 4; ++i) H[i] = pt_h2(__hfma2(c[i], s, b));
  } else {
    const float2 f2 = __half22float2(sb);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 v = __half22float2(c[i]);
      v.x = fmaf(f2.x, v.x, f2.y);
      v.y = fmaf(f2.x, v.y, f2.y);
      const __half2 h = __floats2half2_rn(v.x, v.y);
      const float2 f = __half22float2(h);
      H[i] = pt_h2(h);
      L[i] = pt_h2(__floats2half2_rn(v.x - f.x, v.y - f.y));
    }
  }
}
// Keys for 16-bit inputs, in f16 arithmetic alone: with e = c - 7.5, a key is
// s e + (b + 7.5 s). The first part is fl(s e) and its residual, which an FMA
// gives exactly (15 bits in all), the group's middle a product of its own
// (pt_middles): scores are f32 results whatever the inputs' type. (As f32
// inputs have them, two rounded terms of the whole value, they cost 17 % more:
// a turn of 2048 tokens on 10000 in bf16 533 us instead of 455.)
__device__ __forceinline__ void pt_unpack_keys(uint32_t w, __half2 sb, uint4& hi, uint4& lo) {
  uint32_t* H = &hi.x;
  uint32_t* L = &lo.x;
  const __half2 s = __low2half2(sb);
  const __half2 m0 = pt_u2(0xe00fe00fu);                          // 512 + c less 519.5
  const __half2 r = pt_u2(0x2c002c00u), m1 = pt_u2(0xd0f0d0f0u);  // (512 + 16 c) / 16 less 39.5
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = i < 2 ? w << 1 : w >> 7;
    const __half2 e = i & 1 ? __hfma2(pt_u2((x & 0x01e001e0u) | 0x60006000u), r, m1) : __hadd2(pt_u2((x & 0x001e001eu) | 0x60006000u), m0);
    const __half2 h = __hmul2(e, s);
    H[i] = pt_h2(h);
    L[i] = pt_h2(__hfma2(e, s, __hneg2(h)));
  }
}
// The groups' part of a score, sum_g (sum_{i in g} q_i) (b + 7.5 s)_g, as one
// more product of 16 columns: both factors two f16 terms (22 bits), columns g
// hi hi, 4 + g hi lo and 8 + g lo hi of group g, the others zero.
template <bool KEYS>
__device__ __forceinline__ void pt_middles(uint8_t* x, int row, int g, float v) {
  const __half hi = __float2half_rn(v), lo = __float2half_rn(v - __half2float(hi));
  *reinterpret_cast<__half*>(x + pt_x(row, g)) = hi;
  *reinterpret_cast<__half*>(x + pt_x(row, 4 + g)) = KEYS ? lo : hi;
  *reinterpret_cast<__half*>(x + pt_x(row, 8 + g)) = KEYS ? hi : lo;
}

template <int HD, int GROUP, bool SPLIT>
__global__ void __launch_bounds__(PT_THREADS, 1) k_kv4_prompt(const Kv4AttnArgs a) {
  using Sh = PtShape<HD, GROUP, SPLIT>;
  constexpr int BN = PT_BN, T = Sh::T, KT = Sh::KT, KST = Sh::KST, RST = Sh::RST, NG = HD / GROUP, NW = HD / 64;
  extern __shared__ __align__(1024) uint8_t pt_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pt_raw) + 1023) & ~uintptr_t(1023));
  float* row_mul = reinterpret_cast<float*>(sm + Sh::M_OFF);
  int* row_lim = reinterpret_cast<int*>(row_mul + PT_ROWS);
  float* xch = reinterpret_cast<float*>(row_lim + PT_ROWS);  // [2][rows]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + Sh::BAR_OFF);
  uint64_t *k_empty = k_full + KST, *v_full = k_empty + KST, *v_empty = v_full + KST, *r_full = v_empty + KST, *r_empty = r_full + RST,
           *s_full = r_empty + RST, *p_full = s_full + 2, *o_done = p_full + 2, *drain = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* r_have = reinterpret_cast<int*>(tmem_slot + 4);  // per copied stage: 16-slot pieces that are there
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Kv4Geo& g = a.g;
  if (tid == 0) {
    for (int s = 0; s < KST; ++s) {
      mbar_init(&k_full[s], PT_UNPACK / 2);
      mbar_init(&v_full[s], PT_UNPACK / 2);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < RST; ++s) {
      mbar_init(&r_full[s], 1);
      mbar_init(&r_empty[s], PT_UNPACK / 2);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], PT_SOFT);
      mbar_init(&o_done[s], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    mbar_init_fence();
  }
  if constexpr (!SPLIT) {  // the columns that stay zero
    for (int i = tid; i < (Sh::XQB + KST * Sh::XKB) / 16; i += PT_THREADS)
      reinterpret_cast<uint4*>(sm + Sh::XQ_OFF)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async();
  }
  if (warp == PT_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tg_fence_before();
  __syncthreads();
  tg_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch();
  const int64_t total = pt_total(a, BN);
  const int64_t r0 = total * blockIdx.x / PT_GRID, r1 = total * (blockIdx.x + 1) / PT_GRID;
  pdl_wait();  // the ranges
  auto fail = [&]() {
    if (a.b.status) atomicOr(a.b.status, 1);
    *abort_flag = 1;
  };
  // A wait of a whole warp.
  auto wait = [&](uint64_t* b, unsigned ph) {
    if (__all_sync(0xffffffffu, pt_wait(b, ph) && !*abort_flag)) return true;
    fail();
    return false;
  };
  // One role's walk over the items of the share. j counts the tiles of this
  // CTA, the pipelines' index. The softmax, unpack and MMA roles meet at
  // barrier 1 three times an item: queries staged, queries in TMEM, all over.
  int j = 0;
  constexpr int PT_MEET = PT_SOFT + PT_UNPACK + 32;
  auto bar = [] { asm volatile("bar.sync 1, %0;" ::"n"(PT_MEET) : "memory"); };
  auto for_items = [&](auto body) {
    PtPlace p = {};
    if (r0 < r1) p = pt_find(a, BN, r0);
    for (int64_t f = r0; f < r1; pt_next(a, BN, p)) {
      const int v1 = int(min(int64_t(p.tiles), p.tile + (r1 - f)));
      const int tb = max(0, p.tile - PT_HEAD), nt = v1 - PT_HEAD - tb, slot = p.tile == 0 ? 1 : 0;
      f += v1 - p.tile;
      if (v1 <= PT_HEAD || nt <= 0) continue;
      body(p, tb, nt, v1, slot);
      j += nt;
      __syncwarp();
      // every role takes the same decision to leave, or one would wait for another
      bool over = *abort_flag != 0;
      if (warp <= PT_MMA) {
        over = pt_bar_any<PT_MEET>(1, over);
        tg_fence_after();
      }
      if (over) break;
    }
  };
  // Ranges of an item: exponents of the keys' and values' scales, flags.
  auto ranges = [&](const PtPlace& p, int& kx, int& vx) {
    unsigned mk = 0u, mv = 0u, flags = 0u;
    if (lane < RG_SPLIT) {
      const int4 q = __ldcg(pt_ranges(a) + (int64_t(p.seq) * g.kvh + p.h) * RG_SPLIT + lane);
      mk = unsigned(q.x), mv = unsigned(q.y), flags = unsigned(q.z);
    }
    kx = pt_exp(__reduce_max_sync(0xffffffffu, mk));
    vx = pt_exp(__reduce_max_sync(0xffffffffu, mv));
    return __reduce_or_sync(0xffffffffu, flags);
  };

  if (warp < 8) {
    // ---------------------------------------------------------- softmax ----
    pt_regs_inc<PT_REGS_SOFT>();
    const int hf = warp >> 2, row = tid & (PT_ROWS - 1), pair = 2 + (warp & 3);
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
    constexpr int HB = BN / 2;
    constexpr float SLACK = pt_slack(SPLIT), UP = pt_up(SPLIT);
    const bool two_p = a.dt == DT_F16;
    for_items([&](const PtPlace& p, int tb, int nt, int v1, int slot_of_part) {
      int kx, vx;
      const unsigned flags = ranges(p, kx, vx);
      const bool lost = (flags & 2u) != 0u, vnan = (flags & 1u) != 0u;
      bar();
      // the row's queries (this half's channels) from the key buffers to TMEM
#pragma unroll
      for (int c4 = 0; c4 < HD / 64; ++c4) {
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int ck = hf * (HD / 16) + c4 * 4 + k;  // 16-byte chunk of the row
          kv4_ldv(sm + Sh::K_OFF + (ck >> 3) * (PT_ROWS * 128) + row * 128 + (((ck & 7) ^ (row & 7)) << 4),
                  *reinterpret_cast<uint32_t(*)[4]>(w + 4 * k));
        }
        pt_st16(lanes + Sh::Q_COL + hf * (HD / 4) + c4 * 16, w);
      }
      pt_st_wait();
      tg_fence_before();
      const float mul = row_mul[row];
      const int lim = row_lim[row];
      const int lim_lo = __reduce_min_sync(0xffffffffu, lim);
      bar();
      float m = -INFINITY, l = 0.f;
      // f32 inputs: what O was when it was last taken out of TMEM, relative to
      // the maximum mo; where the parts go, [channels by four][rows]
      float4* const part4 = reinterpret_cast<float4*>(pt_parts(a) + (int64_t(blockIdx.x) * 2 + slot_of_part) * pt_part_floats(HD) + 2 * PT_ROWS) +
                            hf * (HD / 8) * PT_ROWS + row;
      float mo = 0.f;
      bool pending = false;  // a wait that gave up
      for (int i = 0; i < nt; ++i) {
        const int jj = j + i, b = jj & 1;
        // the halves of a row leave together, or one would wait for the other
        const bool dead = !wait(&s_full[b], (jj >> 1) & 1) || pending;
        tg_fence_after();
        uint32_t s[HB];
        pt_ld32(lanes + Sh::S_COL + b * BN + hf * HB, s);
        tg_ld_wait();
        const int s0 = (tb + i) * BN + hf * HB;
        if (s0 + HB - 1 > lim_lo) {
#pragma unroll
          for (int e = 0; e < HB; ++e)
            if (s0 + e > lim) s[e] = 0xff800000u;
        }
        if (lost) {  // slots of pages outside the pool
#pragma unroll
          for (int e = 0; e < HB; ++e)
            if ((e & 15) == 0 && s0 + e < p.len && !kv4_block(g, g.table, g.tstride, p.seq, p.h, s0 + e, nullptr)) {
#pragma unroll
              for (int k = 0; k < 16; ++k) s[e + k] = 0xff800000u;
            }
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < HB; ++e) m4[e & 3] = fmaxf(m4[e & 3], __uint_as_float(s[e]));
        float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * mul;
        // both halves have read S when the pair has met: P may take its place
        tg_fence_before();
        const bool any = pt_bar_any(pair, mx > m + SLACK || dead), flush = SPLIT && i > 0 && i % PT_FLUSH == 0;
        if (flush) {
          pending = !wait(&o_done[b ^ 1], ((jj - 1) >> 1) & 1);
          tg_fence_after();
          pt_add_out<HD>(lanes + Sh::O_COL + hf * (HD / 2), part4, i > PT_FLUSH, mo == -INFINITY ? 0.f : pt_ex2(mo - m));
          mo = m;
        }
        if (any) {
          xch[hf * PT_ROWS + row] = mx;
          if (pt_bar_any(pair, dead)) break;
          mx = fmaxf(mx, xch[(hf ^ 1) * PT_ROWS + row]);
          const bool grow = mx > m + SLACK;
          const float mn = grow ? mx : m;
          const float al = m == -INFINITY ? (grow ? 0.f : 1.f) : pt_ex2(m - mn);
          m = mn;
          l *= al;
          bool late = false;
          if (i > 0 && !flush) {
            // every earlier product has landed before O is scaled
            late = !wait(&o_done[b ^ 1], ((jj - 1) >> 1) & 1);
            tg_fence_after();
#pragma unroll 1
            for (int q = 0; q < HD / 64; ++q) {
              uint32_t o[32];
              pt_ld32(lanes + Sh::O_COL + hf * (HD / 2) + q * 32, o);
              tg_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * al);
              pt_st32(lanes + Sh::O_COL + hf * (HD / 2) + q * 32, o);
            }
            pt_st_wait();
          }
          if (pt_bar_any(pair, late)) break;  // and xch is free again
        }
        tg_fence_after();
        const float mm = m == -INFINITY ? 0.f : m - UP;
        float l4[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t hi[HB / 2], lo[HB / 2];
        const auto weigh = [&](bool two) {
#pragma unroll
          for (int e = 0; e < HB / 2; ++e) {
            const float p0 = pt_ex2(fmaf(__uint_as_float(s[2 * e]), mul, -mm)), p1 = pt_ex2(fmaf(__uint_as_float(s[2 * e + 1]), mul, -mm));
            l4[2 * (e & 1)] += p0;
            l4[2 * (e & 1) + 1] += p1;
            const __half2 hh = __floats2half2_rn(p0, p1);
            hi[e] = pt_h2(hh);
            if (two) {
              const float2 ff = __half22float2(hh);
              lo[e] = pt_h2(__floats2half2_rn(p0 - ff.x, p1 - ff.y));
            }
          }
          pt_st16(lanes + Sh::S_COL + b * BN + hf * 16, hi);
          if (two) pt_st16(lanes + Sh::S_COL + b * BN + 32 + hf * 16, lo);
        };
        if (SPLIT || two_p) weigh(true);
        else weigh(false);
        l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
        pt_st_wait();
        tg_fence_before();
        mbar_arrive(&p_full[b]);
      }
      // ---- output: the last product has landed ----
      const bool whole = tb == 0 && v1 == p.tiles;
      const int last = j + nt - 1;
      wait(&o_done[last & 1], (last >> 1) & 1);
      tg_fence_after();
      xch[hf * PT_ROWS + row] = l;
      // value groups that are NaN went in as zeros: a row that sees one has NaN there
      unsigned bad = 0u;
      if (vnan)
        for (int s = tb * BN; s < min(min((tb + nt) * BN, p.len), lim + 1); ++s) {
          const uint8_t* blk = kv4_block(g, g.table, g.tstride, p.seq, p.h, s, nullptr);
          if (!blk) continue;
          const uint32_t* vp = reinterpret_cast<const uint32_t*>(blk + g.blk / 2 + g.seg * (HD / 2)) + (s & (g.seg - 1)) * NG;
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            const float2 v = kv4_param(vp[i]);
            if (!(fabsf(v.x) < INFINITY) || !(fabsf(v.y) < INFINITY)) bad |= 1u << i;
          }
        }
      __syncwarp();
      pt_bar_any(pair, false);
      l += xch[(hf ^ 1) * PT_ROWS + row];
      const bool none = l == 0.f;
      const float fac = none ? 0.f : whole ? pt_pow2(-vx) / l : pt_pow2(-vx);
      const bool more = SPLIT && nt > PT_FLUSH;  // O was taken out before
      const float fo = !more || mo == -INFINITY ? 0.f : pt_ex2(mo - m);
      const unsigned ci0 = unsigned(p.qt * PT_ROWS + (warp & 3) * 32);
      if (hf == 0) {
        const unsigned ci = ci0 + lane;
        const int tok = int(ci / unsigned(a.rep)), hq = p.h * a.rep + int(ci % unsigned(a.rep));
        if (!whole) {
          float* part = pt_parts(a) + (int64_t(blockIdx.x) * 2 + slot_of_part) * pt_part_floats(HD);
          part[row] = l != l ? INFINITY : m;  // a NaN sum stays NaN when parts are joined
          part[PT_ROWS + row] = l;
        } else if (tok < p.n) {
          pt_lse(a)[int64_t(p.row0 + tok) * a.heads + hq] = none ? -INFINITY : (m + log2f(l * pt_pow2(-int(UP)))) * P_LN2;
        }
      }
      // through shared memory (the key buffers: nothing reads them any more),
      // 32 rows x 32 channels a warp, so that a row's channels are written together
      float* scr = reinterpret_cast<float*>(sm + Sh::K_OFF) + warp * (32 * 33);
      const bool vo = kv4_vec(a.out, a.dt), vg = kv4_vec(a.gate, a.dt);
#pragma unroll 1
      for (int q = 0; q < HD / 64; ++q) {
        const int c0 = hf * (HD / 2) + q * 32;
        uint32_t o[32];
        pt_ld32(lanes + Sh::O_COL + c0, o);
        tg_ld_wait();
        const bool nan = (bad >> (c0 / GROUP)) & 1;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float4 p4 = make_float4(0.f, 0.f, 0.f, 0.f);
          float4* at = part4 + (q * 8 + e / 4) * PT_ROWS;
          if (more) p4 = *at;
          float v[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[k] = nan ? NAN : none ? 0.f : (more ? fmaf(v[k], fo, __uint_as_float(o[e + k])) : __uint_as_float(o[e + k])) * fac;
            o[e + k] = __float_as_uint(v[k]);
          }
          if (!whole) *at = make_float4(v[0], v[1], v[2], v[3]);
        }
        if (!whole) continue;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 32; ++e) scr[lane * 33 + (e & ~7) + pt_channel(e & 7)] = __uint_as_float(o[e]);
        __syncwarp();
        const int ch = (lane & 3) * 8;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int rr = k * 8 + (lane >> 2);
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = scr[rr * 33 + ch + e];
          const unsigned ci = ci0 + rr;
          const int tok = int(ci / unsigned(a.rep)), hq = p.h * a.rep + int(ci % unsigned(a.rep));
          if (tok >= p.n) continue;
          const int64_t at = int64_t(p.row0 + tok);
          if (a.gate.p) {
            float gt[8];
            kv4_ld8(a.gate.p, a.dt, at * a.gate.ts + hq * a.gate.hs + c0 + ch, vg, gt);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= kv4_sigmoid(gt[e]);
          }
          kv4_st8(a.out.p, a.dt, at * a.out.ts + hq * a.out.hs + c0 + ch, vo, v);
        }
      }
      tg_fence_before();
    });
    if (warp == 0) {  // what the join kernel has to do for this share
      PtJoin d = {-1, -1, 0, 0, 0, 0, 0};
      if (r0 < r1) {
        const PtPlace p = pt_find(a, BN, r1 - 1);
        const int64_t begin = r1 - 1 - p.tile, end = begin + p.tiles;
        if (begin >= r0 && end > r1) {
          const int nc = PT_GRID;
          int first = blockIdx.x, last = blockIdx.x;
          while (total * (first + 1) / nc <= begin + PT_HEAD) ++first;
          while (last + 1 < nc && total * (last + 1) / nc < end) ++last;
          if (first < last) d = PtJoin{first, last, p.row0, p.n, p.qt, p.h, total};
        }
      }
      if (lane == 0) pt_joins(a)[blockIdx.x] = d;
    }
  } else if (warp < PT_MMA) {
    // -------------------------------------------------------- unpacking ----
    pt_regs_dec<PT_REGS_UNPACK>();
    const int ut = tid - PT_SOFT, kv = ut >> 8, r = ut & 7, t = (ut >> 3) & 31;
    uint64_t *full = kv ? v_full : k_full, *empty = kv ? v_empty : k_empty;
    uint8_t* dst = sm + (kv ? Sh::V_OFF : Sh::K_OFF) + t * 128 + ((r ^ (t & 7)) << 4);
    for_items([&](const PtPlace& p, int tb, int nt, int v1, int) {
      int kx, vx;
      const unsigned flags = ranges(p, kx, vx);
      // queries: a warp a row, eight channels a lane, two rows at a time; a
      // negative scale goes into them, so that the rows' factors are positive
      const bool vq = kv4_vec(a.q, a.dt), act = lane < HD / 8;
      const float sgn = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
      for (int rb = warp - PT_SOFT / 32; rb < PT_ROWS; rb += 2 * PT_UNPACK / 32) {
        float x[2][8];
        int tok[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const unsigned ci = unsigned(p.qt * PT_ROWS + rb + PT_UNPACK / 32 * k);
          tok[k] = int(ci / unsigned(a.rep));
          const int hq = p.h * a.rep + int(ci - unsigned(tok[k]) * unsigned(a.rep));
#pragma unroll
          for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
          if (tok[k] < p.n && act) kv4_ld8(a.q.p, a.dt, int64_t(p.row0 + tok[k]) * a.q.ts + hq * a.q.hs + lane * 8, vq, x[k]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int qr = rb + PT_UNPACK / 32 * k;
          float am = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) am = fmaxf(am, fabsf(x[k][e]));
          am = warp_max(am);
          // the largest to [2^12, 2^13), or [2^5, 2^6), so that the sum of a group stays below 2^13
          int ex = am > 0.f && am < INFINITY ? (SPLIT ? 12 : 5) - (int(__float_as_uint(am) >> 23) - 127) : 0;
          ex = max(-100, min(100, ex));
          const float up = pt_pow2(ex) * sgn;
          float sum = 0.f;
          if (act) {
            uint4 hi, lo;
            uint32_t *H = &hi.x, *L = &lo.x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // the order the codes come unpacked in
              const float v0 = x[k][i] * up, v4 = x[k][i + 4] * up;
              const __half2 hh = __floats2half2_rn(v0, v4);
              H[i] = pt_h2(hh);
              if (!SPLIT) {
                const float2 ff = __half22float2(hh);
                sum += ff.x + ff.y;
              }
              if (SPLIT) {
                const float2 ff = __half22float2(hh);
                L[i] = pt_h2(__floats2half2_rn(v0 - ff.x, v4 - ff.y));
              }
            }
            const int off = (lane >> 3) * (PT_ROWS * 128) + qr * 128 + (((lane & 7) ^ (qr & 7)) << 4);
            *reinterpret_cast<uint4*>(sm + Sh::K_OFF + off) = hi;
            if (SPLIT) *reinterpret_cast<uint4*>(sm + Sh::Q_OFF + off) = lo;
          }
          if constexpr (!SPLIT) {
#pragma unroll
            for (int o = 1; o < GROUP / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (act && lane % (GROUP / 8) == 0) pt_middles<false>(sm + Sh::XQ_OFF, qr, lane / (GROUP / 8), sum);
          }
          if (lane == 0) {
            row_mul[qr] = sgn == 0.f ? 1.f : fabsf(a.scale) * P_LOG2E * pt_pow2(-ex) * pt_pow2(-kx);
            row_lim[qr] = tok[k] < p.n ? p.len - p.n + tok[k] : p.len - 1;
          }
        }
      }
      fence_proxy_async();
      bar();
      bar();
      // a thread: unit r of slots t and t + 32 of the tile, every 64-channel block
      const bool vnan = kv && (flags & 1u) != 0u;
      const __half2 sc = __float2half2_rn(pt_pow2(kv ? vx : kx));
      const int half = g.blk / 2, lseg = g.seg == 16 ? 4 : g.seg == 32 ? 5 : 6;
      int uo[2], po[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int s = t + 32 * q, in = s & (g.seg - 1), base = (s >> lseg) * half;
        uo[q] = base + in * (HD / 2) + ((r ^ kv4_swz(HD, t)) * (HD / 16));
        po[q] = base + g.seg * (HD / 2) + in * NG * 4;
      }
      // 16-bit inputs: the middle of group r % NG of slot t or t + 32 is this thread's
      const bool mids = !SPLIT && !kv && r < 2 * NG;
      const int xo = (r < NG ? po[0] : po[1]) + r % NG * 4, xr = t + (r < NG ? 0 : 32);
#pragma unroll 1
      for (int i = 0; i < nt; ++i) {
        const int jj = j + i, st = jj % KST, rs = kv ? Sh::RK + jj % Sh::RV : jj % Sh::RK;
        if (!wait(&r_full[rs], (jj / (kv ? Sh::RV : Sh::RK)) & 1)) break;
        const uint8_t* raw = sm + Sh::R_OFF + rs * Sh::RAW;
        uint8_t* d = dst + st * ((kv ? T : KT) * Sh::KB);
        uint32_t w[2][NW], pr[2][NG];
        const int have = r_have[rs], s0 = (tb + i) * BN + t;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          kv4_ldv(raw + uo[q], w[q]);
          kv4_ldv(raw + po[q], pr[q]);
          // past the sequence, or a page outside the pool: zeros (the softmax gives such slots no weight)
          if (s0 + 32 * q >= p.len || !((have >> ((t + 32 * q) >> lseg)) & 1))
#pragma unroll
            for (int k = 0; k < NG; ++k) pr[q][k] = 0u;
          if (vnan)
#pragma unroll
            for (int k = 0; k < NG; ++k)
              if (!(fabsf(kv4_param(pr[q][k]).x) < INFINITY) || !(fabsf(kv4_param(pr[q][k]).y) < INFINITY)) pr[q][k] = 0u;
        }
        float mid = 0.f;
        if (mids) {
          const float2 sb = __half22float2(__hmul2(pt_u2(*reinterpret_cast<const uint32_t*>(raw + xo)), sc));
          mid = fmaf(7.5f, sb.x, sb.y);
        }
        mbar_arrive(&r_empty[rs]);  // the next copy is under way while this tile waits for its buffer
        if (!wait(empty + st, ((jj / KST) & 1) ^ 1)) break;
        if (kv) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int k = 0; k < NW; ++k) {
              uint4 hi, lo;
              pt_unpack<SPLIT>(w[q][k], __hmul2(pt_u2(pr[q][k * 64 / GROUP]), sc), hi, lo);
              *reinterpret_cast<uint4*>(d + q * (32 * 128) + k * (BN * 128)) = hi;
              if (SPLIT) *reinterpret_cast<uint4*>(d + Sh::KB + q * (32 * 128) + k * (BN * 128)) = lo;
            }
        } else {
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int k = 0; k < NW; ++k) {
              uint4 hi, lo;
              const __half2 sb = __hmul2(pt_u2(pr[q][k * 64 / GROUP]), sc);
              if constexpr (SPLIT) pt_unpack<true>(w[q][k], sb, hi, lo);
              else pt_unpack_keys(w[q][k], sb, hi, lo);
              *reinterpret_cast<uint4*>(d + q * (32 * 128) + k * (BN * 128)) = hi;
              *reinterpret_cast<uint4*>(d + Sh::KB + q * (32 * 128) + k * (BN * 128)) = lo;
            }
          if (mids) pt_middles<true>(sm + Sh::XK_OFF + st * Sh::XKB, xr, r % NG, mid);
        }
        fence_proxy_async();
        mbar_arrive(full + st);
      }
    });
  } else {
    pt_regs_dec<PT_REGS_ISSUE>();
    if (warp == PT_MMA) {
      // ------------------------------------------------------ MMA issue ----
      // The warp stays together, so that descriptors live in uniform
      // registers; one elected lane issues.
      constexpr uint32_t ids = pt_idesc(BN, false), idp = pt_idesc(HD, true);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      for_items([&](const PtPlace&, int, int nt, int, int) {
        bar();
        bar();
        tg_fence_after();
        auto qk = [&](int i) {
          const int jj = __shfl_sync(0xffffffffu, j + i, 0), st = jj % KST, b = jj & 1;
          if (!wait(&k_full[st], (jj / KST) & 1)) return false;
          tg_fence_after();
          const uint64_t kd = tg_desc(smem_u32(sm + Sh::K_OFF + st * (KT * Sh::KB)));
          const uint32_t d = tm + Sh::S_COL + b * BN;
          if (pt_elect()) {
            // the small products first; 16 channels are 32 bytes of the 128-byte rows
#pragma unroll
            for (int w = 0; w < NW; ++w)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                pt_mma_ts(d, tm + Sh::Q_COL + w * 32 + k * 8, kd + ((Sh::KB + w * (BN * 128) + k * 32) >> 4), ids, w + k > 0);
            if constexpr (!SPLIT)
              pt_mma_ss(d, pt_desc_x(smem_u32(sm + Sh::XQ_OFF)), pt_desc_x(smem_u32(sm + Sh::XK_OFF + st * Sh::XKB)), ids, true);
            if (SPLIT) {
              const uint64_t qd = tg_desc(smem_u32(sm + Sh::Q_OFF));
#pragma unroll
              for (int w = 0; w < NW; ++w)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  pt_mma_ss(d, qd + ((w * (PT_ROWS * 128) + k * 32) >> 4), kd + ((w * (BN * 128) + k * 32) >> 4), ids, true);
            }
#pragma unroll
            for (int w = 0; w < NW; ++w)
#pragma unroll
              for (int k = 0; k < 4; ++k) pt_mma_ts(d, tm + Sh::Q_COL + w * 32 + k * 8, kd + ((w * (BN * 128) + k * 32) >> 4), ids, true);
            tg_commit(&s_full[b]);
            tg_commit(&k_empty[st]);
          }
          __syncwarp();
          return true;
        };
        bool ok = qk(0);
        for (int i = 0; i < nt && ok; ++i) {
          // S of tile i + 1 takes the columns P of tile i - 1 was read from: products complete in order
          if (i + 1 < nt) ok = qk(i + 1);
          const int jj = __shfl_sync(0xffffffffu, j + i, 0), st = jj % KST, b = jj & 1;
          if (!ok || !wait(&v_full[st], (jj / KST) & 1) || !wait(&p_full[b], (jj >> 1) & 1)) break;
          tg_fence_after();
          const uint64_t vd = pt_desc_n(smem_u32(sm + Sh::V_OFF + st * (T * Sh::KB)), BN * 128);
          const uint32_t pc = tm + Sh::S_COL + b * BN;
          if (pt_elect()) {
            const bool on = SPLIT ? i % PT_FLUSH != 0 : i > 0;  // O goes on
#pragma unroll
            for (int k = 0; k < BN / 16; ++k) {
              if (SPLIT) {
                pt_mma_ts(tm + Sh::O_COL, pc + 32 + k * 8, vd + ((k * 2048) >> 4), idp, k > 0 || on);
                pt_mma_ts(tm + Sh::O_COL, pc + k * 8, vd + ((Sh::KB + k * 2048) >> 4), idp, true);
              }
              pt_mma_ts(tm + Sh::O_COL, pc + k * 8, vd + ((k * 2048) >> 4), idp, SPLIT || k > 0 || on);
            }
            if (!SPLIT && a.dt == DT_F16)
#pragma unroll
              for (int k = 0; k < BN / 16; ++k) pt_mma_ts(tm + Sh::O_COL, pc + 32 + k * 8, vd + ((k * 2048) >> 4), idp, true);
            tg_commit(&o_done[b]);
            tg_commit(&v_empty[st]);
          }
          __syncwarp();
        }
      });
    } else if (warp == PT_COPY || warp == PT_COPY + 1) {
      // --------------------------------------------------- bulk copies ----
      // A stage is a tile's keys with their params, or its values with theirs:
      // one copy a block (one in all from pages of 64 slots on), a lane each.
      const int kv = warp - PT_COPY, ring = kv ? Sh::RV : Sh::RK, base = kv ? Sh::RK : 0;
      const int nblk = g.page / g.seg, np = BN / g.seg, half = g.blk / 2;
      int issued = 0;
      for_items([&](const PtPlace& p, int tb, int nt, int, int) {
        const int* tab = g.table + p.seq * g.tstride;
        // page ids are fetched a tile ahead
        auto page_of = [&](int i) {
          const int s = (tb + i) * BN + lane * g.seg;
          return i < nt && lane < np && s < p.len ? __ldg(tab + (s >> g.pshift)) : -1;
        };
        int pg = page_of(0);
        for (int i = 0; i < nt; ++i, ++issued) {
          const int s = (tb + i) * BN + lane * g.seg, jj = j + i, rs = base + jj % ring;
          const bool on = unsigned(pg) < unsigned(g.npages);
          if (!on && lane < np && s < p.len && a.b.status) atomicOr(a.b.status, KV4_BAD);
          const uint8_t* src = g.pages + pg * g.page_bytes + int64_t(p.h * nblk + (s & (g.page - 1)) / g.seg) * g.blk + kv * half;
          const unsigned have = __ballot_sync(0xffffffffu, on);
          pg = page_of(i + 1);
          if (!wait(&r_empty[rs], ((jj / ring) & 1) ^ 1)) break;
          if (lane == 0) {
            r_have[rs] = int(have);
            mbar_expect_tx(&r_full[rs], unsigned(__popc(have)) * unsigned(half));
          }
          __syncwarp();
          if (on) bulk_g2s_keep(sm + Sh::R_OFF + rs * Sh::RAW + lane * half, src, unsigned(half), &r_full[rs]);
        }
      });
      if (*abort_flag)  // copies in flight land before the CTA may end
        for (int i = max(0, issued - ring); i < issued; ++i) pt_wait(&r_full[base + i % ring], (i / ring) & 1);
    }
  }
  __syncthreads();
  if (warp == PT_MMA) {
    if (*abort_flag) {
      if (pt_elect()) tg_commit(drain);  // the products still in flight
      __syncwarp();
      pt_wait(drain, 0);
    }
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Joins the parts of the item that begins in share x and goes on: a block eight
// rows, a thread eight channels of one (a warp reads four runs of 128 bytes).
template <int HD>
__global__ void __launch_bounds__(HD) k_kv4_prompt_join(const Kv4AttnArgs a) {
  pdl_wait();
  const int UP = pt_up(a.dt == DT_F32);
  const int x = blockIdx.x, j = threadIdx.x >> 3, r = blockIdx.y * 8 + (threadIdx.x & 7);
  const PtJoin d = pt_joins(a)[x];
  if (d.first < 0) return;
  const unsigned ci = unsigned(d.qt * PT_ROWS + r);
  const int tok = int(ci / unsigned(a.rep)), hq = d.h * a.rep + int(ci % unsigned(a.rep));
  const int64_t total = d.total, step = pt_part_floats(HD);
  auto part = [&](int i) { return pt_parts(a) + (int64_t(i) * 2 + (i == x ? 1 : 0)) * step; };
  // shares without tiles (fewer tiles than CTAs) have no part
  auto has = [&](int i) { return i == d.first || total >= PT_GRID || total * i / PT_GRID < total * (i + 1) / PT_GRID; };
  // the row's maximum: four lanes of the warp have the row
  float M = -INFINITY, L = 0.f;
  for (int i = d.first + (j & 3); i <= d.last; i += 4)
    if (has(i)) M = fmaxf(M, __ldcg(part(i) + r));
  M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 8));
  M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 16));
  if (tok >= d.n) return;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll 4
  for (int i = d.first; i <= d.last; ++i) {
    if (!has(i)) continue;
    const float* q = part(i);
    const float4* o4 = reinterpret_cast<const float4*>(q + 2 * PT_ROWS) + 2 * j * PT_ROWS + r;
    const float4 o0 = __ldcg(o4), o1 = __ldcg(o4 + PT_ROWS);
    const float mi = __ldcg(q + r), f = mi == -INFINITY ? 0.f : pt_ex2(mi - M);
    L = fmaf(__ldcg(q + PT_ROWS + r), f, L);
    const float o[8] = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, o1.z, o1.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) v[pt_channel(e)] = fmaf(o[e], f, v[pt_channel(e)]);
  }
  const int64_t row = d.row0 + tok;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = L == 0.f ? v[e] : v[e] / L;  // an empty row: zeros
  if (a.gate.p) {
    float g[8];
    kv4_ld8(a.gate.p, a.dt, row * a.gate.ts + hq * a.gate.hs + j * 8, kv4_vec(a.gate, a.dt), g);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= kv4_sigmoid(g[e]);
  }
  kv4_st8(a.out.p, a.dt, row * a.out.ts + hq * a.out.hs + j * 8, kv4_vec(a.out, a.dt), v);
  if (j == 0) pt_lse(a)[row * a.heads + hq] = L == 0.f ? -INFINITY : (M + log2f(L * pt_pow2(-UP))) * P_LN2;
}

// ------------------------------------------------------- accumulated weight --
// weights[t] += sum over the rows that see slot t of exp(score - lse): S^T = K
// Q^T by tcgen05.mma with 128 slots as M (a thread a slot and half of the
// columns, so the sums stay in a register) and 64 query rows as N. The slots'
// keys are unpacked once, into TMEM; the queries come as f16 tiles that
// k_kv4_queries lays out once for all of them. A CTA owns its slots: every sum
// has one order. Bound: 512 cycles of MMA (16-bit inputs, 256 channels) and 512
// of exponentials a step of 128 x 64. 1000 tokens on 3000 slots (2 kv heads of
// 256 channels, 16 query heads, bf16): 115 us, where the kernel for few rows
// took 1390.
constexpr int WQ_COLS = 64;  // query rows of a tile

template <int HD, bool SPLIT>
struct WqShape {
  static constexpr int T = SPLIT ? 2 : 1;
  static constexpr int TILE = WQ_COLS * HD * 2;             // one term of a tile's queries
  static constexpr int BLOB = T * TILE + WQ_COLS * 16;      // with {factor, log2 of the sum, last slot, 0} a row
  static constexpr int ST = 3;
  static constexpr int BAR_OFF = (ST * BLOB + 1023) / 1024 * 1024;
  static constexpr int TOTAL = BAR_OFF + (2 * ST + 5) * 8 + 16 + 128 * 4 + 1024;
  static constexpr int COLS = 2 * WQ_COLS + HD <= 256 ? 256 : 512;  // TMEM: S twice, two terms of the keys
  static constexpr int K_COL = 2 * WQ_COLS;
};
constexpr int WQ_THREADS = 320;  // 8 warps of slots, the MMA warp, the copy warp

// First tile of a sequence's queries of a kv head (ceil(n rep / 64) of them fit before the next sequence's).
__host__ __device__ inline int64_t wq_first(int64_t row0, int rep, int seq) { return row0 * rep / WQ_COLS + seq; }
__host__ __device__ inline int64_t wq_tiles(int64_t total, int rep, int nseq) { return total * rep / WQ_COLS + nseq + 1; }

// A warp a (row, query head).
template <int HD, bool SPLIT>
__global__ void __launch_bounds__(256) k_kv4_queries(const Kv4AttnArgs a) {
  using Sh = WqShape<HD, SPLIT>;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t wid = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t j = wid / a.heads;
  const int hq = int(wid - j * a.heads), h = hq / a.rep;
  if (j >= a.b.total) return;
  int lo_s = 0, hi_s = a.b.nseq;  // the sequence the row belongs to
  while (lo_s < hi_s) {
    const int mid = (lo_s + hi_s) >> 1;
    if (__ldg(a.b.start + mid + 1) <= j) lo_s = mid + 1; else hi_s = mid;
  }
  if (lo_s >= a.b.nseq) return;
  int row0;
  const int n = kv4_new(a.b, lo_s, row0), len = kv4_len(a.b, lo_s), t = int(j) - row0;
  if (t < 0 || t >= n) return;
  const int ci = t * a.rep + hq - h * a.rep, r = ci % WQ_COLS;
  uint8_t* blob = reinterpret_cast<uint8_t*>(pt_parts(a)) +
                  (h * wq_tiles(a.b.total, a.rep, a.b.nseq) + wq_first(row0, a.rep, lo_s) + ci / WQ_COLS) * Sh::BLOB;
  float x[8], am = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  if (lane < HD / 8) kv4_ld8(a.q.p, a.dt, j * a.q.ts + hq * a.q.hs + lane * 8, kv4_vec(a.q, a.dt), x);
#pragma unroll
  for (int e = 0; e < 8; ++e) am = fmaxf(am, fabsf(x[e]));
  am = warp_max(am);
  int ex = am > 0.f && am < INFINITY ? 12 - (int(__float_as_uint(am) >> 23) - 127) : 0;
  ex = max(-100, min(100, ex));
  const float up = pt_pow2(ex);
  if (lane < HD / 8) {
    uint4 hi, lo;
    uint32_t *H = &hi.x, *L = &lo.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // the order the codes come unpacked in
      const float v0 = x[i] * up, v4 = x[i + 4] * up;
      const __half2 hh = __floats2half2_rn(v0, v4);
      H[i] = pt_h2(hh);
      if (SPLIT) {
        const float2 ff = __half22float2(hh);
        L[i] = pt_h2(__floats2half2_rn(v0 - ff.x, v4 - ff.y));
      }
    }
    const int off = (lane >> 3) * (WQ_COLS * 128) + r * 128 + (((lane & 7) ^ (r & 7)) << 4);
    *reinterpret_cast<uint4*>(blob + off) = hi;
    if (SPLIT) *reinterpret_cast<uint4*>(blob + Sh::TILE + off) = lo;
  }
  if (lane == 0)
    reinterpret_cast<float4*>(blob + Sh::T * Sh::TILE)[r] =
        make_float4(a.scale * P_LOG2E * pt_pow2(-ex), pt_lse(a)[j * a.heads + hq] * P_LOG2E, __int_as_float(len - n + t), 0.f);
}

template <int HD, int GROUP, bool SPLIT>
__global__ void __launch_bounds__(WQ_THREADS, SPLIT ? 1 : 2) k_kv4_prompt_weights(const Kv4AttnArgs a) {
  using Sh = WqShape<HD, SPLIT>;
  constexpr int T = Sh::T, ST = Sh::ST, NG = HD / GROUP, NW = HD / 64, HC = WQ_COLS / 2;
  extern __shared__ __align__(1024) uint8_t wq_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(wq_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sm + Sh::BAR_OFF);
  uint64_t *q_empty = q_full + ST, *s_full = q_empty + ST, *s_empty = s_full + 2, *drain = s_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* half_sum = reinterpret_cast<float*>(tmem_slot + 4);
  pdl_wait();
  const Kv4Geo& g = a.g;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y, seq = blockIdx.z;
  int row0;
  const int n = kv4_new(a.b, seq, row0), len = kv4_len(a.b, seq), tile0 = blockIdx.x * 128;
  if (tile0 >= len || n == 0) return;
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1 + 256);  // the MMAs that read the tile, the threads that read its rows' factors
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 256);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(Sh::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tg_fence_before();
  __syncthreads();
  tg_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto fail = [&]() {
    if (a.b.status) atomicOr(a.b.status, 1);
    *abort_flag = 1;
  };
  auto wait = [&](uint64_t* b, unsigned ph) {
    if (__all_sync(0xffffffffu, pt_wait(b, ph) && !*abort_flag)) return true;
    fail();
    return false;
  };
  // the query tiles that hold a row that sees the first slot
  const int q0 = max(0, tile0 - (len - n)) * a.rep / WQ_COLS, nq = (n * a.rep + WQ_COLS - 1) / WQ_COLS - q0;
  const int row = tid & 127, hf = (tid >> 7) & 1, slot = tile0 + row;
  const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
  bool there = false;
  float kscale = 1.f;
  if (warp < 8) {
    // the slot's keys, half of the units of each 64-channel block, to TMEM
    unsigned mk = 0u;
    if (lane < RG_SPLIT) mk = unsigned(__ldcg(pt_ranges(a) + (int64_t(seq) * g.kvh + h) * RG_SPLIT + lane).x);
    const int kx = pt_exp(__reduce_max_sync(0xffffffffu, mk));
    kscale = pt_pow2(-kx);
    const __half2 sc = __float2half2_rn(pt_pow2(kx));
    const uint8_t* blk = slot < len ? kv4_block(g, g.table, g.tstride, seq, h, slot, a.b.status) : nullptr;
    there = blk != nullptr;
    uint32_t w[4][NW], pr[NG];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < NW; ++k) w[u][k] = 0u;
#pragma unroll
    for (int k = 0; k < NG; ++k) pr[k] = 0u;
    if (blk) {
      const int t = slot & (g.seg - 1);
#pragma unroll
      for (int u = 0; u < 4; ++u) kv4_ldv(blk + t * (HD / 2) + ((hf * 4 + u) ^ kv4_swz(HD, t)) * (HD / 16), w[u]);
      kv4_ldv(blk + g.seg * (HD / 2) + t * NG * 4, pr);
    }
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      uint32_t hi[16], lo[16];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        pt_unpack<true>(w[u][k], __hmul2(pt_u2(pr[k * 64 / GROUP]), sc), *reinterpret_cast<uint4*>(hi + 4 * u), *reinterpret_cast<uint4*>(lo + 4 * u));
      pt_st16(lanes + Sh::K_COL + k * 32 + hf * 16, hi);
      pt_st16(lanes + Sh::K_COL + HD / 2 + k * 32 + hf * 16, lo);
    }
    pt_st_wait();
    tg_fence_before();
  }
  __syncthreads();
  tg_fence_after();
  if (warp < 8) {
    float s4[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < nq; ++i) {
      const int b = i & 1, st = i % ST;
      // the copy is complete when its products are; the wait makes it visible here
      if (!wait(&s_full[b], (i >> 1) & 1) || !wait(&q_full[st], (i / ST) & 1)) break;
      tg_fence_after();
      uint32_t s[HC];
      pt_ld32(lanes + b * WQ_COLS + hf * HC, s);
      tg_ld_wait();
      tg_fence_before();
      mbar_arrive(&s_empty[b]);
      const float4* meta = reinterpret_cast<const float4*>(sm + st * Sh::BLOB + T * Sh::TILE) + hf * HC;
      const int left = n * a.rep - (q0 + i) * WQ_COLS - hf * HC;  // rows of the tile from this half's first on
      if (left >= HC && tile0 + 127 <= __float_as_int(meta[0].z)) {
#pragma unroll
        for (int e = 0; e < HC; ++e) {
          const float4 f = meta[e];
          s4[e & 3] += pt_ex2(fmaf(__uint_as_float(s[e]), f.x * kscale, -f.y));
        }
      } else {
#pragma unroll
        for (int e = 0; e < HC; ++e) {
          const float4 f = meta[e];
          if (e < left && slot <= __float_as_int(f.z)) s4[e & 3] += pt_ex2(fmaf(__uint_as_float(s[e]), f.x * kscale, -f.y));
        }
      }
      mbar_arrive(&q_empty[st]);
    }
    const float sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
    if (hf) half_sum[row] = sum;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (!hf && there) a.weights[(int64_t(seq) * g.kvh + h) * a.wstride + slot] += sum + half_sum[row];
  } else if (warp == 8) {
    constexpr uint32_t ids = pt_idesc(WQ_COLS, false);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    for (int i = 0; i < nq; ++i) {
      const int b = i & 1, st = i % ST;
      if (!wait(&q_full[st], (i / ST) & 1) || !wait(&s_empty[b], ((i >> 1) & 1) ^ 1)) break;
      tg_fence_after();
      const uint64_t qd = tg_desc(smem_u32(sm + st * Sh::BLOB));
      if (pt_elect()) {
        // the small products first
        const uint32_t d = tm + b * WQ_COLS;
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t ak = tm + Sh::K_COL + w * 32 + k * 8;
            const uint64_t bd = qd + ((w * (WQ_COLS * 128) + k * 32) >> 4);
            pt_mma_ts(d, ak + HD / 2, bd, ids, w + k > 0);
            if (SPLIT) pt_mma_ts(d, ak, bd + (Sh::TILE >> 4), ids, true);
          }
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            pt_mma_ts(d, tm + Sh::K_COL + w * 32 + k * 8, qd + ((w * (WQ_COLS * 128) + k * 32) >> 4), ids, true);
        tg_commit(&s_full[b]);
        tg_commit(&q_empty[st]);
      }
      __syncwarp();
    }
  } else {
    const uint8_t* src = reinterpret_cast<const uint8_t*>(pt_parts(a)) +
                         (h * wq_tiles(a.b.total, a.rep, a.b.nseq) + wq_first(row0, a.rep, seq) + q0) * Sh::BLOB;
    int i = 0;
    for (; i < nq; ++i) {
      const int st = i % ST;
      if (!wait(&q_empty[st], ((i / ST) & 1) ^ 1)) break;
      if (lane == 0) {
        mbar_expect_tx(&q_full[st], Sh::BLOB);
        bulk_g2s_keep(sm + st * Sh::BLOB, src + int64_t(i) * Sh::BLOB, Sh::BLOB, &q_full[st]);
      }
      __syncwarp();
    }
    if (*abort_flag)  // copies in flight land before the CTA may end
      for (int k = max(0, i - ST); k < i; ++k) pt_wait(&q_full[k % ST], (k / ST) & 1);
  }
  tg_fence_before();
  __syncthreads();
  tg_fence_after();
  if (warp == 8) {
    if (*abort_flag) {
      if (pt_elect()) tg_commit(drain);  // the products still in flight
      __syncwarp();
      pt_wait(drain, 0);
    }
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Sh::COLS));
  }
}

template <int HD, int GROUP, bool SPLIT>
void run(const Kv4AttnArgs& a, cudaStream_t st) {
  using Sh = PtShape<HD, GROUP, SPLIT>;
  launch(k_kv4_range, dim3(a.b.nseq * a.g.kvh, RG_SPLIT), dim3(256), 0, st, true, a);
  launch(k_kv4_prompt<HD, GROUP, SPLIT>, dim3(PT_GRID), dim3(PT_THREADS), Sh::TOTAL, st, true, a);
  if (a.b.max_len > PT_BN)  // or every item is one tile, and written at once
    launch(k_kv4_prompt_join<HD>, dim3(PT_GRID, PT_ROWS / 8), dim3(HD), 0, st, true, a);
  if (a.weights && a.b.max_len > 0) {
    const int64_t rows = int64_t(a.b.total) * a.heads;
    launch(k_kv4_queries<HD, SPLIT>, dim3(unsigned((rows + 7) / 8)), dim3(256), 0, st, true, a);
    launch(k_kv4_prompt_weights<HD, GROUP, SPLIT>, dim3((a.b.max_len + 127) / 128, a.g.kvh, a.b.nseq), dim3(WQ_THREADS),
           WqShape<HD, SPLIT>::TOTAL, st, true, a);
  }
}

template <int HD, int GROUP>
void run_dt(const Kv4AttnArgs& a, cudaStream_t st) {
  if (a.dt == DT_F32) run<HD, GROUP, true>(a, st);
  else run<HD, GROUP, false>(a, st);
}

}  // namespace

int64_t kv4_prompt_work(const Kv4Geo& g, const Kv4Batch& b, int heads) {
  // the parts' space holds the weight kernel's queries after them (as for f32, the larger)
  const int rep = heads / g.kvh;
  const int64_t parts = int64_t(PT_GRID) * 2 * pt_part_floats(g.hd) * 4;
  const int64_t queries = g.kvh * wq_tiles(b.total, rep, b.nseq) * (2 * WQ_COLS * g.hd * 2 + WQ_COLS * 16);
  return pt_lse_bytes(b.total, heads) + pt_range_bytes(b.nseq, g.kvh) + PT_GRID * int64_t(sizeof(PtJoin)) + std::max(parts, queries);
}

void launch_kv4_prompt(const Kv4AttnArgs& a, cudaStream_t st) {
  if (int64_t(a.b.total) * a.rep > 0x7fffff00) throw Error(ERR_UNSUPPORTED, "kv4: more than 2^31 query rows a kv head");
  if (a.g.hd == 64) run_dt<64, 64>(a, st);
  else if (a.g.hd == 128) a.g.group == 64 ? run_dt<128, 64>(a, st) : run_dt<128, 128>(a, st);
  else a.g.group == 64 ? run_dt<256, 64>(a, st) : run_dt<256, 128>(a, st);
}

}  // namespace swl
