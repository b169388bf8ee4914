// Attention of a batch over the paged latent cache, the prefix that the batch shares read once for all of it.
//
// out[b, s, h] = sum_j p_j k_j[0:512], p = softmax_j(scale * q[b, s, h] . k_j), j over the tokens that step s of sequence b sees:
// the shared prefix, and its own tokens up to the one of step s (the last S of its own tokens are the S steps).  A latent row is
// key (576 columns) and value (its first 512) at once, so a tile of tokens is loaded once and used by two products.
//
// Work.  All rows (b, s, h) in tiles of 64 against the prefix, and each sequence's rows in tiles of 64 against its own
// tokens, in tiles of 128 tokens (two pages): every (row tile, token tile) pair costs the same, and a row tile about kStart pairs more (its
// queries in, its outputs out), so the pairs are laid in one line, row tile by row tile, kStart empty places before each, and each CTA
// takes an equal stretch, whatever the lengths are.  A stretch that covers a part of a row tile
// leaves an unnormalised f32 output with its maximum and sum in the workspace (one pass over the tokens, running maximum and
// sum in 32 bits), and a second, dependent launch joins the parts of each row.  Lengths and tables are read on the device:
// a captured graph follows them.  Nothing is accumulated by atomics: the same inputs give the same bits.
//
// One CTA per SM, warps with fixed roles, one tile after another:
//   8 softmax warps  S from tensor memory, running maximum, P = 2^(S - m) rounded to 16 bits into shared memory; O scaled, read and written out;
//   16 loader warps  fetch the next tile's codes into registers and make 16-bit floats of them in 128-byte-swizzled shared memory, in nine
//                    16 KB chunks of 64 columns;
//   1 planning warp  this CTA's stretches, one after another, into a ring that the others read;
//   1 MMA warp       S = Q K^T (64 x 128, chunk by chunk as they come) and O += P V (64 x 512 in tensor memory), both tcgen05.mma.ws, M = 64.
// Why M = 64: a 128-row O of 512 columns fills the whole tensor memory and leaves no room for S.  The weight-stationary form puts
// a 64-row tile on all 128 lanes and reaches 48 cycles per 64 x 128 x 16 step, the plain form 64 (measured; 32 would be full rate).
// Why 128 tokens: the 64 x 64 x 16 step of S costs 44 cycles.  Why O in four products of 128 columns: the slots of a pair of chunks
// are free for the next tile after a quarter of P V.  The queries' rope columns lie in tensor memory, which makes room for P.
//
// Types.  bf16 pages are multiplied as bf16.  MXFP8 codes become f16, not bf16: one conversion and one product for two codes, a third of what bf16
// takes (which has no conversion from E4M3), and the loaders' instructions are what a tile waits for.  f16 has the bits (a code has four), but not the
// range, so exponents are taken out: of the scales of 8 tokens the largest, E (K' = code * 2^(e - E), exact down to 2^-24 of 2^E), of
// a query row its own (the largest element is brought to 2^14..2^15; what that costs is below 2^-39 of it).  They come back in f32: S = 2^(E + row) S' + S_rope
// (the rope columns are multiplied as bf16 into a second accumulator), and P' = 2^(S + E - m), with m the running maximum of S + E, so
// that P' V' has the weight of P V.  P is rounded because both operands of the matrix instructions are 16 bits; the sums of P stay unrounded in f32.
// The m that P' is relative to follows the true maximum only when it falls behind by more than 2^4 (O is then rescaled): the ratio is
// exact either way.  P' is kept in 2^-24 .. 2^14, with 2^10 at the maximum: tokens are lost below 2^-34 of the largest.
#include <cuda_runtime.h>

#include "latent_page.cuh"
#include "k3g_host.h"

using namespace k3g;

namespace {

constexpr int kMaxBatch = 4096, kMaxRowsPerSeq = 1 << 15, kMaxCtas = 160;
constexpr int kRows = 64, kTile = 128;                       // query rows and tokens of a tile
constexpr int kSoftmax = 256, kLoaders = 512, kThreads = kSoftmax + kLoaders + 128;   // the last four warps: MMAs, planning, two idle
constexpr int kChunk = kTile * 128;                          // 64 columns of a tile's tokens, bf16
constexpr int kQChunk = kRows * 128;
constexpr int kSmemQ = 8 * kQChunk, kSmemP = 2 * kQChunk, kSmemK = 9 * kChunk, kSmem = kSmemQ + kSmemP + kSmemK + 1024;
// tensor memory columns: O 0..255 (four accumulators of 128 output columns, 64 on either half of the lanes), S 256..319 (64 tokens on either
// half), the rope columns' part of S 320..383 (MXFP8), the queries' rope columns 384..415 (the same on both halves)
constexpr int kTmemS = 256, kTmemR = 320, kTmemQ = 384;
constexpr int kLeastE = -80, kMostE = 120;                   // exponents of 8 tokens: sums of 2^-E stay in range
constexpr float kLag = 4.f, kTop = 10.f;
constexpr int kPartFloats = kRows * kLatent;                 // a part's outputs; its 64 (maximum, sum) pairs lie in a table of their own
constexpr int kWaitLimit = 1 << 20, kRing = 4, kReaders = (kSoftmax + kLoaders) / 32 + 1;
constexpr int kStart = 2;

struct AttnArgs {
  const __nv_bfloat16* q; long long q_stride;
  const unsigned char* cache; long long page_stride, pages;       // bytes
  const int* prefix_table; const int* prefix_len; int prefix_pages;
  const int* block_table; const int* lens; int max_pages;
  __nv_bfloat16* out;
  int* status;                       // [kMaxCtas] 1: a wait of this CTA expired
  int2* spans;                       // [row tiles] first and last CTA of each (unwritten where there are no tokens)
  float2* sums;                      // [parts][64] (maximum in log2 units, sum)
  float* parts;                      // [parts][64][512]
  int B, S, heads, prefix_tiles, seq_tiles, ctas;
  float c;                           // |scale| * log2(e), above 0 (scores are compared before they are scaled)
  int flip;                          // the scale is negative
};

__device__ __forceinline__ unsigned su(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }

// ---- lengths and the line of (row tile, token tile) pairs ------------------------------------------------------------------
__device__ __forceinline__ int prefix_tokens(const AttnArgs& a) {
  return a.prefix_pages ? max(0, (int)min((long long)__ldg(a.prefix_len), (long long)a.prefix_pages * kPageTokens)) : 0;
}
__device__ __forceinline__ int own_tokens(const AttnArgs& a, int b) {
  return max(0, (int)min((long long)__ldg(a.lens + b), (long long)a.max_pages * kPageTokens));
}
__device__ __forceinline__ int tiles_of(int tokens) { return (tokens + kTile - 1) / kTile; }
__device__ __forceinline__ int places_of(int tokens) { return tokens ? tiles_of(tokens) + kStart : 0; }   // on the line
struct Segment {                     // one CTA's stretch of one row tile
  int tile;                          // row tile: prefix_tiles of them against the prefix, then seq_tiles for each sequence
  int b;                             // sequence, or -1 for the prefix
  int row0;                          // first row: of all rows (prefix) or of the sequence's rows
  int t0, t1;                        // token tiles (none: the end)
  int tokens;                        // tokens of the prefix / of the sequence
  const int* table;
};

// ---- barriers and tensor memory -----------------------------------------------------------------------------------------------
struct Control {
  unsigned long long full[5], empty[4], q_full, s_full, p_full[2];
  unsigned long long ring_full[kRing], ring_empty[kRing];
  Segment ring[kRing];
  unsigned tmem;
  int abort;
  int first_tile, first_at;
  long long scan[kThreads / 32], left;
  unsigned poison[2][4];
  int exponent[2][16];                                        // E of each 8 tokens of a tile
  float row_scale[kRows];                                     // 2^(what was taken out of a query row)
  float best[4][kRows];                                      // the maxima of a tile, and at a segment's end the sums
};

// Every wait ends: after kWaitLimit polls, or as soon as another wait of the CTA has expired.  The roles then run through what is
// left without waiting (every access stays where it was), and the call's result is NaN.
__device__ __forceinline__ void wait(Control& k, unsigned long long& bar, unsigned parity) {
#pragma unroll 1
  for (int i = 0; i < kWaitLimit; ++i) {
    unsigned ok;
    asm volatile("{.reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}" : "=r"(ok) : "r"(su(&bar)), "r"(parity) : "memory");
    if (ok) return;
    if (*(volatile int*)&k.abort) return;
  }
  *(volatile int*)&k.abort = 1;
}
__device__ __forceinline__ void arrive(unsigned long long& bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(su(&bar)) : "memory"); }
__device__ __forceinline__ void commit(unsigned lead, unsigned long long& bar) {
  asm volatile("{.reg .pred e; setp.ne.b32 e, %1, 0; @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];}" :: "r"(su(&bar)), "r"(lead) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Segment n of the CTA, for a whole warp; `release`: the ring may reuse its place.
__device__ __forceinline__ Segment segment(Control& k, unsigned n, bool release) {
  wait(k, k.ring_full[n % kRing], (n / kRing) & 1);
  const Segment s = k.ring[n % kRing];
  __syncwarp();
  if (release && (threadIdx.x & 31) == 0) arrive(k.ring_empty[n % kRing]);
  return s;
}

// Shared-memory operand descriptor, low word: address and bytes between groups of 64 columns (of the transposed operand).  The high word is the
// same for all: 128-byte swizzle, 1024 bytes between groups of eight 128-byte rows.
__device__ __forceinline__ unsigned operand(unsigned addr, unsigned lead) { return ((addr & 0x3ffffu) >> 4) | ((lead >> 4) << 16); }
// Run by a whole warp, whose elected thread issues: operands that are the same in all lanes stay in uniform registers.
__device__ __forceinline__ void mma_ws(unsigned lead, unsigned d, unsigned a, unsigned b, unsigned shape, bool add) {
  asm volatile("{.reg .pred p, e; .reg .b64 x, y; mov.b64 x, {%1, %6}; mov.b64 y, {%2, %6}; setp.ne.b32 p, %4, 0; setp.ne.b32 e, %5, 0; "
               "@e tcgen05.mma.ws.cta_group::1.kind::f16 [%0], x, y, %3, p;}"
               :: "r"(d), "r"(a), "r"(b), "r"(shape), "r"((unsigned)add), "r"(lead), "r"((1024u >> 4) | (1u << 14) | (2u << 29)) : "memory");
}
__device__ __forceinline__ void mma_ws_tmem(unsigned lead, unsigned d, unsigned a, unsigned b, unsigned shape, bool add) {   // first operand in tensor memory
  asm volatile("{.reg .pred p, e; .reg .b64 y; mov.b64 y, {%2, %6}; setp.ne.b32 p, %4, 0; setp.ne.b32 e, %5, 0; "
               "@e tcgen05.mma.ws.cta_group::1.kind::f16 [%0], [%1], y, %3, p;}"
               :: "r"(d), "r"(a), "r"(b), "r"(shape), "r"((unsigned)add), "r"(lead), "r"((1024u >> 4) | (1u << 14) | (2u << 29)) : "memory");
}
// f32 accumulator, M = 64, N = 128, operands f16 or bf16; `t`: the second operand is stored with its N side contiguous
__device__ __forceinline__ constexpr unsigned shape_of(bool bf16, int t) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((unsigned)t << 16) | ((128u >> 3) << 17) | (4u << 24);
}

#define K3G_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define K3G_I8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
__device__ __forceinline__ void tmem_ld32(unsigned at, unsigned (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : K3G_R8(v, 0), K3G_R8(v, 8), K3G_R8(v, 16), K3G_R8(v, 24) : "r"(at));
}
__device__ __forceinline__ void tmem_st32(unsigned at, const unsigned (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
               :: K3G_I8(v, 0), K3G_I8(v, 8), K3G_I8(v, 16), K3G_I8(v, 24), "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// ---- loaders ----------------------------------------------------------------------------------------------------------------------
// Warp w looks after tokens 8 w .. 8 w + 7 of a tile, in two steps j of four tokens (token 8 w + 4 j + lane / 8), eight lanes to a token:
// an access of the warp is four runs of 128 bytes.
__device__ __forceinline__ unsigned clean(unsigned w, unsigned top, unsigned& bad) {   // a pair of 16-bit floats with NaN and infinities taken out
  if ((w & top) == top) { w &= 0xffff0000u; bad = 1; }
  if ((w & (top << 16)) == (top << 16)) { w &= 0x0000ffffu; bad = 1; }
  return w;
}
// 16-byte unit u (8 columns) of a token's row in a chunk, swizzled
__device__ __forceinline__ int unit_at(int token, int u) { return token * 128 + ((u ^ (token & 7)) << 4); }
__device__ __forceinline__ uint4 fetch(const unsigned char* p) {
  const V8 v = ld_stream(p);
  return make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
}
__device__ __forceinline__ void copy16(unsigned char* dst, const unsigned char* src, bool live) {   // zeros where there is no row
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(su(dst)), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_left() { asm volatile("cp.async.wait_group %0;" :: "n"(LEFT) : "memory"); }

// The token tiles of a CTA one after another, through its segments.
struct Cursor {
  Segment s;
  unsigned n;
  int t;
  __device__ __forceinline__ void start(Control& k) { n = 0; s = segment(k, 0, true); t = s.t0; }
  __device__ __forceinline__ bool live() const { return s.t1 > 0; }
  __device__ __forceinline__ void step(Control& k) {
    if (live() && ++t == s.t1) { s = segment(k, ++n, true); t = s.t0; }
  }
  // page of tokens first .. of the tile, -1 where there is none, and how many of the page's tokens there are
  __device__ __forceinline__ int page(int first, int& tokens) const {
    const int at = t * kTile + (first & 64);               // tokens: at most 2^26
    tokens = live() ? max(0, min(64, s.tokens - at)) : 0;
    return tokens ? __ldg(s.table + (at >> 6)) : -1;
  }
  // steps of a sequence do not see all of its last S - 1 tokens: a value that is not finite must not reach the others through 0 * NaN
  __device__ __forceinline__ bool careful(const AttnArgs& a) const { return live() && s.b >= 0 && a.S > 1 && (t + 1) * kTile > s.tokens - (a.S - 1); }
};

__device__ __forceinline__ void store16(unsigned at, unsigned x, unsigned y, unsigned z, unsigned w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// 2^-d as a pair of f16 (255 stands for NaN), and four E4M3 codes times it: exact but for what falls below f16's 2^-24.
__device__ __forceinline__ unsigned f16_scale(unsigned d) {
  const unsigned h = d <= 14 ? (15u - d) << 10 : d == 255 ? 0x7e00u : 1024u >> min(d - 14u, 31u);
  return h * 0x10001u;
}
__device__ __forceinline__ void mx8_to_f16x4(unsigned codes, unsigned scale, unsigned& lo, unsigned& hi) {
  asm("{.reg .b16 a, b; .reg .b32 x, y; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 x, a; cvt.rn.f16x2.e4m3x2 y, b; mul.rn.f16x2 %0, x, %3; mul.rn.f16x2 %1, y, %3;}"
      : "=r"(lo), "=r"(hi) : "r"(codes), "r"(scale));
}

// What the warp has just written of one or two chunks, without its NaN and infinities (rare: a rolled loop, out of the way).
__device__ __noinline__ void clean_pair(unsigned char* chunk, int steps, int token, int l, unsigned top, unsigned& bad) {
  __syncwarp();                                              // units are cleaned by the lane that owns their column here, whoever wrote them
#pragma unroll 1
  for (int x = 0; x < steps; ++x) {
    uint4* at = reinterpret_cast<uint4*>(chunk + (x >> 1) * kChunk + unit_at(token + 4 * (x & 1), l));
    unsigned b = 0;
    const uint4 v = *at;
    *at = make_uint4(clean(v.x, top, b), clean(v.y, top, b), clean(v.z, top, b), clean(v.w, top, b));
    bad |= b << (x & 1);
  }
}

// Chunks are handed over in pairs (0 1, 2 3, 4 5, 6 7, and the rope chunk), a fence and an arrival for each; a pair's slots are free as soon as
// its 128 columns of P V are done, the rope slot before that.  The page of a tile is looked up two tiles ahead.  Its codes are fetched into registers,
// all in one go, when the tile before it has been handed over: they arrive while that one is multiplied.  (Fetched pair by pair
// they wait for each other: a warp has few scoreboards to wait on.)  bf16 rows are twice as many registers: pairs 0 and 1 are held, the others are
// copied straight into their slots once those are free.
template <bool MX8>
__device__ void load_tiles(const AttnArgs& a, Control& k, unsigned char* slots, int tid) {
  const int lane = tid & 31, first = (tid >> 5) * 8, sub = lane >> 3, l = lane & 7;
  const int row0 = (first & 56) + sub;                       // row in its page of step 0's token
  Cursor cur;
  cur.start(k);
  constexpr int kHeld = MX8 ? 4 : 2, kPer = MX8 ? 2 : 4;     // held[pair][step]: 16 codes; bf16 held[pair][chunk, step]: 8 columns
  uint4 held[kHeld][kPer], scales = make_uint4(0u, 0u, 0u, 0u);   // lane x holds the scale bytes of token `first` + x % 8
#pragma unroll
  for (int p = 0; p < kHeld; ++p)
#pragma unroll
    for (int x = 0; x < kPer; ++x) held[p][x] = scales;
  // where the thread's first unit of step j goes (j even, j odd): the swizzle of token 8 w + 4 j + sub is sub + 4 j
  unsigned put[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int unit = MX8 ? 2 * (l & 3) + (l >> 2) : l;
    put[x] = su(slots) + (MX8 ? (l >> 2) * kChunk : 0) + (first + sub) * 128 + ((unit ^ (sub + 4 * x)) << 4);
  }
  int tokens = 0, next_tokens;                               // tokens of this warp's page in this tile (none of a page that the cache does not hold)
  const unsigned char* page = a.cache;
  int next_id = cur.page(first, next_tokens);
  bool careful = false, next_careful = cur.careful(a);
  for (unsigned i = 0;; ++i) {                               // i: tiles done by this CTA
    if (!cur.live()) return;
    tokens = next_id >= 0 && next_id < a.pages ? next_tokens : 0;
    careful = next_careful;
    if (tokens > 0) {
      page = a.cache + next_id * a.page_stride;
      if (MX8) scales = fetch(page + kPageScales + ((first & 56) + (lane & 7)) * (kLatent / 32));
      else scales = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int p = 0; p < kHeld; ++p)
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
          const int row = row0 + 4 * (x & 1);
          held[p][x] = fetch(MX8 ? page + row * kLatent + p * 128 + l * 16 : page + (row * kRow + (2 * p + (x >> 1)) * 64 + l * 8) * 2);
        }
    }
    cur.step(k);
    next_id = cur.page(first, next_tokens);
    next_careful = cur.careful(a);
    auto copy = [&](int c) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = row0 + 4 * j;
        const unsigned char* src = MX8 ? page + kPageRope + row * 128 + l * 16 : page + (row * kRow + c * 64 + l * 8) * 2;
        copy16(slots + c * kChunk + unit_at(first + 4 * j + sub, l), row < tokens ? src : reinterpret_cast<const unsigned char*>(a.q), row < tokens);
      }
    };
    const bool whole = tokens == kPageTokens;
    int E = 0;
    if (MX8) {
      // E, the largest exponent of the warp's tokens, and each block's distance from it (255: a scale that is NaN)
      const uint4 nan = make_uint4(__vcmpeq4(scales.x, ~0u), __vcmpeq4(scales.y, ~0u), __vcmpeq4(scales.z, ~0u), __vcmpeq4(scales.w, ~0u));
      unsigned m = __vmaxu4(__vmaxu4(scales.x & ~nan.x, scales.y & ~nan.y), __vmaxu4(scales.z & ~nan.z, scales.w & ~nan.w));
      m = max(max(m & 255u, (m >> 8) & 255u), max((m >> 16) & 255u, m >> 24));
      m = (first & 56) + (lane & 7) < tokens ? m : 0u;
      m = __reduce_max_sync(0xffffffffu, m);
      m = min(max(m, (unsigned)(127 + kLeastE)), (unsigned)(127 + kMostE));
      E = (int)m - 127;
      m *= 0x01010101u;
      scales = make_uint4(__vsubus4(m, scales.x) | nan.x, __vsubus4(m, scales.y) | nan.y, __vsubus4(m, scales.z) | nan.z, __vsubus4(m, scales.w) | nan.w);
    }
    unsigned bad = 0;                                        // bit j: step j's token has a value that is not finite
#pragma unroll 1
    for (int p = 0; p < 4; ++p) {                            // rolled: the pair at hand is always held[0]; unrolled, the warps wait for instructions
      if (i > 0) wait(k, k.empty[p], (i - 1) & 1);
      if (p == 0) {
        if (tid < 4) k.poison[(i + 1) & 1][tid] = 0;         // the tile before this one has been read, the next is not there yet
        if (MX8 && lane == 0) k.exponent[i & 1][first >> 3] = E;
        copy(8);
        copies_commit();
      }
      const unsigned at = 2 * p * kChunk;
      if (MX8) {
        unsigned sc[2];
        uint4 u[2], v[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) sc[j] = __shfl_sync(0xffffffffu, scales.x, 4 * j + sub);
#pragma unroll
        for (int j = 0; j < 2; ++j) {                        // 16 codes: two units of one chunk
          const unsigned s = f16_scale((sc[j] >> ((l >> 1) * 8)) & 0xffu);
          // lanes 0..3 and 4..7 write to the same columns of two chunks: in opposite order, so that no bank is wanted twice
          const uint4 q = held[0][j];
          const bool back = l >= 4;
          mx8_to_f16x4(back ? q.z : q.x, s, u[j].x, u[j].y); mx8_to_f16x4(back ? q.w : q.y, s, u[j].z, u[j].w);
          mx8_to_f16x4(back ? q.x : q.z, s, v[j].x, v[j].y); mx8_to_f16x4(back ? q.y : q.w, s, v[j].z, v[j].w);
        }
        if (!whole) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (row0 + 4 * j >= tokens) u[j] = v[j] = make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          store16(put[j & 1] + at + j * 512, u[j].x, u[j].y, u[j].z, u[j].w);
          store16((put[j & 1] + at + j * 512) ^ 16u, v[j].x, v[j].y, v[j].z, v[j].w);
        }
#pragma unroll
        for (int x = 0; x + 1 < kHeld; ++x)
#pragma unroll
          for (int j = 0; j < 2; ++j) held[x][j] = held[x + 1][j];
        scales.x = scales.y; scales.y = scales.z; scales.z = scales.w;
      } else if (p < kHeld) {
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
          uint4 u = held[0][x];
          if (!whole && row0 + 4 * (x & 1) >= tokens) u = make_uint4(0u, 0u, 0u, 0u);
          store16(put[x & 1] + at + (x >> 1) * kChunk + (x & 1) * 512, u.x, u.y, u.z, u.w);
          held[0][x] = held[1][x];
        }
      } else if (p == 2) {
        copy(4); copy(5);
        copies_commit();
        if (i > 0) wait(k, k.empty[3], (i - 1) & 1);
        copy(6); copy(7);
        copies_commit();
        copies_left<1>();
      } else {
        copies_left<0>();
      }
      if (careful) clean_pair(slots + 2 * p * kChunk, 4, first + sub, l, MX8 ? 0x7c00u : 0x7f80u, bad);
      fence_async();
      __syncwarp();
      if (lane == 0) arrive(k.full[p]);
    }
    copies_left<0>();
    if (careful) {
      clean_pair(slots + 8 * kChunk, 2, first + sub, l, 0x7f80u, bad);
      for (int j = 0; j < 2; ++j) {
        const int token = first + 4 * j + sub;
        if ((bad >> j) & 1u) atomicOr(&k.poison[i & 1][token >> 5], 1u << (token & 31));
      }
    }
    fence_async();
    __syncwarp();
    if (lane == 0) arrive(k.full[4]);
  }
}

// ---- MMA ------------------------------------------------------------------------------------------------------------------------------
template <bool MX8>
__device__ void issue_tiles(Control& k, unsigned q, unsigned p, unsigned slots) {
  const unsigned tmem = *(volatile unsigned*)&k.tmem, o = tmem, sc = tmem + kTmemS, sr = tmem + (MX8 ? kTmemR : kTmemS), tq = tmem + kTmemQ;
  unsigned dq = operand(q, 16), dk = operand(slots, 16), dp = operand(p, 16), dv = operand(slots, kChunk);
  unsigned lead;
  asm volatile("{.reg .pred e; elect.sync _|e, 0xffffffff; selp.u32 %0, 1, 0, e;}" : "=r"(lead));
  unsigned i = 0;
  for (unsigned n = 0;; ++n) {
    const Segment s = segment(k, n, true);
    if (s.t1 == 0) return;
    wait(k, k.q_full, n & 1);
    for (int t = s.t0; t < s.t1; ++t, ++i) {
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {                          // rolled, as everything that runs once a tile: unrolled code is waited for
        wait(k, k.full[c], i & 1);
        fence_after();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          mma_ws(lead, sc, dq + ((2 * c * kQChunk + (j >> 2) * kQChunk + (j & 3) * 32) >> 4), dk + ((2 * c * kChunk + (j >> 2) * kChunk + (j & 3) * 32) >> 4),
                 shape_of(!MX8, 0), c + j > 0);
      }
      wait(k, k.full[4], i & 1);
      fence_after();
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_ws_tmem(lead, sr, tq + j * 8, dk + ((8 * kChunk + j * 32) >> 4), shape_of(true, 0), !MX8 || j > 0);
      commit(lead, k.s_full);
#pragma unroll 1
      for (int u = 0; u < 4; ++u) {                          // 128 output columns each
        if (u == 0) { wait(k, k.p_full[0], i & 1); wait(k, k.p_full[1], i & 1); fence_after(); }
#pragma unroll
        for (int x = 0; x < 8; ++x)                          // 16 tokens each
          mma_ws(lead, o + u * 64, dp + (((x >> 2) * kQChunk + (x & 3) * 32) >> 4), dv + ((u * 2 * kChunk + x * 2048) >> 4), shape_of(!MX8, 1), t > s.t0 || x > 0);
        commit(lead, k.empty[u]);
      }
    }
  }
}

// ---- softmax ----------------------------------------------------------------------------------------------------------------------------
// Row r of a segment's tile: its address in q, or null where the tile has no such row.
__device__ __forceinline__ const __nv_bfloat16* query(const AttnArgs& a, const Segment& s, int r) {
  const int rows = (s.b < 0 ? a.B : 1) * a.S * a.heads, at = s.row0 + r;   // at most 2^27
  if (at >= rows) return nullptr;
  const int step = at / a.heads;
  return a.q + ((s.b < 0 ? 0 : s.b * a.S) + step) * a.q_stride + (at - step * a.heads) * kRow;
}
// The latent columns of a segment's queries on their way into shared memory, four threads to a row; zeros where the tile has no row.
__device__ __forceinline__ void fetch_q(const AttnArgs& a, const Segment& s, unsigned char* q, int tid) {
  const int r = tid >> 2;
  const unsigned char* src = reinterpret_cast<const unsigned char*>(query(a, s, r));
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int unit = 4 * i + (tid & 3);
    copy16(q + (unit >> 3) * kQChunk + unit_at(r, unit & 7), src ? src + unit * 16 : reinterpret_cast<const unsigned char*>(a.q), src != nullptr);
  }
  copies_commit();
}
// The rope columns into tensor memory, by the first four warps (every row on both halves of the lanes).
__device__ __forceinline__ void fetch_q_rope(const AttnArgs& a, const Segment& s, unsigned at, int r) {
  const __nv_bfloat16* src = query(a, s, r);
  unsigned v[32];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint4 x = src ? __ldg(reinterpret_cast<const uint4*>(src + kLatent) + i) : make_uint4(0u, 0u, 0u, 0u);
    v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
  }
  tmem_st32(at, v);
  tmem_wait_st();
}
// They have come: for MXFP8 pages made f16 where they lie, the row's largest element brought to 2^14 .. 2^15, each thread what it fetched.
template <bool MX8>
__device__ __forceinline__ void q_ready(Control& k, unsigned char* q, int tid) {
  copies_left<0>();
  if (MX8) {
    const int r = tid >> 2;
    unsigned top = 0;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const int unit = 4 * i + (tid & 3);
      const uint4 x = *reinterpret_cast<const uint4*>(q + (unit >> 3) * kQChunk + unit_at(r, unit & 7));
      top = max(top, absmax8(V8{{x.x, x.y, x.z, x.w}}));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = (int)(top >> 7);                           // exponent field of the largest element; 0: a row of zeros (or of subnormals), 255: not finite
    const int shift = e == 0 || e == 255 ? 0 : e - 127 - 14; // q' = q * 2^-shift
    const float up = __uint_as_float((unsigned)(127 - shift) << 23);
    if ((tid & 3) == 0) k.row_scale[r] = __uint_as_float((unsigned)(127 + shift) << 23);
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const int unit = 4 * i + (tid & 3);
      uint4* at = reinterpret_cast<uint4*>(q + (unit >> 3) * kQChunk + unit_at(r, unit & 7));
      const uint4 x = *at;
      auto half = [&](unsigned w) {
        const __half2 h = __floats2half2_rn(bf_lo(w) * up, bf_hi(w) * up);
        return *reinterpret_cast<const unsigned*>(&h);
      };
      *at = make_uint4(half(x.x), half(x.y), half(x.z), half(x.w));
    }
  }
  fence_async();
  fence_before();
  arrive(k.q_full);
}
// The four warps that share 32 rows.
__device__ __forceinline__ void softmax_barrier(int rows) {
  if (rows == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
  else asm volatile("bar.sync 2, 128;" ::: "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// Warp w: rows 32 (w % 2) .. of the tile, page w / 2 % 2 of each token tile, its tokens 32 (w / 4) ..; of O the columns on the same lanes, two accumulators of
// the four.
template <bool MX8>
__device__ void softmax_tiles(const AttnArgs& a, Control& k, unsigned char* q, unsigned char* p_mem, int tid) {
  const int r = tid & 63, half = (tid >> 6) & 1, part = tid >> 7, rows32 = (tid >> 5) & 1;
  const unsigned lanes = (unsigned)((tid >> 5) & 3) << 21;   // this warp's 32 lanes of tensor memory
  const unsigned tmem = *(volatile unsigned*)&k.tmem + lanes, o = tmem + part * 128, sc = tmem + kTmemS + part * 32, tq = tmem + kTmemQ;
  unsigned char* p_row = p_mem + half * kQChunk;
  Segment s = segment(k, 0, false);
  if (s.t1 == 0) return;
  fetch_q(a, s, q, tid);
  if (part == 0) fetch_q_rope(a, s, tq, r);
  q_ready<MX8>(k, q, tid);
  unsigned i = 0;
  for (unsigned n = 0;; ++n) {
    s = segment(k, n, true);
    if (s.t1 == 0) return;
    int seen = s.tokens;                                     // tokens that the row sees
    if (s.b >= 0) seen = s.tokens - (a.S - 1 - min((s.row0 + r) / a.heads, a.S - 1));
    float row_scale = 1.f, m = -INFINITY, l = 0.f;                            // the maximum that P and O are relative to, and this thread's share of the sum
    for (int t = s.t0; t < s.t1; ++t, ++i) {
      const int base = t * kTile + half * 64;
      int live = min(32, max(0, seen - base - part * 32));   // visible ones of this thread's 32 tokens
      if (live > 0) {
        const int id = __ldg(s.table + (base >> 6));
        if (id < 0 || id >= a.pages) live = 0;
      }
      wait(k, k.s_full, i & 1);
      fence_after();
      unsigned raw[32];
      tmem_ld32(sc, raw);
      int ex[4] = {0, 0, 0, 0};                              // E of the thread's four runs of 8 tokens
      if (MX8) {
        unsigned rope[32];
        tmem_ld32(sc + (kTmemR - kTmemS), rope);
        if (t == s.t0) row_scale = *(volatile float*)&k.row_scale[r];
        tmem_wait_ld();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          ex[g] = *(volatile int*)&k.exponent[i & 1][half * 8 + part * 4 + g];
          const f32x2 f = f2_splat(row_scale * __uint_as_float((unsigned)(ex[g] + 127) << 23));
#pragma unroll
          for (int j = 8 * g; j < 8 * g + 8; j += 2) {
            float u, v;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(raw[j]), __uint_as_float(raw[j + 1])), f, f2_pack(__uint_as_float(rope[j]), __uint_as_float(rope[j + 1]))), u, v);
            raw[j] = __float_as_uint(u); raw[j + 1] = __float_as_uint(v);
          }
        }
      } else {
        tmem_wait_ld();
      }
      // the maximum of the visible scores, and a sum that turns NaN where one is not finite
      if (a.flip) {
#pragma unroll
        for (int j = 0; j < 32; ++j) raw[j] ^= 0x80000000u;
      }
      const bool whole = __all_sync(0xffffffffu, live == 32);
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 32; ++j) raw[j] = j < live ? raw[j] : 0u;
      }
      f32x2 odd2[2] = {f2_splat(0.f), f2_splat(0.f)};
#pragma unroll
      for (int j = 0; j < 16; ++j) odd2[j & 1] = f2_fma(f2_pack(__uint_as_float(raw[2 * j]), __uint_as_float(raw[2 * j + 1])), f2_splat(0.f), odd2[j & 1]);
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 32; ++j) raw[j] = j < live ? raw[j] : 0xff800000u;
      }
      float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 16; ++j) tops[j >> 2] = max3(tops[j >> 2], __uint_as_float(raw[2 * j]), __uint_as_float(raw[2 * j + 1]));
      float odd, odd1, top = fmaxf(fmaxf(fmaf(tops[0], a.c, (float)ex[0]), fmaf(tops[1], a.c, (float)ex[1])), fmaxf(fmaf(tops[2], a.c, (float)ex[2]), fmaf(tops[3], a.c, (float)ex[3])));
      f2_unpack(f2_add(odd2[0], odd2[1]), odd, odd1);
      odd += odd1;
      const unsigned mine = *(volatile unsigned*)&k.poison[i & 1][2 * half + part];
      if (mine && live > 0 && (mine & (~0u >> (32 - live)))) odd = NAN;
      l += odd;
      k.best[2 * part + half][r] = top;
      softmax_barrier(rows32);
      top = fmaxf(fmaxf(k.best[0][r], k.best[1][r]), fmaxf(k.best[2][r], k.best[3][r]));
      if (t == s.t0) m = top;
      else if (__any_sync(0xffffffffu, top > m + kLag)) {    // O of these 32 rows catches up with the maximum
        const float best = fmaxf(m, top), f = best == -INFINITY ? 1.f : exp2_fast(m - best);
        l *= f;
        m = best;
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          unsigned v[32];
          tmem_ld32(o + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * f);
          tmem_st32(o + c, v);
        }
        tmem_wait_st();
      }
      const float off = kTop - (m == -INFINITY ? 0.f : m);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x2 off2 = f2_splat(off + (float)ex[g]);
        f32x2 sum2[2] = {f2_splat(0.f), f2_splat(0.f)};
        unsigned pw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float e0, e1;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(raw[8 * g + 2 * j]), __uint_as_float(raw[8 * g + 2 * j + 1])), f2_splat(a.c), off2), e0, e1);
          e0 = exp2_fast(e0);
          e1 = exp2_fast(e1);
          sum2[j & 1] = f2_add(sum2[j & 1], f2_pack(e0, e1));
          if (MX8) {
            const __half2 h = __floats2half2_rn(e0, e1);
            pw[j] = *reinterpret_cast<const unsigned*>(&h);
          } else {
            pw[j] = pack_bf2(e0, e1);
          }
        }
        *reinterpret_cast<uint4*>(p_row + unit_at(r, part * 4 + g)) = make_uint4(pw[0], pw[1], pw[2], pw[3]);
        float s0, s1;
        f2_unpack(f2_add(sum2[0], sum2[1]), s0, s1);
        l = fmaf(s0 + s1, __uint_as_float((unsigned)(127 - ex[g]) << 23), l);   // a token's weight itself, without its 2^E
      }
      fence_async();
      fence_before();
      arrive(k.p_full[part]);
    }
    // the last product with this segment's queries is done: the next segment's take their place while P V goes on
    const Segment next = segment(k, n + 1, false);
    if (next.t1 > 0) {
      fetch_q(a, next, q, tid);
      if (part == 0) fetch_q_rope(a, next, tq, r);
    }
    // this stretch's unnormalised outputs, maximum and sum
    wait(k, k.empty[3], (i - 1) & 1);
    fence_after();
    const bool live_row = query(a, s, r) != nullptr;
    const long long at = (long long)blockIdx.x + s.tile;
    k.best[2 * part + half][r] = l;
    softmax_barrier(rows32);
    if (half + part == 0 && live_row) a.sums[at * kRows + r] = make_float2(m, (k.best[0][r] + k.best[1][r]) + (k.best[2][r] + k.best[3][r]));
    float* dst = a.parts + at * kPartFloats + r * kLatent + part * 256 + half * 64;
#pragma unroll 1
    for (int c = 0; c < 128; c += 32) {
      unsigned v[32];
      tmem_ld32(o + c, v);
      tmem_wait_ld();
      if (live_row) {
        float* d = dst + (c >> 6) * 128 + (c & 63);
#pragma unroll
        for (int j = 0; j < 32; j += 8)
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" :: "l"(d + j), K3G_I8(v, j) : "memory");
      }
    }
    if (next.t1 > 0) q_ready<MX8>(k, q, tid);                // the next segment's first product overwrites O: after these loads
  }
}

// ---- planning ---------------------------------------------------------------------------------------------------------------------------
// The CTA's segments into the ring, and for the join the first and the last CTA of each row tile.
__device__ void plan(const AttnArgs& a, Control& k, int ptok, int lane) {
  long long left = k.left;
  int tile = k.first_tile, at = k.first_at;
  for (unsigned n = 0;; ++n) {
    Segment s = {0, -1, 0, 0, 0, 0, nullptr};
    while (left > 0) {
      s.b = -1; s.row0 = tile * kRows; s.tokens = ptok; s.table = a.prefix_table;
      if (tile >= a.prefix_tiles) {
        s.b = (tile - a.prefix_tiles) / a.seq_tiles;
        s.row0 = (tile - a.prefix_tiles - s.b * a.seq_tiles) * kRows;
        s.tokens = s.b < a.B ? own_tokens(a, s.b) : 0;
        s.table = a.block_table + (long long)s.b * a.max_pages;
        if (s.b >= a.B) break;
      }
      s.tile = tile;
      const int places = places_of(s.tokens), to = (int)min((long long)places, at + left);
      s.t0 = max(0, at - kStart);
      s.t1 = max(0, to - kStart);
      left -= to - at;
      at = to;
      if (to == places) { tile = places == 0 && s.b >= 0 ? a.prefix_tiles + (s.b + 1) * a.seq_tiles : tile + 1; at = 0; }
      if (s.t1 > s.t0) {
        if (lane == 0 && s.t0 == 0) a.spans[s.tile].x = blockIdx.x;
        if (lane == 0 && s.t1 == places - kStart) a.spans[s.tile].y = blockIdx.x;
        break;
      }
      s.t1 = 0;
    }
    if (n >= kRing) wait(k, k.ring_empty[n % kRing], (n / kRing - 1) & 1);
    if (lane == 0) {
      k.ring[n % kRing] = s;
      arrive(k.ring_full[n % kRing]);
    }
    __syncwarp();
    if (s.t1 == 0) return;
  }
}

template <bool MX8>
__global__ void __launch_bounds__(kThreads, 1) latent_attn_kernel(const __grid_constant__ AttnArgs a) {
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<unsigned long long>(raw) + 1023) & ~1023ull);
  __shared__ Control k;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // the line: places of sequences b0 .. b1 by this thread, then a scan over the block
  const int ptok = prefix_tokens(a);
  const long long prefix_places = (long long)a.prefix_tiles * places_of(ptok);
  const int per = (a.B + kThreads - 1) / kThreads, b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  long long mine = 0;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) mine += a.seq_tiles * places_of(own_tokens(a, b));
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) k.scan[warp] = upto;
  if (tid == 0) {
    auto init = [](unsigned long long& bar, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(su(&bar)), "r"(n)); };
#pragma unroll 1
    for (int c = 0; c < 5; ++c) init(k.full[c], kLoaders / 32);
#pragma unroll 1
    for (int u = 0; u < 4; ++u) { init(k.empty[u], 1); init(k.ring_full[u], 1); init(k.ring_empty[u], kReaders); }
    init(k.p_full[0], kSoftmax / 2); init(k.p_full[1], kSoftmax / 2);
    init(k.q_full, kSoftmax); init(k.s_full, 1);
    k.abort = 0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) k.poison[i >> 2][i & 3] = 0;
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(su(&k.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_async();
  fence_before();
  __syncthreads();
  fence_after();
  long long before = prefix_places, total = prefix_places;
#pragma unroll 1
  for (int i = 0; i < kThreads / 32; ++i) { const long long v = k.scan[i]; if (i < warp) before += v; total += v; }
  before += upto - mine;
  const int ctas = (int)min((long long)gridDim.x, total);    // those with work: CTA i takes places total * i / ctas ..
  const bool busy = (int)blockIdx.x < ctas;
  if (busy) {
    const long long lo = total * blockIdx.x / ctas;
    if (tid == 0) {
      k.left = total * (blockIdx.x + 1ll) / ctas - lo;
      if (lo < prefix_places) { k.first_tile = (int)(lo / places_of(ptok)); k.first_at = (int)(lo % places_of(ptok)); }
    }
#pragma unroll 1
    for (int b = b0; b < b1 && before <= lo; ++b) {
      const int n = places_of(own_tokens(a, b));
      const long long in = lo - before;
      before += a.seq_tiles * n;
      if (before > lo) {                                     // fewer than 2^34 places to a sequence
        k.first_tile = a.prefix_tiles + b * a.seq_tiles + (int)(in / n);
        k.first_at = (int)(in % n);
      }
    }
  }
  __syncthreads();
  if (busy) {
    unsigned char *q = smem, *p = q + kSmemQ, *slots = p + kSmemP;
    if (warp < kSoftmax / 32) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
      softmax_tiles<MX8>(a, k, q, p, tid);
    } else if (warp < (kSoftmax + kLoaders) / 32) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
      load_tiles<MX8>(a, k, slots, tid - kSoftmax);
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
      if (warp == (kSoftmax + kLoaders) / 32) issue_tiles<MX8>(k, su(q), su(p), su(slots));
      else if (warp == (kSoftmax + kLoaders) / 32 + 1) plan(a, k, ptok, lane);
    }
  }
  fence_before();
  __syncthreads();
  if (tid == 0) a.status[blockIdx.x] = k.abort;
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(k.tmem) : "memory");
}

// ---- joining the parts of each row ------------------------------------------------------------------------------------------------------
// GROUPS warps a row, two rows a block or one: lane j of a warp owns columns 128 x + 4 j .. + 3 (x = 0..3), warp g takes every GROUPS-th part.  Parts are
// weighed by 2^(m - max m); the order of the sums depends on the lengths alone.
constexpr int kJoinWarps = 8;
template <int GROUPS>
__global__ void __launch_bounds__(32 * kJoinWarps) latent_attn_join_kernel(const __grid_constant__ AttnArgs a, int ctas, int rows) {
  __shared__ float4 s_out[GROUPS > 1 ? kJoinWarps : 1][128];
  __shared__ float s_l[kJoinWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = warp % GROUPS;
  const int row = blockIdx.x * (kJoinWarps / GROUPS) + warp / GROUPS;
  const bool there = row < rows;
  const int per_seq = a.S * a.heads, b = there ? row / per_seq : 0, in_seq = row - b * per_seq;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int gave_up = 0;
  for (int i = tid; i < ctas; i += 32 * kJoinWarps) gave_up |= a.status[i];
  const int len = __ldg(a.lens + b), ptok = prefix_tokens(a), own = own_tokens(a, b);
  const bool live = there && len >= 0;
  float4 acc[4] = {};
  float l = 0.f;
  if (live) {
    // the parts: those of the row's tile against the prefix, then those against its own tokens; part (CTA, tile) has index CTA + tile
    const int ptile = row / kRows, otile = a.prefix_tiles + b * a.seq_tiles + in_seq / kRows;
    const int2 ps = ptok ? a.spans[ptile] : make_int2(0, -1), os = own ? a.spans[otile] : make_int2(0, -1);
    const int np = ps.y + 1 - ps.x, parts = np + os.y + 1 - os.x;
    auto slot = [&](int i) { return i < np ? (long long)(ps.x + i + ptile) * kRows + row % kRows : (long long)(os.x + (i - np) + otile) * kRows + in_seq % kRows; };
    float best = -INFINITY;
    for (int i = lane; i < parts; i += 32) best = fmaxf(best, a.sums[slot(i)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    const float off = best == -INFINITY ? 0.f : best;
#pragma unroll 2
    for (int i = g; i < parts; i += GROUPS) {
      const long long at = slot(i);
      const float2 ml = a.sums[at];
      float4 v[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) v[x] = __ldcs(reinterpret_cast<const float4*>(a.parts + at * kLatent) + 32 * x + lane);
      const float f = exp2f(ml.x - off);
      l = fmaf(ml.y, f, l);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        acc[x].x = fmaf(v[x].x, f, acc[x].x); acc[x].y = fmaf(v[x].y, f, acc[x].y);
        acc[x].z = fmaf(v[x].z, f, acc[x].z); acc[x].w = fmaf(v[x].w, f, acc[x].w);
      }
    }
  }
  if (GROUPS > 1) {
#pragma unroll
    for (int x = 0; x < 4; ++x) s_out[warp][32 * x + lane] = acc[x];
    if (lane == 0) s_l[warp] = l;
  }
  const bool failed = __syncthreads_or(gave_up);
  if (!live || g > 0) return;                                // no sequence: left as it was
  if (GROUPS > 1) {
    for (int i = 1; i < GROUPS; ++i) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float4 v = s_out[warp + i][32 * x + lane];
        acc[x].x += v.x; acc[x].y += v.y; acc[x].z += v.z; acc[x].w += v.w;
      }
      l += s_l[warp + i];
    }
  }
  // a sum of exactly 0 has seen no token; NaN stays NaN; a call whose kernel gave up a wait has no result
  const float f = failed || l != l ? NAN : l == 0.f ? 0.f : __frcp_rn(l);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    uint2 w = make_uint2(pack_bf2(acc[x].x * f, acc[x].y * f), pack_bf2(acc[x].z * f, acc[x].w * f));
    if (l == 0.f && !failed) w = make_uint2(0u, 0u);
    *reinterpret_cast<uint2*>(a.out + (long long)row * kLatent + 128 * x + 4 * lane) = w;
  }
}

// Workspace: status words, spans, (maximum, sum) pairs, parts; the parts of CTA i and row tile t have index i + t.
struct Space { long long spans, sums, parts, bytes; };
Space space_of(int B, int S, int heads) {
  const long long tiles = ((long long)B * S * heads + kRows - 1) / kRows + (long long)B * (((long long)S * heads + kRows - 1) / kRows);
  const long long parts = tiles + kMaxCtas;
  auto up = [](long long x) { return (x + 255) / 256 * 256; };
  Space s;
  s.spans = up(kMaxCtas * 4);
  s.sums = s.spans + up(tiles * 8);
  s.parts = s.sums + up(parts * kRows * 8);
  s.bytes = s.parts + parts * kPartFloats * 4;
  return s;
}

template <int GROUPS>
cudaError_t launch_join(const AttnArgs& a, int ctas, int rows, cudaStream_t stream) {
  constexpr int per = kJoinWarps / GROUPS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((rows - 1) / per + 1), 1, 1); cfg.blockDim = dim3(32 * kJoinWarps, 1, 1); cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, latent_attn_join_kernel<GROUPS>, a, ctas, rows);
}

}  // namespace

K3G_API int k3g_latent_attn_workspace(int B, int S, int heads, long long* host_bytes) {
  K3G_REQUIRE_PTR(host_bytes);
  K3G_REQUIRE(B > 0 && S > 0 && heads > 0, K3G_ESHAPE);
  K3G_REQUIRE(B <= kMaxBatch && (long long)S * heads <= kMaxRowsPerSeq, K3G_ELIMIT);
  *host_bytes = space_of(B, S, heads).bytes;
  return K3G_OK;
}

K3G_API int k3g_latent_attn(const void* q, long long q_stride, const void* cache, int cache_mx8, long long layer_off, long long page_stride,
                            long long pages, const void* prefix_table, const void* prefix_len, int prefix_pages, const void* block_table,
                            const void* lens, int max_pages, void* out, void* workspace, long long workspace_bytes, int B, int S, int heads,
                            float scale, void* stream) {
  K3G_REQUIRE_PTR(q); K3G_REQUIRE_PTR(cache); K3G_REQUIRE_PTR(lens); K3G_REQUIRE_PTR(out); K3G_REQUIRE_PTR(workspace);
  K3G_REQUIRE_ALIGNED(q); K3G_REQUIRE_ALIGNED(cache); K3G_REQUIRE_ALIGNED(out); K3G_REQUIRE_ALIGNED(workspace);
  K3G_REQUIRE(B >= 0 && prefix_pages >= 0 && max_pages >= 0 && pages >= 0 && pages < (1ll << 31), K3G_ESHAPE);
  if (B == 0) return K3G_OK;
  if (prefix_pages > 0) { K3G_REQUIRE_PTR(prefix_table); K3G_REQUIRE_PTR(prefix_len); }
  if (max_pages > 0) K3G_REQUIRE_PTR(block_table);
  const long long unit = cache_mx8 ? 1 : 2, page = cache_mx8 ? kMx8Page : 2 * kBf16Page;
  K3G_REQUIRE(q_stride % 8 == 0 && layer_off * unit % 16 == 0 && page_stride * unit % 16 == 0, K3G_EALIGN);
  K3G_REQUIRE(S > 0 && heads > 0 && q_stride >= (long long)heads * kRow && layer_off >= 0 && page_stride * unit >= layer_off * unit + page, K3G_ESHAPE);
  K3G_REQUIRE(B <= kMaxBatch && (long long)S * heads <= kMaxRowsPerSeq && prefix_pages <= (1 << 20) && max_pages <= (1 << 20), K3G_ELIMIT);
  const Space sp = space_of(B, S, heads);
  K3G_REQUIRE(workspace_bytes >= sp.bytes, K3G_EWORKSPACE);
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  auto kernel = cache_mx8 ? latent_attn_kernel<true> : latent_attn_kernel<false>;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  unsigned char* ws = (unsigned char*)workspace;
  const long long rows = (long long)B * S * heads;
  const int ctas = sms < kMaxCtas ? sms : kMaxCtas;
  AttnArgs a = {(const __nv_bfloat16*)q, q_stride, (const unsigned char*)cache + layer_off * unit, page_stride * unit, pages,
                (const int*)prefix_table, (const int*)prefix_len, prefix_pages, (const int*)block_table, (const int*)lens, max_pages,
                (__nv_bfloat16*)out, (int*)ws, (int2*)(ws + sp.spans), (float2*)(ws + sp.sums), (float*)(ws + sp.parts),
                B, S, heads, (int)((rows + kRows - 1) / kRows), (S * heads + kRows - 1) / kRows, ctas, fmaxf(fabsf(scale) * 1.44269504088896341f, 1e-30f), scale < 0.f};
  kernel<<<ctas, kThreads, kSmem, k3g_stream(stream)>>>(a);
  const int rc = k3g_launch_status();
  if (rc != K3G_OK) return rc;
  // Few rows mean many parts for each: several warps share them (a card's 148 SMs hold about 1200 such warps at once and more).
  const int n = (int)rows;
  e = n <= 148 ? launch_join<8>(a, ctas, n, k3g_stream(stream)) : n <= 1184 ? launch_join<4>(a, ctas, n, k3g_stream(stream)) : launch_join<1>(a, ctas, n, k3g_stream(stream));
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  return k3g_launch_status();
}
