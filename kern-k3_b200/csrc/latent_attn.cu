// Attention of a batch over the paged latent cache, the prefix that the batch shares read once for all of it.
//
// out[b, s, h] = sum_j p_j k_j[0:512], p = softmax_j(scale * q[b, s, h] . k_j), j over the tokens that step s of sequence b sees:
// the shared prefix, and its own tokens up to the one of step s (the last S of its own tokens are the S steps).  A latent row is
// key (576 columns) and value (its first 512) at once, so a tile of tokens is loaded once and used by two products.
//
// Work.  All rows (b, s, h) in tiles of 64 against the prefix, and each sequence's rows in tiles of 64 against its own
// tokens, in tiles of 128 tokens (two pages).  Every (row tile, token tile) pair costs the same, 3.5 us, and a row tile about as much again
// (its queries in, its outputs out): the pairs are laid in one line, row tile by row tile, kStart empty places before each, and each CTA takes an equal
// stretch, whatever the lengths are.  A stretch that covers a part of a row tile leaves an unnormalised f32 output with its maximum and sum in the
// workspace (one pass over the tokens, running maximum and sum in 32 bits), and a second, dependent launch joins the parts of each row.
// Lengths and tables are read on the device: a captured graph follows them.  Nothing is accumulated by atomics: the same inputs give the same bits.
//
// One CTA per SM, warps with fixed roles, one token tile after another:
//   1 planning warp  this CTA's stretches, one after another, and the pages of their tiles, into rings that the others read;
//   8 loader warps   fetch the next tile into registers and make 16-bit floats of it in 128-byte-swizzled shared memory, nine 16 KB chunks of 64
//                    columns;
//   1 MMA warp       S = Q K^T (64 x 128, two chunks at a time as they come) and O += P V (64 x 512 in tensor memory), both tcgen05.mma.ws, M = 64;
//   8 softmax warps  S from tensor memory, running maximum, P = 2^(S - m) rounded to 16 bits into shared memory; O scaled, read and written out.
// Why M = 64: a 128-row O of 512 columns fills the whole tensor memory and leaves no room for S.  The weight-stationary form puts
// a 64-row tile on all 128 lanes and reaches 48 cycles per 64 x 128 x 16 step, the plain form 64 (measured; 32 would be full rate).
// Why 128 tokens: a 64 x 64 x 16 step costs 44 cycles.  Tiles of one page in two buffers, which let all roles work at once, took 425 us where this took
// 340.  O is made in four products of 128 columns: a pair of chunks is refilled as soon as its quarter of P V is done.
// The queries' rope columns lie in tensor memory, which makes room for P.
//
// What bounds it.  By the formulas the cache's bytes with few rows, the tensor cores with many (640 flops a byte for 64 rows).  A pair takes
// 6300 cycles, in two phases that one buffer of 128 tokens keeps apart.  From P to S, 4400: the products, 68 steps of 64 x 128 x 16 that read 6 KB
// of shared memory each, which is their 48 cycles (3300 in all; at full rate they would be 32, and ncu counts those: 2170 a pair, 31% of the time), and
// the loaders' conversions and stores between them.  From S to P, 1900: S out of tensor memory, maximum, vote, exponentials.  What the loaders wait for
// counts: conversions between the stores, polls ahead of the waits and the next tile's place read last brought 321 us down to 298 (for the long document
// below, before blocks and tokens of zeros were looked for, which costs 2%).  No gain came from more loader warps (16 instead of 8: 346
// us instead of 321), from P V in products of 256 columns, which read less but free the chunks later (349 instead of 339), from one
// accumulator for latent and rope columns (315 instead of 309), or from the rope columns' product before the last pair of chunks (308
// instead of 303).  A call's start, the parts' way out and the join take 17 us beside the pairs.
// Measured: 8 x 96 rows against 131072 MXFP8 tokens 305 us (319 in a long run with other inputs every time: 686 TFLOP/s, 42% of a dense bf16
// product), 48 x 4 x 24 rows against 16384 and their own 512 252 us, 32 x 24 rows against 8229 and 1024 43 us, 64 x 12 rows against
// their own 4096 42 us (2.1 TB/s), 16 x 2 x 48 rows against bf16 pages 48 us (53 with the next tile asked for before this one was copied), one sequence of 500 tokens 12.5 us.
//
// Types.  bf16 pages are multiplied as bf16.  MXFP8 codes become f16, not bf16: one conversion and one product for two codes, a third of what bf16
// takes (which has no conversion from E4M3), and the loaders' instructions are what a tile waits for.  f16 has the bits (a code has four), but not the
// range, so exponents are taken out: of the scales of 16 tokens (but those of blocks of zeros) the largest less kRoom, E (K' = code * 2^(e - E): blocks whose
// scale is 2^-32 of the largest become 0, others keep what is above 2^-24 of 2^E, 2^-39 of the largest element; 16 tokens that are all zeros do not move
// m, and their weights are summed relative to their own maximum), of a query row its own (the largest element
// is brought to 2^14..2^15; what that costs is below 2^-39 of it).  They come back in f32: S = 2^(E + row) S' + S_rope
// (the rope columns are multiplied as bf16 into a second accumulator), and P' = 2^(S + E - m), with m the running maximum of S + E, so
// that P' V' has the weight of P V.  P is rounded because both operands of the matrix instructions are 16 bits; the sums of P stay unrounded in f32.
// The m that P' is relative to follows the true maximum only when it falls behind by more than 2^4 (O is then rescaled): the ratio is
// exact either way.  P' is kept in 2^-24 .. 2^14, with 2^10 at the maximum: tokens whose weight times 2^E is below 2^-34 of the largest such product are lost.
#include <cuda_runtime.h>

#include "latent_page.cuh"
#include "k3g_host.h"

using namespace k3g;

namespace {

constexpr int kMaxBatch = 4096, kMaxRowsPerSeq = 1 << 15, kMaxCtas = 160;
constexpr int kRows = 64, kTile = 2 * kPageTokens;           // query rows and tokens of a tile
constexpr int kSoftmax = 256, kLoaders = 256, kThreads = kSoftmax + kLoaders + 128;   // the last four warps: MMAs, planning, two idle
constexpr int kChunk = kTile * 128, kQChunk = kRows * 128;   // 64 columns of a tile's tokens, of its rows, at 16 bits
constexpr int kSmemQ = 8 * kQChunk, kSmemP = 2 * kQChunk, kSmemK = 9 * kChunk, kSmem = kSmemQ + kSmemP + kSmemK + 1024;
// tensor memory columns: O 0..255 (four accumulators of 128 output columns, 64 on either half of the lanes), S 256..319 (a page on either
// half), the rope columns' part of S 320..383 (MXFP8), the queries' rope columns 384..415 (the same on both halves)
constexpr int kTmemS = 256, kTmemR = 320, kTmemQ = 384;
constexpr int kRoom = 7;                                     // E is the largest scale's exponent less this: codes reach 448 = 2^8.8, f16 2^16
constexpr int kLeastE = -80, kMostE = 120;                   // sums of 2^-E stay in range
constexpr int kZeros = kLeastE - 1;                          // 16 tokens that are all zeros: as if their E was the least, and each row's sum finds its own
constexpr float kLag = 4.f, kTop = 10.f;                     // the long document above 340 us when it was chosen, with a lag of 0 (O rescaled for every new maximum) 359
constexpr int kPartFloats = kRows * kLatent;                 // a part's outputs; its 64 (maximum, sum) pairs lie in a table of their own
constexpr int kWaitLimit = 1 << 20, kRing = 4, kReaders = kSoftmax / 32 + 1, kTiles = 2;
constexpr int kStart = 2;                                     // the drafted tokens above 276 us when it was chosen, with 1 336, with 4 283

struct AttnArgs {
  const __nv_bfloat16* q; long long q_stride;
  const unsigned char* cache; long long page_stride, pages;       // bytes
  const int* prefix_table; const int* prefix_len; int prefix_pages;
  const int* block_table; const int* lens; int max_pages;
  __nv_bfloat16* out;
  int* status;                       // [kMaxCtas] 1: a wait of this CTA expired
  int2* spans;                       // [row tiles] first and last CTA of each (unwritten where there are no tokens)
  float2* sums;                      // [parts][64] (maximum in log2 units, sum)
  float* parts;                      // [parts][64 groups of 8 columns][64 rows][8]: what a warp writes at a time lies together
  int B, S, heads, prefix_tiles, seq_tiles;
  float c;                           // |scale| * log2(e), above 0 (scores are compared before they are scaled)
  int flip;                          // the scale is negative
};

__device__ __forceinline__ unsigned su(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }

// ---- lengths and the line of (row tile, token tile) pairs ------------------------------------------------------------------
__device__ __forceinline__ int tokens_of(int len, int pages) { return max(0, min(len, pages * kPageTokens)); }   // pages: 2^20 at most
__device__ __forceinline__ int prefix_tokens(const AttnArgs& a) { return a.prefix_pages ? tokens_of(ld_ordered(a.prefix_len), a.prefix_pages) : 0; }
__device__ __forceinline__ int own_tokens(const AttnArgs& a, int b) { return tokens_of(ld_ordered(a.lens + b), a.max_pages); }
__device__ __forceinline__ int tiles_of(int tokens) { return (tokens + kTile - 1) / kTile; }
__device__ __forceinline__ int places_of(int tokens) { return tokens ? tiles_of(tokens) + kStart : 0; }   // on the line
struct Segment {                     // one CTA's stretch of one row tile
  int tile;                          // row tile: prefix_tiles of them against the prefix, then seq_tiles for each sequence
  int b;                             // sequence, or -1 for the prefix
  int row0;                          // first row: of all rows (prefix) or of the sequence's rows
  int t0, t1;                        // token tiles (none: the end)
  int tokens;                        // tokens of the prefix / of the sequence
};
struct Tile {                        // where a tile's pages are
  const unsigned char* page[2];
  int tokens[2];                     // of each (none of a page that the cache does not hold)
  int live, careful;                 // 0: the end; steps of a sequence do not all see all of its tokens
};

// ---- barriers and tensor memory -----------------------------------------------------------------------------------------------
struct Control {
  unsigned long long full[5], empty[4], q_full[4], s_full, s_read, p_full, o_free, drained;
  unsigned long long ring_full[kRing], ring_empty[kRing], tile_full[kTiles], tile_empty[kTiles];
  Tile tile[kTiles];
  Segment ring[kRing];
  unsigned tmem;
  int abort;
  int first_tile, first_at;
  long long left;
  unsigned poison[2][4];                                      // tokens of a tile with values that are not finite (tiles by turns)
  int exponent[8], tokens[2];                                // of a tile: E of each 16 tokens, and how many there are in either page
  signed char row_shift[2][kRows];                            // the power of two that was taken out of a query row, segments by turns
  union {
    float best[4][kRows];                                     // the maxima of a page, and at a segment's end the sums
    long long scan[kThreads / 32];                            // before the first
  };
};

// Every wait ends: after kWaitLimit polls, or as soon as another wait of the CTA has expired.  The roles then run through what is
// left without waiting (every access stays where it was: the rings hold end marks before the plan's first entries, and a mixed one of two entries
// names rows and pages of either), the products on their way are waited for before tensor memory is given back, and the call's result is NaN.
__device__ __forceinline__ void wait(Control& k, unsigned long long& bar, unsigned parity, unsigned nap = 0) {
  unsigned ok;
  asm volatile("{.reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}" : "=r"(ok) : "r"(su(&bar)), "r"(parity) : "memory");
  if (ok) return;
#pragma unroll 1
  for (int i = 0; i < kWaitLimit; ++i) {
    asm volatile("{.reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}" : "=r"(ok) : "r"(su(&bar)), "r"(parity) : "memory");
    if (ok) return;
    if (*(volatile int*)&k.abort) return;
    if (nap) __nanosleep(nap);
  }
  *(volatile int*)&k.abort = 1;
}
// The first poll of a wait, for a warp that has something to do until it needs the answer.
__device__ __forceinline__ unsigned poll(unsigned long long& bar, unsigned parity) {
  unsigned ok;
  asm volatile("{.reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}" : "=r"(ok) : "r"(su(&bar)), "r"(parity) : "memory");
  return ok;
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
// Warp w looks after tokens 16 w .. + 15 of a tile, a lane after two of them, 8 apart, and of each pair of chunks after 32 columns: one scale
// block.  Eight lanes that load together read 64 bytes of four tokens each, and store to all banks: two units of four tokens, swizzled.  (32 bytes
// of eight tokens: 336 us for the long document above instead of 321; 128 bytes of two, for which half of the lanes turn their words round: 320.)
__device__ __forceinline__ unsigned clean(unsigned w, unsigned top, unsigned& bad) {   // a pair of 16-bit floats with NaN and infinities taken out
  if ((w & top) == top) { w &= 0xffff0000u; bad = 1; }
  if ((w & (top << 16)) == (top << 16)) { w &= 0x0000ffffu; bad = 1; }
  return w;
}
// 16-byte unit u (8 columns) of a token's row in a chunk, swizzled
__device__ __forceinline__ int unit_at(int token, int u) { return token * 128 + ((u ^ (token & 7)) << 4); }
// Shared memory is addressed by 32-bit numbers here: the compiler does not see the address space behind the aligned base pointer.
__device__ __forceinline__ void copy16(unsigned dst, const unsigned char* src, bool live) {   // zeros where there is no row
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void store16(unsigned at, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 load16(unsigned at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_left() { asm volatile("cp.async.wait_group %0;" :: "n"(LEFT) : "memory"); }

// 2^(byte - base) as a pair of f16 (byte 255: NaN), and four E4M3 codes times it.  Scales are 2^kRoom times the base at most, and 448 * 2^kRoom is below f16's
// largest; from 2^-24 up the factor is one of f16's, and the product is exact but for what falls below 2^-24.  A block of zeros may have any byte: a
// factor that f16 does not hold is cut to its largest.
__device__ __forceinline__ unsigned f16_scale(unsigned base, unsigned byte) {
  unsigned h;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %1;" : "=r"(h) : "f"(__uint_as_float((unsigned)max((int)(byte + 127 - base), 0) << 23)));
  return byte == 255 ? 0x7e007e00u : h;
}
__device__ __forceinline__ void mx8_to_f16x4(unsigned codes, unsigned scale, unsigned& lo, unsigned& hi) {
  asm("{.reg .b16 a, b; .reg .b32 x, y; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 x, a; cvt.rn.f16x2.e4m3x2 y, b; mul.rn.f16x2 %0, x, %3; mul.rn.f16x2 %1, y, %3;}"
      : "=r"(lo), "=r"(hi) : "r"(codes), "r"(scale));
}

// What the lane has just written of chunk units, without its NaN and infinities (rare: a rolled loop, out of the way).
__device__ __forceinline__ void clean_units(unsigned chunk, int token, int unit, int units, unsigned top, unsigned& bad) {
#pragma unroll 1
  for (int x = unit; x < unit + units; ++x) {
    const unsigned at = chunk + unit_at(token, x);
    const uint4 v = load16(at);
    store16(at, make_uint4(clean(v.x, top, bad), clean(v.y, top, bad), clean(v.z, top, bad), clean(v.w, top, bad)));
  }
}

// Chunks are handed over in pairs (0 1, 2 3, 4 5, 6 7, and the rope chunk), a fence and an arrival for each; a pair's slots are free as soon as
// its 128 columns of P V are done, the rope slot before that.  The next tile's codes are fetched into registers when this one has been
// handed over (any earlier and a warp, which has few scoreboards, would wait for new data with the old), in portions: what a tile's loads
// move (80 KB, 64 bytes a clock) would else be in the way of the softmax warps' reads of S and stores of P.
template <bool MX8>
struct Loader {
  const AttnArgs& a;
  Control& k;
  unsigned slots, put_at[4];                                 // the thread's units of its first token's first pair of chunks; the other token's are 1024 bytes on
  int tid, lane, token, block;
  // a tile on its way: MXFP8, 32 codes of each pair of chunks, the scale bytes; bf16, 32 columns of two pairs; of two tokens each
  V16 code[4][2];
  V8 scales[2];
  struct Where {
    const unsigned char* page;
    int tokens;
    bool careful, live;
  } here, next;
  __device__ __forceinline__ Loader(const AttnArgs& a, Control& k, unsigned slots, int t) : a(a), k(k), slots(slots), tid(t), lane(t & 31),
      token((t >> 5) * 16 + ((t >> 1) & 7)), block((t & 1) + 2 * (lane >> 4)) {
#pragma unroll
    for (int x = 0; x < 4; ++x) put_at[x] = slots + (block >> 1) * kChunk + unit_at(token, (block & 1) * 4 + x);
  }
  __device__ __forceinline__ Where where(unsigned i) {       // tile i's pages
    wait(k, k.tile_full[i % kTiles], (i / kTiles) & 1);
    const Tile& t = k.tile[i % kTiles];
    const int half = tid >> 7;
    Where w;
    w.page = *(const unsigned char* const volatile*)&t.page[half];
    w.tokens = *(const volatile int*)&t.tokens[half];
    w.live = *(const volatile int*)&t.live != 0;
    w.careful = *(const volatile int*)&t.careful != 0;
    __syncwarp();
    if (lane == 0) arrive(k.tile_empty[i % kTiles]);
    return w;
  }
  template <int P0, int P1>
  __device__ __forceinline__ void load(const Where& w) {     // code[P0 .. P1)
    if (w.tokens) {                                          // rows behind the last token are in the page: read, and not used
      const unsigned char* src = w.page + (token & 63) * (MX8 ? kLatent : 2 * kRow) + block * (MX8 ? 32 : 64);
      if (MX8 && P0 == 0) {
        const unsigned char* sc = w.page + kPageScales + (token & 63) * (kLatent / 32);
        scales[0] = ld_stream_ordered(sc);
        scales[1] = ld_stream_ordered(sc + 8 * (kLatent / 32));
      }
#pragma unroll
      for (int p = P0; p < P1; ++p)
#pragma unroll
        for (int g = 0; g < 2; ++g) code[p][g] = ld_stream32_ordered(src + (MX8 ? p * 128 + g * 8 * kLatent : (p >> 1) * 256 + (p & 1) * 32 + g * 16 * kRow));
    } else {
      if (P0 == 0) scales[0] = scales[1] = V8{{0u, 0u, 0u, 0u}};
#pragma unroll
      for (int p = P0; p < P1; ++p) code[p][0] = code[p][1] = V16{{0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u}};
    }
  }
  __device__ __forceinline__ void hand_over(int p) {
    fence_async();
    __syncwarp();
    if (lane == 0) arrive(k.full[p]);
  }
  __device__ __forceinline__ void copy(int c) {              // a chunk of the warp's tokens straight into its slot: eight lanes to a token
    const int at = (tid >> 5) * 16 + (lane >> 3), unit = lane & 7;
    const unsigned char* src = MX8 ? here.page + kPageRope + (at & 63) * 128 + unit * 16 : here.page + ((at & 63) * kRow + c * 64 + unit * 8) * 2;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const bool there = (at & 63) + 4 * x < here.tokens;
      copy16(slots + c * kChunk + unit_at(at + 4 * x, unit), there ? src + x * (MX8 ? 4 * 128 : 8 * kRow) : reinterpret_cast<const unsigned char*>(a.q), there);
    }
  }
  __device__ __forceinline__ void clean_copy(int c, unsigned i) {
#pragma unroll 1
    for (int x = 0; x < 4; ++x) {
      const int at = (tid >> 5) * 16 + (lane >> 3) + 4 * x;
      unsigned bad = 0;
      clean_units(slots + c * kChunk, at, lane & 7, 1, 0x7f80u, bad);
      if (bad) atomicOr(&k.poison[i & 1][at >> 5], 1u << (at & 31));
    }
  }
  struct Units { uint4 u[4]; };
  __device__ __forceinline__ Units convert(int p, int g, unsigned most) {   // token g of pair p (bf16: 0 or 1)
    Units o;
    if (MX8) {
      const unsigned s = f16_scale(most, (scales[g].w[p] >> (block * 8)) & 0xffu);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        mx8_to_f16x4(code[p][g].w[2 * x], s, o.u[x].x, o.u[x].y);
        mx8_to_f16x4(code[p][g].w[2 * x + 1], s, o.u[x].z, o.u[x].w);
      }
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const V16& v = code[(2 * p + (x >> 1)) & 3][g];
        o.u[x] = make_uint4(v.w[4 * (x & 1)], v.w[4 * (x & 1) + 1], v.w[4 * (x & 1) + 2], v.w[4 * (x & 1) + 3]);
      }
    }
    if ((token & 63) + 8 * g >= here.tokens) o.u[0] = o.u[1] = o.u[2] = o.u[3] = make_uint4(0u, 0u, 0u, 0u);
    return o;
  }
  __device__ __forceinline__ static unsigned base_of(unsigned most) { return (unsigned)max((int)most - 1 - kRoom, 127 + kLeastE); }
  // The largest scale byte again, of blocks that are not all zeros: those have byte 127 whatever lies beside them, and where the others' are below it
  // it would take the range from them.  Run only where 127 is the largest byte: latents whose blocks hold magnitudes up to 224 get there through a block
  // of zeros alone.  (From registers: 318 us for the long document, with the look left out 315; in a rolled loop from L2 318.)
  __device__ __forceinline__ unsigned base_of_blocks() const {
    unsigned most = 0;
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const unsigned byte = (scales[g].w[p] >> (block * 8)) & 0xffu;
        unsigned any = 0;
#pragma unroll
        for (int x = 0; x < 8; ++x) any |= code[p][g].w[x];
        if (byte != 255 && (any & 0x7f7f7f7fu) != 0 && (token & 63) + 8 * g < here.tokens) most = max(most, byte + 1);
      }
    most = __reduce_max_sync(0xffffffffu, most);
    return most ? base_of(most) : 127 + kZeros;
  }
  unsigned bad[2];                                           // the thread's tokens have values that are not finite
  __device__ __forceinline__ void put(int p, int g, const Units& o) {
#pragma unroll
    for (int x = 0; x < 4; ++x) store16(put_at[x] + 2 * p * kChunk + g * 1024, o.u[x]);
  }
  __device__ __forceinline__ void clean_put(int p) {
    if (here.careful) {
      clean_units(slots + (2 * p + (block >> 1)) * kChunk, token, (block & 1) * 4, 4, MX8 ? 0x7c00u : 0x7f80u, bad[0]);
      clean_units(slots + (2 * p + (block >> 1)) * kChunk, token + 8, (block & 1) * 4, 4, MX8 ? 0x7c00u : 0x7f80u, bad[1]);
    }
  }
  __device__ __forceinline__ void empty(unsigned i, int p) { if (i > 0) wait(k, k.empty[p], (i - 1) & 1); }
  // tile i of the CTA into the slots, and the next one on its way
  __device__ __forceinline__ void tile(unsigned i) {
    unsigned most = 0;
    bad[0] = bad[1] = 0;
    if (MX8) {
      // the largest scale byte of the warp's tokens but for 255 (NaN): four lanes share a token, each looks at four of its sixteen bytes, counted up by one
      // modulo 256
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const unsigned w = block < 2 ? (block == 0 ? scales[g].w[0] : scales[g].w[1]) : (block == 2 ? scales[g].w[2] : scales[g].w[3]);
        unsigned m;
        asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(((w & 0x00ff00ffu) + 0x00010001u) & 0x00ff00ffu), "r"((((w >> 8) & 0x00ff00ffu) + 0x00010001u) & 0x00ff00ffu));
        if ((token & 63) + 8 * g < here.tokens) most = max(most, max(m & 0xffffu, m >> 16));
      }
      most = __reduce_max_sync(0xffffffffu, most);
      most = most == 128 ? base_of_blocks() : base_of(most);
    }
    Units u = convert(0, 0, most), v = convert(0, 1, most);
    empty(i, 0);
    if (tid < 4) k.poison[(i + 1) & 1][tid] = 0;             // the tile before this one has been read, the next is not there yet
    if (MX8 && lane == 0) k.exponent[tid >> 5] = (int)most - 127;   // E
    if ((tid & 127) == 0) k.tokens[tid >> 7] = here.tokens;
    put(0, 0, u);
    const unsigned e1 = poll(k.empty[1], (i - 1) & 1);
    u = convert(1, 0, most);                                 // while the stores before it go out
    put(0, 1, v);
    clean_put(0);
    hand_over(0);
    v = convert(1, 1, most);
    if (!e1) empty(i, 1);
    put(1, 0, u);
    copy(8);
    copies_commit();
    if (MX8) {
      const unsigned e2 = poll(k.empty[2], (i - 1) & 1);
      u = convert(2, 0, most);
      put(1, 1, v);
      clean_put(1);
      hand_over(1);
      v = convert(2, 1, most);
      if (!e2) empty(i, 2);
      put(2, 0, u);
      const unsigned e3 = poll(k.empty[3], (i - 1) & 1);
      u = convert(3, 0, most);
      put(2, 1, v);
      clean_put(2);
      hand_over(2);
      v = convert(3, 1, most);
      if (!e3) empty(i, 3);
      put(3, 0, u);
      put(3, 1, v);
      clean_put(3);
      hand_over(3);
    } else {                                                 // the other half of bf16 pages is copied
      put(1, 1, v);
      clean_put(1);
      hand_over(1);
      empty(i, 2);
      copy(4); copy(5);
      copies_commit();
      empty(i, 3);
      copy(6); copy(7);
      copies_commit();
      copies_left<1>();
      if (here.careful) { clean_copy(4, i); clean_copy(5, i); }
      hand_over(2);
      copies_left<0>();
      if (here.careful) { clean_copy(6, i); clean_copy(7, i); }
      hand_over(3);
    }
    copies_left<0>();
    if (here.careful) {
      clean_copy(8, i);
      if (bad[0]) atomicOr(&k.poison[i & 1][token >> 5], 1u << (token & 31));
      if (bad[1]) atomicOr(&k.poison[i & 1][token >> 5], 256u << (token & 31));
    }
    hand_over(4);
    next = where(i + 1);
    if (MX8) {
      load<0, 3>(next);
      wait(k, k.s_read, i & 1);
      load<3, 4>(next);
    } else {
      load<0, 4>(next);
    }
    here = next;
  }
  __device__ __forceinline__ void run() {
    here = where(0);
    load<0, 4>(here);
    for (unsigned i = 0; here.live; ++i) tile(i);
  }
};

// ---- MMA ------------------------------------------------------------------------------------------------------------------------------
template <bool MX8>
__device__ void issue_tiles(Control& k, unsigned q, unsigned p, unsigned slots) {
  const unsigned tmem = *(volatile unsigned*)&k.tmem, sc = tmem + kTmemS, sr = tmem + (MX8 ? kTmemR : kTmemS);
  const unsigned dq = operand(q, 16), dk = operand(slots, 16), dp = operand(p, 16), dv = operand(slots, kChunk);
  unsigned lead;
  asm volatile("{.reg .pred e; elect.sync _|e, 0xffffffff; selp.u32 %0, 1, 0, e;}" : "=r"(lead));
  unsigned i = 0;
  for (unsigned n = 0;; ++n) {
    const Segment s = segment(k, n, true);
    if (s.t1 == 0) break;
    for (int t = s.t0; t < s.t1; ++t, ++i) {
      unsigned ok = 0;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {                          // rolled, as everything that runs once a tile: unrolled code is waited for
        if (t == s.t0) wait(k, k.q_full[c], n & 1);          // the queries come by pairs of chunks, too
        if (!ok) wait(k, k.full[c], i & 1);
        fence_after();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j == 6) ok = poll(k.full[c + 1], i & 1);       // asked while the products are issued
          mma_ws(lead, sc, dq + (((2 * c + (j >> 2)) * kQChunk + (j & 3) * 32) >> 4), dk + (((2 * c + (j >> 2)) * kChunk + (j & 3) * 32) >> 4),
                 shape_of(!MX8, 0), c + j > 0);
        }
      }
      if (!ok) wait(k, k.full[4], i & 1);
      fence_after();
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_ws_tmem(lead, sr, tmem + kTmemQ + j * 8, dk + ((8 * kChunk + j * 32) >> 4), shape_of(true, 0), !MX8 || j > 0);
      commit(lead, k.s_full);
      wait(k, k.p_full, i & 1);
      if (t == s.t0 && n > 0) wait(k, k.o_free, (n - 1) & 1);
      fence_after();
#pragma unroll 1
      for (int u = 0; u < 4; ++u) {                          // 128 output columns each
#pragma unroll
        for (int x = 0; x < 8; ++x)                          // 16 tokens each
          mma_ws(lead, tmem + u * 64, dp + (((x >> 2) * kQChunk + (x & 3) * 32) >> 4), dv + ((u * 2 * kChunk + x * 2048) >> 4), shape_of(!MX8, 1),
                 t > s.t0 || x > 0);
        commit(lead, k.empty[u]);
      }
    }
  }
  commit(lead, k.drained);                                   // no product is on its way when the CTA ends, whoever gave up a wait
#pragma unroll 1
  for (int x = 0; x < kWaitLimit && !poll(k.drained, 0); ++x) {}
}

// ---- softmax ----------------------------------------------------------------------------------------------------------------------------
// Row r of a segment's tile: its address in q, or null where the tile has no such row.
__device__ __forceinline__ const __nv_bfloat16* query(const AttnArgs& a, const Segment& s, int r) {
  const int rows = (s.b < 0 ? a.B : 1) * a.S * a.heads, at = s.row0 + r;   // at most 2^27
  if (at >= rows) return nullptr;
  const int step = at / a.heads;
  return a.q + ((s.b < 0 ? 0 : s.b * a.S) + step) * a.q_stride + (at - step * a.heads) * kRow;
}
// A segment's queries.  Four threads to a row bring its latent columns into shared memory, zeros where the tile has no row: for bf16 pages
// copied, for MXFP8 pages made f16, the row's largest element brought to 2^14 .. 2^15.  The rope columns go into tensor memory,
// 32 of a row from each thread (each row on both halves of the lanes).  They are handed over by pairs of chunks, the rope columns with the first.
template <bool MX8>
__device__ __forceinline__ void fetch_q(const AttnArgs& a, Control& k, const Segment& s, unsigned n, unsigned q, unsigned rope_at, int tid) {
  const int r = tid >> 2;
  const __nv_bfloat16* src = query(a, s, r);
  const uint4* from = reinterpret_cast<const uint4*>(src) + (tid & 3);
  auto read = [](const uint4* p) { const V8 v = ld_plain(p); return make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]); };
  const __nv_bfloat16* rope_src = query(a, s, tid & 63);
  uint4 x[16];
  unsigned top = 0, rope[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (MX8) {
      x[i] = src ? read(from + 4 * i) : make_uint4(0u, 0u, 0u, 0u);
    } else {
      const int unit = 4 * i + (tid & 3);
      copy16(q + (unit >> 3) * kQChunk + unit_at(r, unit & 7), reinterpret_cast<const unsigned char*>(src ? from + 4 * i : reinterpret_cast<const uint4*>(a.q)), src != nullptr);
      if (i % 4 == 3) copies_commit();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 y = rope_src ? read(reinterpret_cast<const uint4*>(rope_src + kLatent + (tid >> 7) * 32) + i) : make_uint4(0u, 0u, 0u, 0u);
    rope[4 * i] = y.x; rope[4 * i + 1] = y.y; rope[4 * i + 2] = y.z; rope[4 * i + 3] = y.w;
  }
  float up = 1.f;
  if (MX8) {
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, absmax8(V8{{x[i].x, x[i].y, x[i].z, x[i].w}}));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = (int)(top >> 7);                           // exponent field of the largest element; 0: subnormals or zeros, 255: not finite
    const int shift = e == 255 ? 0 : max(e - 127 - 14, -120);   // q' = q * 2^-shift
    up = __uint_as_float((unsigned)(127 - shift) << 23);
    if ((tid & 3) == 0) k.row_shift[n & 1][r] = (signed char)shift;
  }
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
               :: K3G_I8(rope, 0), K3G_I8(rope, 8), "r"(rope_at + (tid >> 7) * 16) : "memory");
  tmem_wait_st();
  fence_before();
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (MX8) {
      auto half = [&](unsigned w) {
        const __half2 h = __floats2half2_rn(bf_lo(w) * up, bf_hi(w) * up);
        return *reinterpret_cast<const unsigned*>(&h);
      };
#pragma unroll
      for (int i = 4 * c; i < 4 * c + 4; ++i) {
        const int unit = 4 * i + (tid & 3);
        store16(q + (unit >> 3) * kQChunk + unit_at(r, unit & 7), make_uint4(half(x[i].x), half(x[i].y), half(x[i].z), half(x[i].w)));
      }
    } else {
      if (c == 0) copies_left<3>();
      if (c == 1) copies_left<2>();
      if (c == 2) copies_left<1>();
      if (c == 3) copies_left<0>();
    }
    fence_async();
    arrive(k.q_full[c]);
  }
}
// The four warps that share 32 rows.
__device__ __forceinline__ void softmax_barrier(int rows) {
  if (rows == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
  else asm volatile("bar.sync 2, 128;" ::: "memory");
}
__device__ __forceinline__ bool softmax_vote(int rows, bool mine) {   // the same barrier, and whether it is true for one of them
  unsigned any;
  if (rows == 0) asm volatile("{.reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.or.pred q, 1, 128, p; selp.u32 %0, 1, 0, q;}" : "=r"(any) : "r"((unsigned)mine) : "memory");
  else asm volatile("{.reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.or.pred q, 2, 128, p; selp.u32 %0, 1, 0, q;}" : "=r"(any) : "r"((unsigned)mine) : "memory");
  return any != 0;
}
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// Warp w: rows 32 (w % 2) .. of the tile, of page w / 2 % 2 of each token tile 32 tokens (32 (w / 4) ..), of O the columns on the same lanes, 32 of each
// accumulator.
template <bool MX8>
__device__ void softmax_tiles(const AttnArgs& a, Control& k, unsigned q, unsigned p_mem, int tid) {
  const int r = tid & 63, half = (tid >> 6) & 1, part = tid >> 7, rows32 = (tid >> 5) & 1, first = half * 64 + part * 32;
  const unsigned lanes = (unsigned)((tid >> 5) & 3) << 21;   // this warp's 32 lanes of tensor memory
  const unsigned tmem = *(volatile unsigned*)&k.tmem + lanes, o = tmem + part * 32, sc = tmem + kTmemS + part * 32, tq = tmem + kTmemQ;
  {
    const Segment s = segment(k, 0, false);
    if (s.t1 == 0) return;
    fetch_q<MX8>(a, k, s, 0, q, tq, tid);
  }
  unsigned i = 0;
  for (unsigned n = 0;; ++n) {
    const Segment s = segment(k, n, true);
    if (s.t1 == 0) return;
    int seen = s.tokens;                                     // tokens that the row sees
    if (s.b >= 0) seen = s.tokens - (a.S - 1 - min((s.row0 + r) / a.heads, a.S - 1));
    float row_scale = 1.f;
    float m = -INFINITY, l = 0.f;                            // the maximum that P and O are relative to, and this thread's share of the sum
#pragma unroll 1
    for (int t = s.t0; t < s.t1; ++t, ++i) {
      // what the loaders left about the tile is read when they have handed it over: with S itself it would queue behind their next loads
      wait(k, k.full[4], i & 1);
      int ex[2] = {0, 0};                                    // E of the thread's two runs of 16 tokens
      if (MX8) { ex[0] = *(volatile int*)&k.exponent[first >> 4]; ex[1] = *(volatile int*)&k.exponent[(first >> 4) + 1]; }
      // visible ones of this thread's 32 tokens, if not below 0 or above 32
      const int live = min(seen - t * kTile - half * 64, *(volatile int*)&k.tokens[half]) - part * 32;
      unsigned mine = 0;                                     // those with values that are not finite, in tiles that not all rows see all of
      if (s.b >= 0 && a.S > 1 && live > 0) mine = *(volatile unsigned*)&k.poison[i & 1][2 * half + part] & (~0u >> (32 - min(live, 32)));
      const bool zeros = MX8 && min(ex[0], ex[1]) == kZeros;
      wait(k, k.s_full, i & 1);
      fence_after();
      if (MX8 && t == s.t0) row_scale = __uint_as_float((unsigned)(127 + *(volatile signed char*)&k.row_shift[n & 1][r]) << 23);
      unsigned raw[32];
      tmem_ld32(sc, raw);
      if (MX8) {
        unsigned rope[32];
        tmem_ld32(sc + (kTmemR - kTmemS), rope);
        const f32x2 f[2] = {f2_splat(row_scale * __uint_as_float((unsigned)(ex[0] + 127) << 23)), f2_splat(row_scale * __uint_as_float((unsigned)(ex[1] + 127) << 23))};
        tmem_wait_ld();
        if ((tid & 31) == 0) arrive(k.s_read);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float u, v;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(raw[j]), __uint_as_float(raw[j + 1])), f[j >> 4], f2_pack(__uint_as_float(rope[j]), __uint_as_float(rope[j + 1]))), u, v);
          raw[j] = __float_as_uint(u); raw[j + 1] = __float_as_uint(v);
        }
      } else {
        tmem_wait_ld();
      }
      if (a.flip) {
#pragma unroll
        for (int j = 0; j < 32; ++j) raw[j] ^= 0x80000000u;
      }
      if (live < 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) raw[j] = j < live ? raw[j] : 0xff800000u;
      }
      if (mine) l = NAN;
      // the row's maximum only where a score is above what P and O are relative to (or tokens are all zeros, below): all four threads of all 32 rows vote
      float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 16; ++j) tops[j >> 2] = max3(tops[j >> 2], __uint_as_float(raw[2 * j]), __uint_as_float(raw[2 * j + 1]));
      float top = fmaxf(fmaf(fmaxf(tops[0], tops[1]), a.c, (float)ex[0]), fmaf(fmaxf(tops[2], tops[3]), a.c, (float)ex[1]));
      if (softmax_vote(rows32, t == s.t0 || zeros || top > m + kLag)) {
        k.best[2 * part + half][r] = top;
        softmax_barrier(rows32);
        top = fmaxf(fmaxf(k.best[0][r], k.best[1][r]), fmaxf(k.best[2][r], k.best[3][r]));
        if (t == s.t0) {
          m = top;
        } else {                                             // O of these 32 rows catches up with the maximum; the product before this one is done
          const float best = fmaxf(m, top), h = best == -INFINITY ? 1.f : exp2_fast(0.5f * (m - best)), f = h * h;
          l = l * h * h;                                     // by halves: where E has grown by more than f32's range, the sum has not
          m = best;
#pragma unroll 1
          for (int c = 0; c < 256; c += 64) {
            unsigned v[32];
            tmem_ld32(o + c, v);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * f);
            tmem_st32(o + c, v);
          }
          tmem_wait_st();
        }
        if (zeros) {                                         // P' does not count there, so the exponentials may be relative to these tokens' own maximum
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            float best = -INFINITY;
#pragma unroll
            for (int j = 16 * g; j < 16 * g + 16; j += 2) best = max3(best, __uint_as_float(raw[j]), __uint_as_float(raw[j + 1]));
            if (ex[g] == kZeros) ex[g] = min(max(__float2int_rd(m - best * a.c), kZeros), kMostE);
          }
        }
      }
      const float off = kTop - (m == -INFINITY ? 0.f : m);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const f32x2 off2 = f2_splat(off + (float)ex[g]);
        f32x2 sum2[2] = {f2_splat(0.f), f2_splat(0.f)};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          unsigned pw[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = 16 * g + 8 * u + 2 * j;
            float e0, e1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(raw[at]), __uint_as_float(raw[at + 1])), f2_splat(a.c), off2), e0, e1);
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
          store16(p_mem + half * kQChunk + unit_at(r, part * 4 + 2 * g + u), make_uint4(pw[0], pw[1], pw[2], pw[3]));
        }
        float s0, s1;
        f2_unpack(f2_add(sum2[0], sum2[1]), s0, s1);
        l = fmaf(s0 + s1, __uint_as_float((unsigned)(127 - ex[g]) << 23), l);   // a token's weight itself, without its 2^E
      }
      fence_async();
      fence_before();
      arrive(k.p_full);
    }
    // the last product with this segment's queries is done: the next segment's take their place while P V goes on
    const Segment next = segment(k, n + 1, false);
    if (next.t1 > 0) fetch_q<MX8>(a, k, next, n + 1, q, tq, tid);
    // this stretch's unnormalised outputs, maximum and sum; the outputs by 128 columns, as P V leaves them
    const bool live_row = query(a, s, r) != nullptr;
    const long long at = (long long)blockIdx.x + s.tile;
    softmax_barrier(rows32);                                 // the last tile's maxima have been read by all four warps
    k.best[2 * part + half][r] = l;
    softmax_barrier(rows32);
    if (half + part == 0 && live_row) a.sums[at * kRows + r] = make_float2(m, (k.best[0][r] + k.best[1][r]) + (k.best[2][r] + k.best[3][r]));
    softmax_barrier(rows32);                                 // the sums are read before a maximum takes their place
    float* dst = a.parts + at * kPartFloats + ((half * 8 + part * 4) * kRows + r) * 8;
#pragma unroll 1
    for (int u = 0; u < 4; ++u) {
      wait(k, k.empty[u], (i - 1) & 1);
      fence_after();
      unsigned v[32];
      tmem_ld32(o + u * 64, v);
      tmem_wait_ld();
      if (live_row) {
#pragma unroll
        for (int j = 0; j < 32; j += 8)
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" :: "l"(dst + (u * 16 + j / 8) * (kRows * 8)), K3G_I8(v, j) : "memory");
      }
    }
    fence_before();
    arrive(k.o_free);
  }
}

// ---- planning ---------------------------------------------------------------------------------------------------------------------------
// The CTA's segments and their tiles into the rings, and for the join the first and the last CTA of each row tile.
__device__ __forceinline__ void plan_tile(Control& k, unsigned i, const Tile& t, int lane) {
  if (i >= kTiles) wait(k, k.tile_empty[i % kTiles], (i / kTiles - 1) & 1, 200);
  if (lane == 0) {
    k.tile[i % kTiles] = t;
    arrive(k.tile_full[i % kTiles]);
  }
  __syncwarp();
}
__device__ __forceinline__ void prefetch(const unsigned char* p, int bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" :: "l"(p), "r"(bytes) : "memory");
}
__device__ void plan(const AttnArgs& a, Control& k, int ptok, int page_bytes, int lane) {
  long long left = k.left;
  int tile = k.first_tile, at = k.first_at;
  unsigned i = 0;
  for (unsigned n = 0;; ++n) {
    Segment s = {0, -1, 0, 0, 0, 0};
    const int* table = a.prefix_table;
    while (left > 0) {
      s.b = -1; s.row0 = tile * kRows; s.tokens = ptok;
      if (tile >= a.prefix_tiles) {
        s.b = (tile - a.prefix_tiles) / a.seq_tiles;
        if (s.b >= a.B) break;
        s.row0 = (tile - a.prefix_tiles - s.b * a.seq_tiles) * kRows;
        s.tokens = own_tokens(a, s.b);
        table = a.block_table + (long long)s.b * a.max_pages;
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
    if (n >= kRing) wait(k, k.ring_empty[n % kRing], (n / kRing - 1) & 1, 200);
    if (lane == 0) {
      k.ring[n % kRing] = s;
      arrive(k.ring_full[n % kRing]);
    }
    __syncwarp();
    if (s.t1 == 0) {
      plan_tile(k, i, Tile{{a.cache, a.cache}, {0, 0}, 0, 0}, lane);
      return;
    }
    const int pages = (s.tokens + kPageTokens - 1) / kPageTokens;
    int ids = 0;                                             // of page base + lane
#pragma unroll 1
    for (int t = s.t0; t < s.t1; ++t, ++i) {
      const int off = (t - s.t0) * 2 % 32;
      if (off == 0) ids = 2 * t + lane < pages ? ld_ordered(table + 2 * t + lane) : -1;
      Tile w;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int id = __shfl_sync(0xffffffffu, ids, off + h);
        const bool held = id >= 0 && id < a.pages;
        w.page[h] = a.cache + (held ? id : 0) * a.page_stride;
        w.tokens[h] = held ? max(0, min(kPageTokens, s.tokens - (2 * t + h) * kPageTokens)) : 0;
      }
      w.live = 1;
      // steps of a sequence do not see all of its last S - 1 tokens: a value that is not finite must not reach the others through 0 * NaN
      w.careful = s.b >= 0 && a.S > 1 && (t + 1) * kTile > s.tokens - (a.S - 1);
      plan_tile(k, i, w, lane);
      // L2 has the pages before the loaders ask for them (two or three tiles ahead: 340 us for the long document when it was added, without it 346)
      if (lane < 2 && (lane ? w.tokens[1] : w.tokens[0])) prefetch(lane ? w.page[1] : w.page[0], page_bytes);
    }
  }
}

template <bool MX8>
__global__ void __launch_bounds__(kThreads, 1) latent_attn_kernel(const __grid_constant__ AttnArgs a) {
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<unsigned long long>(raw) + 1023) & ~1023ull);
  __shared__ Control k;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    auto init = [](unsigned long long& bar, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(su(&bar)), "r"(n)); };
    for (int u = 0; u < 5; ++u) init(k.full[u], kLoaders / 32);
#pragma unroll 1
    for (int u = 0; u < 4; ++u) { init(k.empty[u], 1); init(k.q_full[u], kSoftmax); }
    init(k.s_full, 1); init(k.s_read, kSoftmax / 32); init(k.p_full, kSoftmax);
#pragma unroll 1
    for (int u = 0; u < kRing; ++u) { init(k.ring_full[u], 1); init(k.ring_empty[u], kReaders); }
#pragma unroll 1
    for (int u = 0; u < kTiles; ++u) { init(k.tile_full[u], 1); init(k.tile_empty[u], kLoaders / 32); }
    init(k.o_free, kSoftmax); init(k.drained, 1);
    k.abort = 0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) k.poison[i >> 2][i & 3] = 0;
#pragma unroll 1
    for (int u = 0; u < kRing; ++u) k.ring[u] = Segment{0, -1, 0, 0, 0, 0};
#pragma unroll 1
    for (int u = 0; u < kTiles; ++u) k.tile[u] = Tile{{a.cache, a.cache}, {0, 0}, 0, 0};
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(su(&k.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  follow_launch();                                           // what came before this launch is done; the join may begin, and waits for this one
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
  fence_async();
  fence_before();
  __syncthreads();
  fence_after();
  long long at = lane < kThreads / 32 ? k.scan[lane] : 0, upto_warp = at;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto_warp, o);
    if (lane >= o) upto_warp += v;
  }
  const long long total = prefix_places + __shfl_sync(0xffffffffu, upto_warp, 31);
  long long before = prefix_places + __shfl_sync(0xffffffffu, upto_warp - at, warp) + upto - mine;
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
      asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
      softmax_tiles<MX8>(a, k, su(q), su(p), tid);
    } else if (warp < (kSoftmax + kLoaders) / 32) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
      Loader<MX8>(a, k, su(slots), tid - kSoftmax).run();
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
      if (warp == (kSoftmax + kLoaders) / 32) issue_tiles<MX8>(k, su(q), su(p), su(slots));
      else if (warp == (kSoftmax + kLoaders) / 32 + 3) plan(a, k, ptok, MX8 ? kMx8Page : 2 * kBf16Page, lane);
    }
  }
  fence_before();
  __syncthreads();
  if (tid == 0) a.status[blockIdx.x] = k.abort;
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(k.tmem) : "memory");
}

// ---- joining the parts of each row ------------------------------------------------------------------------------------------------------
// A team of four warps for four rows that follow one another, warp w its columns 128 w .. + 127: a lane has of one row 16 columns, and the eight lanes
// that load together read 128 bytes that lie together when the rows lie in one tile.  GROUPS teams share the parts of their rows.
// Parts are weighed by 2^(m - max m), the maximum a running one; the order of the sums depends on the lengths alone.
template <int GROUPS>
__global__ void __launch_bounds__(128 * GROUPS) latent_attn_join_kernel(const __grid_constant__ AttnArgs a, int ctas, int rows) {
  __shared__ float4 s_out[GROUPS > 1 ? GROUPS - 1 : 1][4][128];
  __shared__ float2 s_sum[GROUPS > 1 ? GROUPS - 1 : 1][128];
  const int tid = threadIdx.x, lane = tid & 31, quarter = (tid >> 5) & 3, g = tid >> 7, t = tid & 127;
  const int row = blockIdx.x * 4 + ((lane >> 1) & 3);
  const bool there = row < rows;
  const int per_seq = a.S * a.heads, b = there ? row / per_seq : 0, in_seq = row - b * per_seq;
  // read before the wait: the attention kernel lets this one begin when what came before it has ended; from L2, which has what that wrote
  const int len = ld_l2(a.lens + b), ptok = a.prefix_pages ? tokens_of(ld_l2(a.prefix_len), a.prefix_pages) : 0, own = tokens_of(len, a.max_pages);
  const bool live = there && len >= 0;
  // the parts: those of the row's tile against the prefix, then those against its own tokens; part (CTA, tile) has index CTA + tile
  const int ptile = row / kRows, otile = a.prefix_tiles + b * a.seq_tiles + in_seq / kRows;
  follow_launch();
  int gave_up = 0;
  for (int i = tid; i < ctas; i += 128 * GROUPS) gave_up |= a.status[i];
  const int2 ps = live && ptok ? a.spans[ptile] : make_int2(0, -1), os = live && own ? a.spans[otile] : make_int2(0, -1);
  const int np = ps.y + 1 - ps.x, parts = np + os.y + 1 - os.x;
  const int col = (quarter * 16 + (lane >> 3)) * (kRows * 8) + (lane & 1) * 4;   // of the lane's first columns within a part; the next 4 groups on
  float4 acc[4] = {};
  float l = 0.f, best = -INFINITY;
#pragma unroll 2
  for (int i = g; i < parts; i += GROUPS) {
    const long long part = i < np ? ps.x + i + ptile : os.x + (i - np) + otile;
    const int r = (i < np ? row : in_seq) % kRows;
    const float2 ml = a.sums[part * kRows + r];
    float4 v[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = __ldcs(reinterpret_cast<const float4*>(a.parts + part * kPartFloats + col + r * 8 + x * 4 * (kRows * 8)));
    const float top = fmaxf(best, ml.x), off = top == -INFINITY ? 0.f : top, h0 = exp2f(0.5f * (best - off)), h = exp2f(0.5f * (ml.x - off)), f0 = h0 * h0, f = h * h;
    best = top;
    l = ml.y * h * h + l * h0 * h0;                          // by halves: maxima of S + E may lie further apart than f32's exponents, sums do not
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      acc[x].x = fmaf(v[x].x, f, acc[x].x * f0); acc[x].y = fmaf(v[x].y, f, acc[x].y * f0);
      acc[x].z = fmaf(v[x].z, f, acc[x].z * f0); acc[x].w = fmaf(v[x].w, f, acc[x].w * f0);
    }
  }
  if (GROUPS > 1 && g > 0) {
#pragma unroll
    for (int x = 0; x < 4; ++x) s_out[g - 1][x][t] = acc[x];
    s_sum[g - 1][t] = make_float2(best, l);
  }
  const bool failed = __syncthreads_or(gave_up);
  if (!live || g > 0) return;                                // no sequence: left as it was
  if (GROUPS > 1) {
#pragma unroll
    for (int i = 0; i < GROUPS - 1; ++i) {
      const float2 ml = s_sum[i][t];
      const float top = fmaxf(best, ml.x), off = top == -INFINITY ? 0.f : top, h0 = exp2f(0.5f * (best - off)), h = exp2f(0.5f * (ml.x - off)), f0 = h0 * h0, f = h * h;
      best = top;
      l = ml.y * h * h + l * h0 * h0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float4 v = s_out[i][x][t];
        acc[x].x = fmaf(v.x, f, acc[x].x * f0); acc[x].y = fmaf(v.y, f, acc[x].y * f0);
        acc[x].z = fmaf(v.z, f, acc[x].z * f0); acc[x].w = fmaf(v.w, f, acc[x].w * f0);
      }
    }
  }
  // a sum of exactly 0 has seen no token; NaN stays NaN; a call whose kernel gave up a wait has no result
  const float f = failed || l != l ? NAN : l == 0.f ? 0.f : __frcp_rn(l);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    uint2 w = make_uint2(pack_bf2(acc[x].x * f, acc[x].y * f), pack_bf2(acc[x].z * f, acc[x].w * f));
    if (l == 0.f && !failed) w = make_uint2(0u, 0u);
    *reinterpret_cast<uint2*>(a.out + (long long)row * kLatent + (quarter * 16 + (lane >> 3) + 4 * x) * 8 + (lane & 1) * 4) = w;
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
  s.bytes = s.parts + parts * kPartFloats * 4 + 16;          // parts are stored 32 bytes at a time: the space begins at such a border
  return s;
}

template <int GROUPS>
cudaError_t launch_join(const AttnArgs& a, int ctas, int rows, cudaStream_t stream) {
  return k3g_launch_behind(latent_attn_join_kernel<GROUPS>, (unsigned)((rows - 1) / 4 + 1), 128 * GROUPS, 0, 1, stream, a, ctas, rows);
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
  const long long grain = 32;
  K3G_REQUIRE(q_stride % 8 == 0 && layer_off * unit % grain == 0 && page_stride * unit % grain == 0 && (reinterpret_cast<uintptr_t>(cache) & (grain - 1)) == 0, K3G_EALIGN);
  K3G_REQUIRE(S > 0 && heads > 0 && q_stride >= (long long)heads * kRow && layer_off >= 0 && page_stride * unit >= layer_off * unit + page, K3G_ESHAPE);
  K3G_REQUIRE(B <= kMaxBatch && (long long)S * heads <= kMaxRowsPerSeq && prefix_pages <= (1 << 20) && max_pages <= (1 << 20), K3G_ELIMIT);
  K3G_REQUIRE(scale - scale == 0.f, K3G_ERANGE);             // finite
  const Space sp = space_of(B, S, heads);
  K3G_REQUIRE(workspace_bytes >= sp.bytes, K3G_EWORKSPACE);
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  auto kernel = cache_mx8 ? latent_attn_kernel<true> : latent_attn_kernel<false>;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  unsigned char* ws = (unsigned char*)((reinterpret_cast<uintptr_t>(workspace) + 31) & ~(uintptr_t)31);
  const long long rows = (long long)B * S * heads;
  const int ctas = sms < kMaxCtas ? sms : kMaxCtas;
  AttnArgs a = {(const __nv_bfloat16*)q, q_stride, (const unsigned char*)cache + layer_off * unit, page_stride * unit, pages,
                (const int*)prefix_table, (const int*)prefix_len, prefix_pages, (const int*)block_table, (const int*)lens, max_pages,
                (__nv_bfloat16*)out, (int*)ws, (int2*)(ws + sp.spans), (float2*)(ws + sp.sums), (float*)(ws + sp.parts),
                B, S, heads, (int)((rows + kRows - 1) / kRows), (S * heads + kRows - 1) / kRows, fmaxf(fabsf(scale) * 1.44269504088896341f, 1e-30f), scale < 0.f};
  e = k3g_launch_behind(kernel, (unsigned)ctas, kThreads, kSmem, 1, k3g_stream(stream), a);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  // Few rows mean many parts for each and few blocks: several teams share a row's parts.  Whole calls with 1, 2 and 4 teams, own 512 tokens and a prefix of 8192: 768 rows 51.8, 44.0, 42.1 us; 1152 rows 58.7, 52.4, 50.9; 1200 rows 58.1, 52.5,
  // 53.3; 2400 rows 89.1, 85.8, 89.6; 4608 rows 142.8, 142.5, 146.0 (without the prefix 30.2, 30.4, 34.4).
  const int n = (int)rows;
  e = n <= 8 * sms ? launch_join<4>(a, ctas, n, k3g_stream(stream)) : n <= 24 * sms ? launch_join<2>(a, ctas, n, k3g_stream(stream)) : launch_join<1>(a, ctas, n, k3g_stream(stream));
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  return k3g_launch_status();
}
