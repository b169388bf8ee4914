// Attention of a batch over the paged latent cache, the prefix that the batch shares read once for all of it.
//
// out[b, s, h] = sum_j p_j k_j[0:512], p = softmax_j(scale * q[b, s, h] . k_j), j over the tokens that step s of sequence b sees:
// the shared prefix, and its own tokens up to the one of step s (the last S of its own tokens are the S steps).  A latent row is
// key (576 columns) and value (its first 512) at once, so a tile of tokens is loaded once and used by two products.
//
// Work.  All rows (b, s, h) in tiles of 64 against the prefix, and each sequence's rows in tiles of 64 against its own
// tokens, in tiles of 128 tokens (two pages): every (row tile, token tile) pair costs the same, so the pairs are laid in one line
// (row tile by row tile) and each CTA takes an equal stretch, whatever the lengths are.  A stretch that covers a part of a row tile
// leaves an unnormalised f32 output with its maximum and sum in the workspace (one pass over the tokens, running maximum and
// sum in 32 bits), and a second, dependent launch joins the parts of each row.  Lengths and tables are read on the device:
// a captured graph follows them.  Nothing is accumulated by atomics: the same inputs give the same bits.
//
// One CTA per SM, 13 warps with fixed roles, one tile after another:
//   8 loader warps   fetch the next tile's codes into registers a whole tile ahead, and when a slot is free convert them to bf16
//                    (exact: four significant bits times a power of two) into 128-byte-swizzled shared memory, in nine 16 KB chunks of 64 columns;
//   1 MMA warp       S = Q K^T (64 x 128, nine chunks as they come) and O += P V (64 x 512 in tensor memory), both tcgen05.mma.ws with M = 64;
//   4 softmax warps  S from tensor memory, running maximum, P = 2^(S - m) rounded to bf16 into the slot of the rope chunk (which V does not have).
// Why M = 64: a 128-row O of 512 columns fills the whole tensor memory and leaves no room for S.  The weight-stationary form puts
// a 64-row tile on all 128 lanes and reaches 80 cycles per 64 x 256 x 16 step, the plain form 128 (measured; 64 would be full rate).
// Why 128 tokens: the 64 x 64 x 16 step of S costs 44 cycles, the 64 x 128 x 16 step 48.
// P is rounded to bf16 because the matrix instructions take both operands in one type; the sums of P are kept unrounded in f32.
// The running maximum that P is relative to follows the true one only when it falls behind by more than 2^8 (O is then rescaled): the ratio is
// exact either way, and P <= 2^8 keeps its relative precision.
#include <cuda_runtime.h>

#include "latent_page.cuh"
#include "k3g_host.h"

using namespace k3g;

namespace {

constexpr int kMaxBatch = 4096, kMaxRowsPerSeq = 1 << 15, kMaxCtas = 160;
constexpr int kRows = 64, kTile = 128;                       // query rows and tokens of a tile
constexpr int kLoaders = 256, kSoftmax = 128, kThreads = kLoaders + kSoftmax + 32;
constexpr int kChunk = kTile * 128;                          // 64 columns of a tile's tokens, bf16
constexpr int kQChunk = kRows * 128;
constexpr int kSmemQ = 9 * kQChunk, kSmemK = 9 * kChunk, kSmem = kSmemQ + kSmemK + 1024;
constexpr int kTmemS = 256;                                  // columns: O 0..255 (two accumulators of 256 output columns on 128 lanes each), S 256..319
constexpr float kLag = 8.f;
constexpr int kPartFloats = kRows * kLatent;                 // a part's outputs; its 64 (maximum, sum) pairs lie in a table of their own
constexpr int kWaitLimit = 1 << 20;

struct AttnArgs {
  const __nv_bfloat16* q; long long q_stride;
  const unsigned char* cache; long long page_stride, pages;       // bytes
  const int* prefix_table; const int* prefix_len; int prefix_pages;
  const int* block_table; const int* lens; int max_pages;
  __nv_bfloat16* out;
  int* status;                       // [kMaxCtas] 1: a wait of this CTA expired
  long long* starts;                 // [B + 1] first pair of each sequence's own tokens, and the number of pairs
  float2* sums;                      // [parts][64] (maximum in log2 units, sum)
  float* parts;                      // [parts][64][512]
  int B, S, heads, prefix_tiles, seq_tiles, ctas;
  float c;                           // scale * log2(e)
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
// the CTA that takes pair p, and the first pair of CTA i, of `total` pairs dealt to n CTAs
__device__ __forceinline__ long long cta_of(long long p, long long total, int n) { return ((p + 1) * n - 1) / total; }
__device__ __forceinline__ long long first_of(long long i, long long total, int n) { return total * i / n; }

struct Segment {                     // one CTA's stretch of one row tile
  int tile;                          // row tile: prefix_tiles of them against the prefix, then seq_tiles for each sequence
  int b;                             // sequence, or -1 for the prefix
  int row0;                          // first row: of all rows (prefix) or of the sequence's rows
  int t0, t1;                        // token tiles
  int tokens;                        // tokens of the prefix / of the sequence
  const int* table;
  int table_pages;
};
struct Walk { long long left; int tile, t; };

__device__ __forceinline__ bool next_segment(const AttnArgs& a, int ptok, Walk& w, Segment& s) {
  if (w.left <= 0) return false;
  int nt;
  if (w.tile < a.prefix_tiles) {
    s.b = -1; s.row0 = w.tile * kRows; s.tokens = ptok; s.table = a.prefix_table; s.table_pages = a.prefix_pages;
    nt = tiles_of(ptok);
  } else {
    int b = (w.tile - a.prefix_tiles) / a.seq_tiles, n = 0;
    while (b < a.B && (n = own_tokens(a, b)) == 0) { ++b; w.tile = a.prefix_tiles + b * a.seq_tiles; w.t = 0; }
    if (b >= a.B) return false;
    s.b = b; s.row0 = (w.tile - a.prefix_tiles - b * a.seq_tiles) * kRows; s.tokens = n;
    s.table = a.block_table + (long long)b * a.max_pages; s.table_pages = a.max_pages;
    nt = tiles_of(n);
  }
  s.tile = w.tile; s.t0 = w.t;
  s.t1 = (int)min((long long)nt, w.t + w.left);
  w.left -= s.t1 - s.t0;
  w.t = s.t1;
  if (w.t == nt) { ++w.tile; w.t = 0; }
  return true;
}

// ---- barriers and tensor memory -----------------------------------------------------------------------------------------------
struct Control {
  unsigned long long full[9], empty[2], q_full, s_full, p_full[2];
  unsigned tmem;
  int abort;
  int first_tile, first_t;
  long long scan[kThreads / 32];
  unsigned poison[2][4];
  float best[2][kRows], sum[2][kRows];
};

// Every wait ends: after kWaitLimit polls, or as soon as another wait of the CTA has expired.  The roles then run through what is
// left without waiting (every access stays where it was), and the call's result is NaN.
__device__ __forceinline__ void wait(Control& k, unsigned long long& bar, unsigned parity) {
  for (int i = 0; i < kWaitLimit; ++i) {
    unsigned ok;
    asm volatile("{.reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}" : "=r"(ok) : "r"(su(&bar)), "r"(parity) : "memory");
    if (ok) return;
    if (*(volatile int*)&k.abort) return;
  }
  *(volatile int*)&k.abort = 1;
}
__device__ __forceinline__ void arrive(unsigned long long& bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(su(&bar)) : "memory"); }
__device__ __forceinline__ void commit(unsigned long long& bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(su(&bar)) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory operand descriptor: 128-byte swizzle, `stride` bytes between groups of eight 128-byte rows, `lead` bytes between
// groups of 64 columns (used by the transposed operand only).
__device__ __forceinline__ unsigned long long operand(unsigned addr, unsigned lead, unsigned stride) {
  return (unsigned long long)((addr & 0x3ffffu) >> 4) | ((unsigned long long)(lead >> 4) << 16) | ((unsigned long long)(stride >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ws(unsigned d, unsigned long long a, unsigned long long b, unsigned shape, bool add) {
  asm volatile("{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.ws.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}"
               :: "r"(d), "l"(a), "l"(b), "r"(shape), "r"((unsigned)add) : "memory");
}
// f32 accumulator, bf16 operands, M = 64; `t`: the second operand is stored with its N side contiguous
__device__ __forceinline__ constexpr unsigned shape_of(int n, int t) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)t << 16) | ((unsigned)(n >> 3) << 17) | (4u << 24);
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
// Thread l looks after token l / 2 of a tile and, of each chunk of 64 columns, half l % 2: 32 columns, one scale block.
__device__ __forceinline__ unsigned clean(unsigned w, bool& bad) {   // a pair of bf16 with NaN and infinities taken out
  if ((w & 0x7f80u) == 0x7f80u) { w &= 0xffff0000u; bad = true; }
  if ((w & 0x7f800000u) == 0x7f800000u) { w &= 0x0000ffffu; bad = true; }
  return w;
}
// Four 16-byte units of the thread's half row into chunk memory, swizzled.
__device__ __forceinline__ void put_half(unsigned char* chunk, int token, int half, unsigned (&w)[16], bool careful, bool& bad) {
  if (careful) {
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = clean(w[i], bad);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<uint4*>(chunk + token * 128 + (((half * 4 + i) ^ (token & 7)) << 4)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}

// What the thread holds of a tile before it goes to shared memory.
template <bool MX8> struct Held;
template <> struct Held<true> {
  uint4 code[8][2], rope[4], scale, ahead;
  __device__ __forceinline__ void load(int c, const unsigned char* page, int row, int half) {
    if (c < 8) {
      const uint4* p = reinterpret_cast<const uint4*>(page + row * kLatent + c * 64 + half * 32);
      code[c][0] = __ldg(p); code[c][1] = __ldg(p + 1);
      if (c == 0) ahead = __ldg(reinterpret_cast<const uint4*>(page + kPageScales + row * (kLatent / 32)));
    } else {
      const uint4* p = reinterpret_cast<const uint4*>(page + kPageRope + row * 128 + half * 64);
#pragma unroll
      for (int i = 0; i < 4; ++i) rope[i] = __ldg(p + i);
    }
  }
  __device__ __forceinline__ void zero(int c) {
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    if (c < 8) { code[c][0] = code[c][1] = z; if (c == 0) ahead = z; }
    else rope[0] = rope[1] = rope[2] = rope[3] = z;
  }
  __device__ __forceinline__ void words(int c, int half, unsigned (&w)[16]) {
    if (c == 0) scale = ahead;
    if (c < 8) {
      const unsigned four = c < 2 ? scale.x : c < 4 ? scale.y : c < 6 ? scale.z : scale.w;   // blocks 2 c and 2 c + 1
      const float s = ue8m0_value((four >> ((c & 1) * 16 + half * 8)) & 0xffu);
      const unsigned q[8] = {code[c][0].x, code[c][0].y, code[c][0].z, code[c][0].w, code[c][1].x, code[c][1].y, code[c][1].z, code[c][1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) mx8_to_bf16x4(q[i], s, w[2 * i], w[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) { w[4 * i] = rope[i].x; w[4 * i + 1] = rope[i].y; w[4 * i + 2] = rope[i].z; w[4 * i + 3] = rope[i].w; }
    }
  }
};
// bf16 rows are twice as many registers: the chunks whose slots are freed first are held a tile ahead, the others are fetched
// when their slots are free and arrive while the first ones are multiplied.
template <> struct Held<false> {
  uint4 early[4][4], late[4];
  __device__ __forceinline__ void load(int c, const unsigned char* page, int row, int half) {
    const uint4* p = reinterpret_cast<const uint4*>(page + (row * kRow + c * 64 + half * 32) * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) (c < 4 ? early[c & 3][i] : late[i]) = __ldg(p + i);
  }
  __device__ __forceinline__ void zero(int c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) (c < 4 ? early[c & 3][i] : late[i]) = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void words(int c, int, unsigned (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4& v = c < 4 ? early[c & 3][i] : late[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
};

// Address of the thread's row of a token tile; null where there is none (behind the last token, a page that the cache does not hold).
__device__ __forceinline__ const unsigned char* page_of(const AttnArgs& a, const Segment& s, int t, int token) {
  const long long at = (long long)t * kTile + token;
  if (at >= s.tokens) return nullptr;
  const int id = __ldg(s.table + (at >> 6));
  return id >= 0 && id < a.pages ? a.cache + id * a.page_stride : nullptr;
}

template <bool MX8>
__device__ void load_tiles(const AttnArgs& a, Control& k, unsigned char* slots, int ptok, Walk w, int tid) {
  const int token = tid >> 1, half = tid & 1, row = token & 63;
  Segment s, n;
  if (!next_segment(a, ptok, w, s)) return;
  Held<MX8> held;
  constexpr int kAhead = MX8 ? 9 : 4;
  const unsigned char* page = page_of(a, s, s.t0, token);
#pragma unroll
  for (int c = 0; c < kAhead; ++c) { if (page) held.load(c, page, row, half); else held.zero(c); }
  int t = s.t0;
  for (unsigned i = 0;; ++i) {                               // i: tiles done by this CTA
    // the tile after this one, in this segment or the next
    bool more = true;
    n = s;
    int nt = t + 1;
    if (nt == s.t1) { more = next_segment(a, ptok, w, n); nt = n.t0; }
    const unsigned char* next = more ? page_of(a, n, nt, token) : nullptr;
    // steps of a sequence do not see all of its last S - 1 tokens: a value that is not finite must not reach the others through 0 * NaN
    const bool careful = s.b >= 0 && a.S > 1 && (long long)(t + 1) * kTile > s.tokens - (a.S - 1);
    bool bad = false;
#pragma unroll
    for (int c = 0; c < 9; ++c) {
      if (c == 0 && i > 0) wait(k, k.empty[0], (i - 1) & 1);
      if (c == 4 && i > 0) wait(k, k.empty[1], (i - 1) & 1);
      if (c >= kAhead) { if (page) held.load(c, page, row, half); else held.zero(c); }
      unsigned words[16];
      held.words(c, half, words);
      put_half(slots + c * kChunk, token, half, words, careful, bad);
      if (c == 8 && careful && bad) atomicOr(&k.poison[i & 1][token >> 5], 1u << (token & 31));
      fence_async();
      __syncwarp();
      if ((tid & 31) == 0) arrive(k.full[c]);
      if (c < kAhead) { if (next) held.load(c, next, row, half); else held.zero(c); }
    }
    if (!more) return;
    s = n; t = nt; page = next;
  }
}

// ---- MMA ------------------------------------------------------------------------------------------------------------------------------
__device__ void issue_tiles(const AttnArgs& a, Control& k, unsigned q, unsigned slots, int ptok, Walk w) {
  const unsigned o = k.tmem, sc = k.tmem + kTmemS, p = slots + 8 * kChunk;
  const unsigned long long dq = operand(q, 16, 1024), dk = operand(slots, 16, 1024), dp = operand(p, 16, 1024), dv = operand(slots, kChunk, 1024);
  Segment s;
  unsigned i = 0, seg = 0;
  while (next_segment(a, ptok, w, s)) {
    wait(k, k.q_full, seg & 1);
    ++seg;
    for (int t = s.t0; t < s.t1; ++t, ++i) {
#pragma unroll
      for (int c = 0; c < 9; ++c) {
        wait(k, k.full[c], i & 1);
          fence_after();
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma_ws(sc, dq + ((c * kQChunk + j * 32) >> 4), dk + ((c * kChunk + j * 32) >> 4), shape_of(128, 0), c + j > 0);
      }
      commit(k.s_full);
#pragma unroll
      for (int u = 0; u < 2; ++u) {                          // output columns 0..255, then 256..511
#pragma unroll
        for (int v = 0; v < 2; ++v) {                        // the first 32 tokens of both pages, then the others
          if (u == 0) { wait(k, k.p_full[v], i & 1); fence_after(); }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int step = (x >> 1) * 4 + v * 2 + (x & 1);   // 16 tokens each
            mma_ws(o + u * 128, dp + (((step >> 2) * kQChunk + (step & 3) * 32) >> 4), dv + ((u * 4 * kChunk + step * 2048) >> 4), shape_of(256, 1),
                   t > s.t0 || v + x > 0);
          }
        }
        commit(k.empty[u]);
      }
    }
  }
}

// ---- softmax ----------------------------------------------------------------------------------------------------------------------------
// Query rows of a segment into shared memory: two threads per row, 16 bytes at a time, zeros where the tile has no row.
__device__ __forceinline__ void fetch_q(const AttnArgs& a, const Segment& s, unsigned q, int tid) {
  const int r = tid >> 1;
  const long long rows = s.b < 0 ? (long long)a.B * a.S * a.heads : (long long)a.S * a.heads;
  const long long at = (long long)s.row0 + r;
  const bool live = at < rows;
  const long long step = live ? at / a.heads : 0;
  const __nv_bfloat16* src = a.q + ((s.b < 0 ? 0 : (long long)s.b * a.S) + step) * a.q_stride + (live ? at - step * a.heads : 0) * kRow;
#pragma unroll 4
  for (int i = 0; i < 36; ++i) {
    const int unit = 2 * i + (tid & 1);
    const unsigned dst = q + (unit >> 3) * kQChunk + r * 128 + (((unit & 7) ^ (r & 7)) << 4);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src + unit * 8), "r"(live ? 16 : 0) : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ void q_ready(Control& k) {
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  fence_async();
  arrive(k.q_full);
}
__device__ __forceinline__ void softmax_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Thread t: row t % 64 of the tile, tokens of page t / 64 of each token tile.
__device__ void softmax_tiles(const AttnArgs& a, Control& k, unsigned q, unsigned char* p_slot, int ptok, Walk w, int tid) {
  const int r = tid & 63, half = tid >> 6;
  const unsigned lanes = (unsigned)(tid >> 5) << 21;         // this warp's 32 lanes of tensor memory
  const unsigned o = k.tmem + lanes, sc = k.tmem + kTmemS + lanes;
  unsigned char* p_row = p_slot + half * kQChunk + r * 128;
  Segment s, n;
  if (!next_segment(a, ptok, w, s)) return;
  fetch_q(a, s, q, tid);
  q_ready(k);
  unsigned i = 0;
  for (bool more = true; more;) {
    // tokens that the row sees
    int seen = s.tokens;
    if (s.b >= 0) {
      const int at = s.row0 + r;
      seen = s.tokens - (a.S - 1 - min(at / a.heads, a.S - 1));
    }
    float m = -INFINITY, l = 0.f;                            // the maximum that P and O are relative to, and this thread's share of the sum
    more = next_segment(a, ptok, w, n);
    for (int t = s.t0; t < s.t1; ++t, ++i) {
      const long long base = (long long)t * kTile + half * 64;
      int live = (int)min(64ll, max(0ll, seen - base));      // visible tokens of this thread's page
      if (live > 0) {
        const int id = __ldg(s.table + (base >> 6));
        if (id < 0 || id >= a.pages) live = 0;
      }
      wait(k, k.s_full, i & 1);
      fence_after();
      unsigned x[2][32];
      tmem_ld32(sc, x[0]);
      tmem_ld32(sc + 32, x[1]);
      tmem_wait_ld();
      if (t + 1 == s.t1 && more) fetch_q(a, n, q, tid);      // the last product with this segment's rows is done
      float top = -INFINITY, odd = 0.f;                      // odd turns NaN where a score is not finite
      const bool whole = __all_sync(0xffffffffu, live == 64);
#pragma unroll
      for (int j = 0; j < 64; ++j) {
        float v = __uint_as_float(x[j >> 5][j & 31]) * a.c;
        if (whole || j < live) odd = fmaf(v, 0.f, odd); else v = -INFINITY;
        x[j >> 5][j & 31] = __float_as_uint(v);
        top = fmaxf(top, v);
      }
      const unsigned long long mine = ((unsigned long long)k.poison[i & 1][2 * half + 1] << 32) | k.poison[i & 1][2 * half];
      if (mine && live > 0 && (mine & (~0ull >> (64 - live)))) odd = NAN;
      l += odd;
      k.best[half][r] = top;
      softmax_barrier();
      top = fmaxf(top, k.best[half ^ 1][r]);
      if (tid < 4) k.poison[i & 1][tid] = 0;
      const bool first = t == s.t0;
      if (first) m = top;
      else if (__any_sync(0xffffffffu, top > m + kLag)) {    // O of these 32 rows catches up with the maximum
        const float best = fmaxf(m, top), f = best == -INFINITY ? 1.f : exp2_fast(m - best);
        l *= f;
        m = best;
        for (int c = 0; c < 256; c += 32) {
          unsigned v[32];
          tmem_ld32(o + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * f);
          tmem_st32(o + c, v);
        }
        tmem_wait_st();
      }
      const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          unsigned pw[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e0 = exp2_fast(__uint_as_float(x[g][8 * u + 2 * j]) - off), e1 = exp2_fast(__uint_as_float(x[g][8 * u + 2 * j + 1]) - off);
            l += e0 + e1;
            pw[j] = pack_bf2(e0, e1);
          }
          *reinterpret_cast<uint4*>(p_row + (((g * 4 + u) ^ (r & 7)) << 4)) = make_uint4(pw[0], pw[1], pw[2], pw[3]);
        }
        fence_async();
        fence_before();
        arrive(k.p_full[g]);
      }
    }
    // this stretch's unnormalised outputs, maximum and sum
    wait(k, k.empty[1], (i - 1) & 1);
    fence_after();
    const long long rows = s.b < 0 ? (long long)a.B * a.S * a.heads : (long long)a.S * a.heads;
    const bool live_row = s.row0 + r < rows;
    const long long part = (long long)blockIdx.x + s.tile;
    k.sum[half][r] = l;
    softmax_barrier();
    if (half == 0 && live_row) a.sums[part * kRows + r] = make_float2(m, k.sum[0][r] + k.sum[1][r]);
    float* dst = a.parts + part * kPartFloats + r * kLatent + half * 128;
    for (int c = 0; c < 256; c += 32) {
      unsigned v[32];
      tmem_ld32(o + c, v);
      tmem_wait_ld();
      if (live_row) {
        float* d = dst + (c >> 7) * 256 + (c & 127);
#pragma unroll
        for (int j = 0; j < 32; j += 8)
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" :: "l"(d + j), K3G_I8(v, j) : "memory");
      }
    }
    if (more) {
      fence_before();                                        // the next segment's first product overwrites O: after these loads
      q_ready(k);
      s = n;
    }
  }
}

template <bool MX8>
__global__ void __launch_bounds__(kThreads, 1) latent_attn_kernel(const __grid_constant__ AttnArgs a) {
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<unsigned long long>(raw) + 1023) & ~1023ull);
  __shared__ Control k;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // the line of pairs: own tokens of sequences b0 .. b1 by this thread, then a scan over the block
  const int ptok = prefix_tokens(a);
  const long long prefix_pairs = (long long)a.prefix_tiles * tiles_of(ptok);
  const int per = (a.B + kThreads - 1) / kThreads, b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += (long long)a.seq_tiles * tiles_of(own_tokens(a, b));
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) k.scan[warp] = upto;
  if (tid == 0) {
    for (int c = 0; c < 9; ++c) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(su(&k.full[c])), "r"(kLoaders / 32));
    for (int u = 0; u < 2; ++u) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(su(&k.empty[u])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(su(&k.p_full[u])), "r"(kSoftmax));
    }
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(su(&k.q_full)), "r"(kSoftmax));
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(su(&k.s_full)));
    k.abort = 0;
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
  long long before = prefix_pairs, total = prefix_pairs;
  for (int i = 0; i < kThreads / 32; ++i) { if (i < warp) before += k.scan[i]; total += k.scan[i]; }
  before += upto - mine;
  const int n = (int)min((long long)gridDim.x, total);
  const long long lo = n ? first_of(blockIdx.x, total, n) : 0, hi = n ? first_of(blockIdx.x + 1ll, total, n) : 0;
  const bool busy = (int)blockIdx.x < n;
  if (tid == 0 && busy && lo < prefix_pairs) { k.first_tile = (int)(lo / tiles_of(ptok)); k.first_t = (int)(lo % tiles_of(ptok)); }
  for (int b = b0; b < b1; ++b) {
    const int nt = tiles_of(own_tokens(a, b));
    if (blockIdx.x == 0) a.starts[b] = before;
    if (busy && lo >= before && lo < before + (long long)a.seq_tiles * nt) {
      k.first_tile = a.prefix_tiles + b * a.seq_tiles + (int)((lo - before) / nt);
      k.first_t = (int)((lo - before) % nt);
    }
    before += (long long)a.seq_tiles * nt;
  }
  if (blockIdx.x == 0 && tid == 0) a.starts[a.B] = total;
  __syncthreads();
  if (busy) {
    Walk w = {hi - lo, k.first_tile, k.first_t};
    if (warp < kLoaders / 32) load_tiles<MX8>(a, k, smem + kSmemQ, ptok, w, tid);
    else if (warp < (kLoaders + kSoftmax) / 32) softmax_tiles(a, k, su(smem), smem + kSmemQ + 8 * kChunk, ptok, w, tid - kLoaders);
    else if (lane == 0) issue_tiles(a, k, su(smem), su(smem) + kSmemQ, ptok, w);
  }
  fence_before();
  __syncthreads();
  if (tid == 0) a.status[blockIdx.x] = k.abort;
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(k.tmem) : "memory");
}

// ---- joining the parts of each row ------------------------------------------------------------------------------------------------------
// One block per row, GROUPS x 128 threads: thread j of a group owns columns 4 j .. 4 j + 3, group g takes every GROUPS-th part.  Parts are
// weighed by 2^(m - max m); the order of the sums depends on the lengths alone.
template <int GROUPS>
__global__ void __launch_bounds__(128 * GROUPS) latent_attn_join_kernel(const __grid_constant__ AttnArgs a, int ctas) {
  __shared__ float4 s_out[GROUPS][128];
  __shared__ float s_l[GROUPS];
  const int tid = threadIdx.x, j = tid & 127, g = tid >> 7;
  const long long row = blockIdx.x;
  const int per_seq = a.S * a.heads, b = (int)(row / per_seq), in_seq = (int)(row % per_seq);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int gave_up = 0;
  for (int i = tid; i < ctas; i += 128 * GROUPS) gave_up |= a.status[i];
  const bool failed = __syncthreads_or(gave_up);
  if (__ldg(a.lens + b) < 0) return;                         // no sequence: left as it was
  const long long total = a.starts[a.B];
  const int n = (int)min((long long)ctas, total);
  // the parts: those of the row's tile against the prefix, then those against its own tokens
  const int pt = tiles_of(prefix_tokens(a)), ot = tiles_of(own_tokens(a, b));
  const int ptile = (int)(row / kRows), otile = a.prefix_tiles + b * a.seq_tiles + in_seq / kRows;
  const long long pa = (long long)ptile * pt, oa = a.starts[b] + (long long)(in_seq / kRows) * ot;
  const long long p0 = pt ? cta_of(pa, total, n) : 0, p1 = pt ? cta_of(pa + pt - 1, total, n) + 1 : 0;
  const long long o0 = ot ? cta_of(oa, total, n) : 0, o1 = ot ? cta_of(oa + ot - 1, total, n) + 1 : 0;
  const int np = (int)(p1 - p0), parts = np + (int)(o1 - o0);
  auto slot = [&](int i) { return i < np ? (p0 + i + ptile) * kRows + row % kRows : (o0 + (i - np) + otile) * kRows + in_seq % kRows; };
  float best = -INFINITY;
  for (int i = 0; i < parts; ++i) best = fmaxf(best, a.sums[slot(i)].x);
  const float off = best == -INFINITY ? 0.f : best;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int i = g; i < parts; i += GROUPS) {
    const long long at = slot(i);
    const float2 ml = a.sums[at];
    const float4 v = *reinterpret_cast<const float4*>(a.parts + at * kLatent + 4 * j);
    const float f = exp2f(ml.x - off);
    l = fmaf(ml.y, f, l);
    acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
  }
  if (GROUPS > 1) {
    s_out[g][j] = acc;
    if (j == 0) s_l[g] = l;
    __syncthreads();
    if (g > 0) return;
    for (int i = 1; i < GROUPS; ++i) {
      const float4 v = s_out[i][j];
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
      l += s_l[i];
    }
  }
  // a sum of exactly 0 has seen no token; NaN stays NaN; a call whose kernel gave up a wait has no result
  const float f = failed ? NAN : l == 0.f ? 0.f : __frcp_rn(l);
  if (l == 0.f && !failed) acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (l != l) acc = make_float4(l, l, l, l);
  *reinterpret_cast<uint2*>(a.out + row * kLatent + 4 * j) = make_uint2(pack_bf2(acc.x * f, acc.y * f), pack_bf2(acc.z * f, acc.w * f));
}

// Workspace: status words, starts, (maximum, sum) pairs, parts; the parts of CTA i and row tile t have index i + t.
struct Space { long long starts, sums, parts, bytes; };
Space space_of(int B, int S, int heads) {
  const long long tiles = ((long long)B * S * heads + kRows - 1) / kRows + (long long)B * (((long long)S * heads + kRows - 1) / kRows);
  const long long parts = tiles + kMaxCtas;
  auto up = [](long long x) { return (x + 255) / 256 * 256; };
  Space s;
  s.starts = up(kMaxCtas * 4);
  s.sums = s.starts + up((B + 1ll) * 8);
  s.parts = s.sums + up(parts * kRows * 8);
  s.bytes = s.parts + parts * kPartFloats * 4;
  return s;
}

template <int GROUPS>
cudaError_t launch_join(const AttnArgs& a, int ctas, unsigned rows, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows, 1, 1); cfg.blockDim = dim3(128 * GROUPS, 1, 1); cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, latent_attn_join_kernel<GROUPS>, a, ctas);
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
                (__nv_bfloat16*)out, (int*)ws, (long long*)(ws + sp.starts), (float2*)(ws + sp.sums), (float*)(ws + sp.parts),
                B, S, heads, (int)((rows + kRows - 1) / kRows), (S * heads + kRows - 1) / kRows, ctas, scale * 1.44269504088896341f};
  kernel<<<ctas, kThreads, kSmem, k3g_stream(stream)>>>(a);
  const int rc = k3g_launch_status();
  if (rc != K3G_OK) return rc;
  // Few rows mean many parts for each: four groups of threads share them.
  e = rows <= 592 ? launch_join<4>(a, ctas, (unsigned)rows, k3g_stream(stream)) : launch_join<1>(a, ctas, (unsigned)rows, k3g_stream(stream));
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  return k3g_launch_status();
}
