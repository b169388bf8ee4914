// MXFP8 latent cache: rows quantised as they are appended, and pages read back as contiguous bf16 rows.
//
// For a row x of 576 bf16 and each block of 32 of its first 512 columns: e = the smallest integer with 448 * 2^e >= max|x|
// (0 for an all-zero block), code = E4M3(x * 2^-e) to nearest even, scale byte e + 127; the last 64 columns stay bf16.
// Reading back gives code * 2^e, which bf16 holds exactly.  No counterpart in the reference, whose cache is bf16
// (source/k3_mla_prep_v2.cu:200-211 writes it, source/k3_mla_v2.cu:22-33 reads it).
//
// Bound by HBM: 1808 bytes a row either way.  ONE WARP PER ROW: lane l owns columns 16 l .. 16 l + 15, so a block of 32 is
// two neighbouring lanes (its maximum is one shuffle), codes move as one 16-byte access per lane, and lanes 0..7 move the
// rope columns.  No shared memory, no block barrier.  One row and no loop: 131072 rows are stored in 39 us (6.1 TB/s, 93% of a
// copy), with a loop over rows 44, with two or four rows loaded ahead 40 and 41; 65500 rows are read back in 22.5 us (5.3 TB/s:
// nearly twice as many bytes are written as read), with two rows ahead 24.8.  Launched behind what comes before, 37.2 and 20.4 us (6.4 and
// 5.8 TB/s); 16383 rows are stored in 5.0 us, 96 in 1.5.
#include "latent_page.cuh"
#include "k3g_host.h"

using namespace k3g;

namespace {

constexpr int kWarps = 8;

__global__ void __launch_bounds__(32 * kWarps) latent_mx8_store_kernel(const __nv_bfloat16* rows, long long row_stride,
                                                                       const long long* slot_mapping,
                                                                       unsigned char* cache, long long page_stride,
                                                                       long long slots, int T) {
  const int lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  follow_launch();
  if (t >= T) return;
  const long long slot = ld_ordered(slot_mapping + t);
  const __nv_bfloat16* row = rows + t * row_stride;
  const V8 a = ld_stream_ordered(row + 16 * lane), b = ld_stream_ordered(row + 16 * lane + 8);
  V8 r;
  if (lane < 8) r = ld_stream_ordered(row + kLatent + 8 * lane);
  unsigned m = max_bf16_bits(absmax8(a), absmax8(b));
  m = max_bf16_bits(m, __shfl_xor_sync(0xffffffffu, m, 1));
  const int e = ue8m0_exp_from_bf16(m);
  const float s = pow2_neg(e);
  V8 q;
  quant8(a, s, q.w[0], q.w[1]);
  quant8(b, s, q.w[2], q.w[3]);
  if (slot < 0 || slot >= slots) return;                     // no slot: nothing is appended
  unsigned char* page = cache + (slot >> 6) * page_stride;
  const int at = (int)(slot & 63);
  st_plain(page + at * kLatent + 16 * lane, q);
  if (lane < 8) st_plain(page + kPageRope + at * (2 * kRopeCols) + 16 * lane, r);
  if ((lane & 1) == 0) page[kPageScales + at * (kLatent / 32) + (lane >> 1)] = (unsigned char)(e + 127);
}

__global__ void __launch_bounds__(32 * kWarps) latent_mx8_gather_kernel(const unsigned char* cache, const int* block_table,
                                                                        long long page_stride, long long pages, const int* lens,
                                                                        __nv_bfloat16* out, int n) {
  const int lane = threadIdx.x & 31;
  follow_launch();
  const int len = ld_ordered(lens);
  const long long t = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (t >= n) return;
  V8 a = {{0u, 0u, 0u, 0u}}, b = a, r = a;
  const int id = t < len ? ld_ordered(block_table + (t >> 6)) : -1;
  if (id >= 0 && id < pages) {
    const unsigned char* page = cache + id * page_stride;
    const int at = (int)(t & 63);
    const V8 q = ld_stream_ordered(page + at * kLatent + 16 * lane);
    if (lane < 8) r = ld_stream_ordered(page + kPageRope + at * (2 * kRopeCols) + 16 * lane);
    const unsigned s = ue8m0_pair(ld_ordered(page + kPageScales + at * (kLatent / 32) + (lane >> 1)));
    mx8_to_bf16x4(q.w[0], s, a.w[0], a.w[1]);
    mx8_to_bf16x4(q.w[1], s, a.w[2], a.w[3]);
    mx8_to_bf16x4(q.w[2], s, b.w[0], b.w[1]);
    mx8_to_bf16x4(q.w[3], s, b.w[2], b.w[3]);
  }
  __nv_bfloat16* row = out + t * kRow;
  st_stream(row + 16 * lane, a);
  st_stream(row + 16 * lane + 8, b);
  if (lane < 8) st_stream(row + kLatent + 8 * lane, r);
}

}  // namespace

K3G_API int k3g_latent_mx8_store(const void* rows, long long row_stride, const void* slot_mapping, void* cache, long long layer_off,
                                 long long page_stride, long long pages, int T, void* stream) {
  K3G_REQUIRE_PTR(rows); K3G_REQUIRE_PTR(slot_mapping); K3G_REQUIRE_PTR(cache);
  K3G_REQUIRE_ALIGNED(rows); K3G_REQUIRE_ALIGNED(cache);
  K3G_REQUIRE(row_stride % 8 == 0 && layer_off % 32 == 0 && page_stride % 32 == 0 && (reinterpret_cast<uintptr_t>(cache) & 31u) == 0, K3G_EALIGN);
  K3G_REQUIRE(T >= 0 && pages >= 0 && pages < (1ll << 31), K3G_ESHAPE);
  if (T == 0) return K3G_OK;
  K3G_REQUIRE(row_stride >= kRow && layer_off >= 0 && page_stride >= layer_off + kMx8Page, K3G_ESHAPE);
  const cudaError_t e = k3g_launch_behind(latent_mx8_store_kernel, (T - 1) / kWarps + 1, 32 * kWarps, 0, 1, k3g_stream(stream), (const __nv_bfloat16*)rows, row_stride,
                                          (const long long*)slot_mapping, (unsigned char*)cache + layer_off, page_stride, pages * kPageTokens, T);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  return k3g_launch_status();
}

K3G_API int k3g_latent_mx8_gather(const void* cache, const void* block_table, long long layer_off, long long page_stride, long long pages,
                                  const void* lens, void* out, int n, void* stream) {
  K3G_REQUIRE_PTR(cache); K3G_REQUIRE_PTR(block_table); K3G_REQUIRE_PTR(lens); K3G_REQUIRE_PTR(out);
  K3G_REQUIRE_ALIGNED(cache); K3G_REQUIRE_ALIGNED(out);
  K3G_REQUIRE(layer_off % 32 == 0 && page_stride % 32 == 0 && (reinterpret_cast<uintptr_t>(cache) & 31u) == 0, K3G_EALIGN);
  K3G_REQUIRE(n >= 0 && pages >= 0 && pages < (1ll << 31), K3G_ESHAPE);
  if (n == 0) return K3G_OK;
  K3G_REQUIRE(layer_off >= 0 && page_stride >= layer_off + kMx8Page, K3G_ESHAPE);
  const cudaError_t e = k3g_launch_behind(latent_mx8_gather_kernel, (n - 1) / kWarps + 1, 32 * kWarps, 0, 1, k3g_stream(stream),
                                          (const unsigned char*)cache + layer_off, (const int*)block_table, page_stride, pages, (const int*)lens, (__nv_bfloat16*)out, n);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  return k3g_launch_status();
}
