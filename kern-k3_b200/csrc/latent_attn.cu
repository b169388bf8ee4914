// Attention of a batch over the paged latent cache, the prefix that the batch shares read once for all of it.
//
// out[b, s, h] = sum_j p_j k_j[0:512], p = softmax_j(scale * q[b, s, h] . k_j), j over the tokens that step s of sequence b sees:
// the shared prefix, and its own tokens up to the one of step s (the last S of its own tokens are the S steps).
#include "latent_page.cuh"
#include "k3g_host.h"

using namespace k3g;

namespace {

constexpr int kMaxBatch = 4096, kMaxRowsPerSeq = 1 << 15;

struct AttnArgs {
  const __nv_bfloat16* q; long long q_stride;
  const unsigned char* cache; long long page_stride, pages;       // bytes
  const int* prefix_table; const int* prefix_len; int prefix_pages;
  const int* block_table; const int* lens; int max_pages;
  __nv_bfloat16* out;
  int B, S, heads;
  float scale;
};

// One warp per query row: lane l owns columns l, l + 32, ... of the row.
template <bool MX8>
__global__ void __launch_bounds__(128) latent_attn_simple_kernel(const AttnArgs a) {
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (long long)a.B * a.S * a.heads) return;
  const long long tok = row / a.heads;
  const int h = (int)(row % a.heads), b = (int)(tok / a.S), s = (int)(tok % a.S);
  const int len = a.lens[b];
  if (len < 0) return;
  float q[kRow / 32], o[kLatent / 32] = {}, m = -INFINITY, l = 0.f;
  for (int i = 0; i < kRow / 32; ++i) q[i] = __bfloat162float(a.q[tok * a.q_stride + (long long)h * kRow + lane + 32 * i]);
  for (int part = 0; part < 2; ++part) {
    const int pages = part ? a.max_pages : a.prefix_pages;
    const int* table = part ? a.block_table + (long long)b * a.max_pages : a.prefix_table;
    const int lim = pages * kPageTokens;
    const int n = part ? min(len, lim) - (a.S - 1 - s) : (pages ? min(a.prefix_len[0], lim) : 0);
    for (int t = 0; t < n; ++t) {
      const int id = table[t >> 6];
      if (id < 0 || id >= a.pages) continue;
      const unsigned char* page = a.cache + id * a.page_stride;
      const int at = t & 63;
      float k[kRow / 32];
      for (int i = 0; i < kRow / 32; ++i) {
        if (!MX8) k[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(page)[at * kRow + lane + 32 * i]);
        else if (i < kLatent / 32) {
          unsigned lo, hi;
          mx8_to_bf16x4(page[at * kLatent + lane + 32 * i], ue8m0_value(page[kPageScales + at * 16 + i]), lo, hi);
          k[i] = bf_lo(lo);
        } else k[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(page + kPageRope)[at * kRopeCols + lane + 32 * (i - kLatent / 32)]);
      }
      float x = 0.f;
      for (int i = 0; i < kRow / 32; ++i) x = fmaf(q[i], k[i], x);
      x = butterfly_sum<32>(x) * a.scale;
      const float mm = fmaxf(m, x), f = m == -INFINITY ? 0.f : expf(m - mm);
      const float p = isfinite(x) ? expf(x - mm) : NAN;          // a token that is not finite spoils the rows that see it
      m = mm;
      l = l * f + p;
      for (int i = 0; i < kLatent / 32; ++i) o[i] = o[i] * f + p * k[i];
    }
  }
  for (int i = 0; i < kLatent / 32; ++i) a.out[row * kLatent + lane + 32 * i] = __float2bfloat16_rn(l == 0.f ? 0.f : o[i] / l);
}

}  // namespace

K3G_API int k3g_latent_attn_workspace(int B, int S, int heads, long long* host_bytes) {
  K3G_REQUIRE_PTR(host_bytes);
  K3G_REQUIRE(B > 0 && S > 0 && heads > 0, K3G_ESHAPE);
  K3G_REQUIRE(B <= kMaxBatch && (long long)S * heads <= kMaxRowsPerSeq, K3G_ELIMIT);
  *host_bytes = 16;
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
  long long need = 0;
  const int rc = k3g_latent_attn_workspace(B, S, heads, &need);
  if (rc != K3G_OK) return rc;
  K3G_REQUIRE(prefix_pages <= (1 << 20) && max_pages <= (1 << 20), K3G_ELIMIT);
  K3G_REQUIRE(workspace_bytes >= need, K3G_EWORKSPACE);
  AttnArgs a = {(const __nv_bfloat16*)q, q_stride, (const unsigned char*)cache + layer_off * unit, page_stride * unit, pages,
                (const int*)prefix_table, (const int*)prefix_len, prefix_pages, (const int*)block_table, (const int*)lens, max_pages,
                (__nv_bfloat16*)out, B, S, heads, scale};
  const unsigned grid = (unsigned)(((long long)B * S * heads + 3) / 4);
  if (cache_mx8) latent_attn_simple_kernel<true><<<grid, 128, 0, k3g_stream(stream)>>>(a);
  else latent_attn_simple_kernel<false><<<grid, 128, 0, k3g_stream(stream)>>>(a);
  return k3g_launch_status();
}
