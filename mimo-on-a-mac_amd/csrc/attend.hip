// Attention of a step's new tokens over the paged K/V cache (mimo_cache_attend).
#include "cache.h"
#include "device.h"

namespace mimo {

struct AttendArgs {
  const uint16_t* q;
  int64_t q_stride;
  int N, Hq, Hkv, G, Dk, Dv, B, max_pages, n_pages, page_shift, window, sinks;
  const int32_t *starts, *lens, *table;
  const void *k, *v;
  const float *k_scale, *v_scale, *sink_logits;
  float scale;
  uint16_t* out;
  int32_t* status;
};

// The simple form: one block per (token, head), each wave takes every fourth key, lanes along the head dimension.
template <bool E4M3>
__global__ void __launch_bounds__(256) attend_simple_kernel(AttendArgs a) {
  const int n = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint16_t* o = a.out + ((size_t)n * a.Hq + h) * a.Dv;
  int lo = 0, hi = a.B;                              // the last request that starts at or before n
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.starts[mid] <= n) lo = mid; else hi = mid;
  }
  const int b = lo, s0 = a.starts[b], s1 = a.starts[b + 1], len = a.lens[b];
  const bool mine = n >= s0 && n < s1;
  const bool bad = mine && (len < s1 - s0 || len > (a.max_pages << a.page_shift));
  if (!mine || bad) {
    if (bad && a.status && threadIdx.x == 0) a.status[0] = MIMO_ERR_SHAPE;
    for (int d = threadIdx.x; d < a.Dv; d += 256) o[d] = 0;
    return;
  }
  const int p = len - s1 + n, kv = h / a.G;
  const float ks = E4M3 ? a.k_scale[kv] : 1.0f, vs = E4M3 ? a.v_scale[kv] : 1.0f;
  float q[3], acc[2] = {0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
  const int nk = a.Dk / 64, nv = a.Dv / 64;
  for (int c = 0; c < 3; ++c) q[c] = c < nk ? bf16_to_f32(a.q[n * a.q_stride + h * a.Dk + 64 * c + lane]) : 0.0f;
  auto load = [&](const void* base, size_t at) {
    if constexpr (E4M3) return e4m3_unpack2(static_cast<const uint8_t*>(base)[at]).x;
    else return bf16_to_f32(static_cast<const uint16_t*>(base)[at]);
  };
  for (int j = wave; j <= p; j += 4) {
    if (a.window && p - j >= a.window && j >= a.sinks) continue;
    int id = a.table[(size_t)b * a.max_pages + (j >> a.page_shift)];
    if (id < 0 || id >= a.n_pages) {
      if (a.status && lane == 0) a.status[0] = MIMO_ERR_SLOT;
      id = 0;
    }
    const size_t row = ((((size_t)id * a.Hkv + kv) << a.page_shift)) + (j & ((1 << a.page_shift) - 1));
    float s = 0.0f;
    for (int c = 0; c < nk; ++c) s += q[c] * load(a.k, row * a.Dk + 64 * c + lane);
    s = dpp_sum_f32(s) * ks * a.scale;
    const float top = fmaxf(m, s), was = m == top ? 1.0f : __expf(m - top), w = s == top && s != -INFINITY ? 1.0f : (s == -INFINITY ? 0.0f : __expf(s - top));
    l = l * was + w;
    for (int c = 0; c < nv; ++c) acc[c] = acc[c] * was + w * load(a.v, row * a.Dv + 64 * c + lane);
    m = top;
  }
  __shared__ float sm[4], sl[4], sa[4][128];
  if (lane == 0) sm[wave] = m, sl[wave] = l;
  sa[wave][lane] = acc[0];
  sa[wave][64 + lane] = acc[1];
  __syncthreads();
  const float sink = a.sink_logits ? a.sink_logits[h] : -INFINITY;
  const float top = fmaxf(fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), sink);
  float tot = sink == -INFINITY ? 0.0f : __expf(sink - top);
  for (int w = 0; w < 4; ++w) tot += sm[w] == -INFINITY ? 0.0f : sl[w] * __expf(sm[w] - top);
  for (int d = threadIdx.x; d < a.Dv; d += 256) {
    float x = 0.0f;
    for (int w = 0; w < 4; ++w) x += sm[w] == -INFINITY ? 0.0f : sa[w][d] * __expf(sm[w] - top);
    o[d] = tot == 0.0f ? 0 : f32_to_bf16(x * vs / tot);
  }
}

}  // namespace mimo

using namespace mimo;

extern "C" {

size_t mimo_cache_attend_workspace_size(int N, int heads, int kv_heads, int v_dim) {
  if (N < 0 || heads < 1 || kv_heads < 1 || v_dim < 1) return 0;
  return 256;
}

int mimo_cache_attend(const uint16_t* q, int64_t q_stride, int N, int heads, const mimo_kv_cache* cache, int B,
                      const int32_t* starts, const int32_t* lens, const int32_t* table, int max_pages, int max_new, float scale,
                      int window, int sink_tokens, const float* sink_logits, uint16_t* out, int32_t* status, void* ws,
                      size_t ws_bytes, void* stream) {
  if (int e = check_cache(cache, "cache_attend")) return e;
  MIMO_REQUIRE(N >= 0 && N <= (1 << 20), MIMO_ERR_SHAPE, "cache_attend: %d tokens (0 to 2^20)", N);
  if (N == 0) return MIMO_OK;
  MIMO_REQUIRE(q && starts && lens && table && out, MIMO_ERR_ARG, "cache_attend: null pointer");
  MIMO_REQUIRE(heads >= 1 && heads % cache->kv_heads == 0 && heads <= 1024, MIMO_ERR_SHAPE,
               "cache_attend: %d heads on %d K/V heads (a multiple, at most 1024)", heads, cache->kv_heads);
  MIMO_REQUIRE(B >= 1 && B <= (1 << 20) && max_pages >= 1 && max_new >= 0 && (int64_t)max_pages * cache->page_size <= 0x7fffffff,
               MIMO_ERR_SHAPE, "cache_attend: need 1 <= B <= 2^20, max_pages >= 1, max_new >= 0 (got %d, %d, %d)", B, max_pages, max_new);
  MIMO_REQUIRE(window >= 0 && sink_tokens >= 0, MIMO_ERR_SHAPE, "cache_attend: window and sink_tokens must be >= 0");
  MIMO_REQUIRE(scale == scale && scale - scale == 0.0f, MIMO_ERR_ARG, "cache_attend: scale must be finite");
  MIMO_REQUIRE(q_stride >= (int64_t)heads * cache->k_dim, MIMO_ERR_SHAPE, "cache_attend: rows closer than their length");
  MIMO_REQUIRE(aligned16(q) && aligned16(out) && q_stride % 8 == 0, MIMO_ERR_ALIGN,
               "cache_attend: 16-byte alignment of q, its rows and out");
  const size_t need = mimo_cache_attend_workspace_size(N, heads, cache->kv_heads, cache->v_dim);
  MIMO_REQUIRE(ws && ws_bytes >= need, MIMO_ERR_WORKSPACE, "cache_attend: workspace %zu < %zu", ws_bytes, need);
  MIMO_REQUIRE(aligned16(ws), MIMO_ERR_ALIGN, "cache_attend: 16-byte alignment of the workspace");
  AttendArgs a{q, q_stride, N, heads, cache->kv_heads, heads / cache->kv_heads, cache->k_dim, cache->v_dim, B, max_pages,
               cache->n_pages, __builtin_ctz(cache->page_size), window, sink_tokens, starts, lens, table, cache->k, cache->v,
               cache->k_scale, cache->v_scale, sink_logits, scale, out, status};
  hipStream_t st = as_stream(stream);
  {
    ProfScope p(st, "cache_attend");
    if (cache->dtype == MIMO_KV_E4M3) attend_simple_kernel<true><<<dim3(N, heads), 256, 0, st>>>(a);
    else attend_simple_kernel<false><<<dim3(N, heads), 256, 0, st>>>(a);
  }
  return check_launch("cache_attend");
}

}  // extern "C"
