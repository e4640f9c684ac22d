// The paged K/V cache: page tables and slots from request lengths (mimo_cache_step) and the write of new keys and values
// with their rotary positions (mimo_cache_append).  The reference keeps one request's caches as MLX arrays that grow
// (engine/mimo_stream/model.py:169-170) and rotates q and k in its Attention (engine/mimo_stream/mimo_v2.py:110-150);
// here many requests share one pool of pages and no length ever goes to the host.
#include "cache.h"

#include "device.h"
#include "host.h"

namespace mimo {

// ------------------------------------------------------------------ step
// B requests go from lens to target tokens.  new = max(0, target - lens), starts = its exclusive scan; with
// pages(l) = ceil(l / page), a request gives back pages pages(target) .. pages(lens) - 1 or takes as many as it grows by.
// Both lists run over the requests in order and each request's pages in order: F[i], the i-th page given back, goes to
// place n_free + freed - 1 - i of the free stack, and T[j], the j-th page taken, comes from place n_free + freed - 1 - j:
// T[j] = F[j] while j < freed, else free[n_free - 1 - (j - freed)].  So a step that is taken back restores the stack, and
// places below n_free are only read, places from n_free on only written: no order between blocks matters.
//
// Every block scans all requests for itself (a few KB from L2), so that one launch does the whole step and the blocks share
// tokens, table entries and returned pages.  A token in a page taken in this step gets its page from T directly.
//
// Bound by latency, not by its bytes (6 KB and 1 MB): the requests' lengths, three block-wide scans side by side (wave prefix
// sums by row shifts, no LDS loop), a search of 8 to 12 LDS reads per token, its page.  256 decoding requests 5.2 us, an empty
// launch of which is 3; 1024 requests with 49219 new tokens 9.7 us in 49 blocks (74 in one block, 11.4 with scans in LDS).
constexpr int ST_THREADS = 1024;
constexpr int ST_MAX_REQS = 4096;
constexpr int ST_MAX_TOKENS = 1 << 20;              // the scan's 1024 partial sums of at most this stay below 2^31

struct StepArgs {
  const int32_t *lens, *target, *n_free;
  int32_t *table, *free_pages;
  int B, max_pages, n_pages, page_shift, N, max_new;
  int32_t *lens_out, *n_free_out, *starts, *slots, *positions, *status;
  int32_t *commit_lens, *commit_n_free;             // null unless a single block runs and the new state replaces the old
};

// Exclusive scan of one value per thread over the block's 1024 threads, for three values at once; totals in tot[3].
__device__ __forceinline__ void st_scan3(int v[3], int tot[3], int* sh) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int inc[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    inc[q] = dpp_prefix_i32(v[q]);
    if (lane == 63) sh[16 * q + wave] = inc[q];
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    const int before = dpp_prefix_i32(lane < ST_THREADS / 64 ? sh[16 * q + lane] : 0);   // of the waves' sums
    v[q] = (wave ? __builtin_amdgcn_readlane(before, wave - 1) : 0) + inc[q] - v[q];
    tot[q] = __builtin_amdgcn_readlane(before, 63);
  }
  __syncthreads();
}

__global__ void __launch_bounds__(ST_THREADS) cache_step_kernel(StepArgs a) {
  __shared__ int scan_sh[48];
  __shared__ int s_bad;
  extern __shared__ int s_scans[];                   // the exclusive scans, B + 1 each
  const int t = threadIdx.x, B = a.B, sh = a.page_shift;
  int *s_new = s_scans, *s_free = s_new + B + 1, *s_take = s_free + B + 1;
  const int per = (B + ST_THREADS - 1) / ST_THREADS;
  const int b0 = min(B, t * per), b1 = min(B, b0 + per);
  const int cap = min(a.max_pages, 0x7fffffff >> sh) << sh;
  if (t == 0) s_bad = 0;
  __syncthreads();
  auto pages = [&](int l) { return (l >> sh) + ((l & ((1 << sh) - 1)) != 0); };
  const int n_free = a.n_free[0];
  int v[3] = {0, 0, 0}, tot[3];
  bool bad = n_free < 0 || n_free > a.n_pages;
  long long wide = 0;                                // new tokens in 64 bits: 32 may wrap for invalid lengths
  for (int b = b0; b < b1; ++b) {
    const int l = a.lens[b], g = a.target[b];
    const bool ok = l >= 0 && l <= cap && g >= 0 && g <= cap && g - l <= a.max_new;
    bad |= !ok;
    if (!ok) continue;
    wide += max(0, g - l);
    v[0] = (int)min(wide, (long long)a.N + 1);
    v[1] += max(0, pages(l) - pages(g));
    v[2] += max(0, pages(g) - pages(l));
  }
  if (bad) s_bad = MIMO_ERR_SHAPE;
  st_scan3(v, tot, scan_sh);
  for (int b = b0; b < b1; ++b) {
    s_new[b] = v[0], s_free[b] = v[1], s_take[b] = v[2];
    if (s_bad) continue;
    const int l = a.lens[b], g = a.target[b];
    v[0] += max(0, g - l);
    v[1] += max(0, pages(l) - pages(g));
    v[2] += max(0, pages(g) - pages(l));
  }
  if (t == 0) s_new[B] = tot[0], s_free[B] = tot[1], s_take[B] = tot[2];
  __syncthreads();
  const int freed = tot[1], taken = tot[2];
  int status = s_bad;
  if (!status && tot[0] > a.N) status = MIMO_ERR_SHAPE;
  if (!status && (long long)taken - freed > n_free) status = MIMO_ERR_PAGES;
  if (!status && (long long)n_free + freed - taken > a.n_pages) status = MIMO_ERR_SHAPE;
  const bool first = blockIdx.x == 0;
  if (status) {                                      // nothing moves: no new tokens, lengths and the stack as they were
    if (first) {
      for (int b = t; b <= B; b += ST_THREADS) {
        a.starts[b] = 0;
        if (b < B) a.lens_out[b] = a.lens[b];
      }
      if (t == 0) a.n_free_out[0] = n_free, a.status[0] = status;
    }
    for (int n = blockIdx.x * ST_THREADS + t; n < a.N; n += gridDim.x * ST_THREADS) a.slots[n] = -1, a.positions[n] = 0;
    return;
  }
  // the request whose exclusive scan holds i: the last b with scan[b] <= i
  auto owner = [&](const int* scan, int i) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (scan[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
  };
  auto released = [&](int i) {                       // F[i]
    const int b = owner(s_free, i);
    return a.table[(size_t)b * a.max_pages + pages(a.target[b]) + (i - s_free[b])];
  };
  auto fresh = [&](int j) { return j < freed ? released(j) : a.free_pages[n_free - 1 - (j - freed)]; };   // T[j]
  for (int n = blockIdx.x * ST_THREADS + t; n < a.N; n += gridDim.x * ST_THREADS) {
    int slot = -1, pos = 0;
    if (n < tot[0]) {
      const int b = owner(s_new, n), l = a.lens[b];
      pos = l + n - s_new[b];
      const int pi = pos >> sh, had = pages(l);
      const int id = pi < had ? a.table[(size_t)b * a.max_pages + pi] : fresh(s_take[b] + pi - had);
      if (id >= 0 && id < a.n_pages) slot = (id << sh) + (pos & ((1 << sh) - 1));
    }
    a.slots[n] = slot;
    a.positions[n] = pos;
  }
  const int from = blockIdx.x * ST_THREADS + t, all = gridDim.x * ST_THREADS;
  for (int j = from; j < taken; j += all) {
    const int b = owner(s_take, j);
    a.table[(size_t)b * a.max_pages + pages(a.lens[b]) + (j - s_take[b])] = fresh(j);
  }
  for (int i = from; i < freed - taken; i += all) a.free_pages[n_free + i] = released(freed - 1 - i);
  if (!first) return;
  for (int b = t; b <= B; b += ST_THREADS) a.starts[b] = s_new[b];
  if (a.commit_lens) __syncthreads();                // every read of the old lengths is done
  for (int b = t; b < B; b += ST_THREADS) {
    const int g = a.target[b];
    a.lens_out[b] = g;
    if (a.commit_lens) a.commit_lens[b] = g;
  }
  if (t == 0) {
    a.n_free_out[0] = n_free + freed - taken;
    if (a.commit_lens) a.commit_n_free[0] = n_free + freed - taken;
    a.status[0] = MIMO_OK;
  }
}

// lens = lens_out, n_free = n_free_out after a step over many blocks: 1.6 us (1024 requests), 1.9 more in a graph
__global__ void __launch_bounds__(256) cache_commit_kernel(const int32_t* from, int32_t* lens, int B, const int32_t* nf_from,
                                                           int32_t* n_free) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < B) lens[b] = from[b];
  if (b == 0) n_free[0] = nf_from[0];
}

// ------------------------------------------------------------------ append
// Bound by HBM for many tokens, by its launch for few.  4096 tokens of 64 q and 8 K/V heads (243 MB) 52 us, 4.7 TB/s, a large
// copy's rate (39.4 us again and again on the same rows, which the last-level cache holds in part); 1777 tokens into E4M3 10.1
// us (4 TB/s: 7 blocks on a CU in all, the start counts); 64 tokens 3.5 us.  One pass: q, k and v are read and written once, in 16-byte pieces (a pair of them where they rotate).
//
// Angles are pos * turn_i turns in 64 bits (a position of 131072 times a first frequency of 1 / 2 pi leaves 32 bits with
// no useful fraction), reduced to a fraction of a turn before the 32-bit sine and cosine; one rotation is
// (x_i cos - x_{i + r/2} sin, x_{i + r/2} cos + x_i sin) in 32 bits, rounded once to what is stored.
struct AppendArgs {
  const uint16_t *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;             // elements between two tokens
  int Hq, Hkv, Dk, Dv, N, rot;
  const double* turns;
  const int32_t *positions, *slots;
  uint16_t* q_out;
  void *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  int page_shift, n_slots;
  int32_t* status;
};

constexpr int AP_MAX_ROT = 256;
// Blocks that the card holds at once: up to that many are made of few tokens.  64 tokens 3.5 us, 512 tokens 7.7; with 512
// blocks 4.2 and 9.4; with 8192 no change.
constexpr int AP_BLOCKS = 2048;

__device__ __forceinline__ void ap_unpack(uint4 x, float* f) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}
__device__ __forceinline__ uint4 ap_pack(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)f32_to_bf16(f[2 * i]) | ((uint32_t)f32_to_bf16(f[2 * i + 1]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// E4M3 of x / scale, clamped to +-448 (NaN stays NaN): the hardware conversion rounds to nearest even
__device__ __forceinline__ float ap_clamp(float x) { return x > 448.0f ? 448.0f : (x < -448.0f ? -448.0f : x); }
__device__ __forceinline__ uint2 ap_pack_e4m3(const float* f, float scale) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(ap_clamp(f[4 * i] / scale), ap_clamp(f[4 * i + 1] / scale), 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(ap_clamp(f[4 * i + 2] / scale), ap_clamp(f[4 * i + 3] / scale), r, true);
    w[i] = (uint32_t)r;
  }
  return make_uint2(w[0], w[1]);
}

// A token is gridDim.y blocks of 256 threads, a thread one unit of 8 values (of a pair, two) at a time; the first unit is on
// its way while the token's angles are worked out.
template <bool E4M3>
__global__ void __launch_bounds__(256) cache_append_kernel(AppendArgs a) {
#pragma clang fp contract(off)
  __shared__ float s_cos[AP_MAX_ROT / 2], s_sin[AP_MAX_ROT / 2];
  const int n = blockIdx.x, half = a.rot >> 1;
  const int pos = a.positions[n], slot = a.slots[n];
  const bool keep = slot >= 0 && slot < a.n_slots;
  if (slot >= a.n_slots && threadIdx.x == 0 && a.status) a.status[0] = MIMO_ERR_SLOT;
  // units of 8 values: per q and k head rot / 16 pairs of units and (Dk - rot) / 8 units that stay, then v
  const int pairs = a.rot >> 4, U = pairs + ((a.Dk - a.rot) >> 3), Uv = a.Dv >> 3;
  const int nq = a.q ? a.Hq * U : 0, nk = a.Hkv * U, all = keep ? nq + nk + a.Hkv * Uv : nq;
  struct Unit {
    int kind, h, d;                                        // 0 q, 1 k, 2 v; head; first dimension
    bool pair;
    uint4 x, y;
  };
  auto load = [&](int u) __attribute__((always_inline)) {
    Unit r;
    r.kind = u < nq ? 0 : (u < nq + nk ? 1 : 2);
    const int w = r.kind == 0 ? u : (r.kind == 1 ? u - nq : u - nq - nk), per = r.kind == 2 ? Uv : U;
    r.h = w / per;
    const int c = w - r.h * per;
    r.pair = r.kind != 2 && c < pairs;
    r.d = r.kind == 2 || r.pair ? 8 * c : a.rot + 8 * (c - pairs);
    const uint16_t* row = r.kind == 0 ? a.q + n * a.q_stride + r.h * a.Dk : (r.kind == 1 ? a.k + n * a.k_stride + r.h * a.Dk : a.v + n * a.v_stride + r.h * a.Dv);
    r.x = *reinterpret_cast<const uint4*>(row + r.d);
    r.y = make_uint4(0, 0, 0, 0);
    if (r.pair) r.y = *reinterpret_cast<const uint4*>(row + r.d + half);
    return r;
  };
  int u = blockIdx.y * 256 + threadIdx.x;
  Unit first{};
  if (u < all) first = load(u);
  for (int i = threadIdx.x; i < half; i += 256) {
    const double t = (double)pos * a.turns[i];
    const float f = (float)(t - floor(t));
    float sn, cs;
    sincospif(2.0f * f, &sn, &cs);
    s_cos[i] = cs, s_sin[i] = sn;
  }
  __syncthreads();
  const int mask = (1 << a.page_shift) - 1;
  const size_t prow = keep ? ((size_t)(slot >> a.page_shift) * a.Hkv << a.page_shift) + (slot & mask) : 0;
  auto put = [&](void* pages, int h, int D, int d, const float* f, const float* scale) {
    const size_t at = (prow + ((size_t)h << a.page_shift)) * D + d;
    if constexpr (E4M3) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pages) + at) = ap_pack_e4m3(f, scale[h]);
    else *reinterpret_cast<uint4*>(static_cast<uint16_t*>(pages) + at) = ap_pack(f);
  };
  for (bool again = false; u < all; u += gridDim.y * 256, again = true) {
    const Unit r = again ? load(u) : first;
    float x[8], y[8];
    ap_unpack(r.x, x);
    if (r.kind == 2) {
      put(a.v_pages, r.h, a.Dv, r.d, x, a.v_scale);
      continue;
    }
    if (r.pair) {
      ap_unpack(r.y, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float cs = s_cos[r.d + i], sn = s_sin[r.d + i], p = x[i], q = y[i];
        x[i] = p * cs - q * sn;
        y[i] = q * cs + p * sn;
      }
    }
    if (r.kind == 0) {
      uint16_t* o = a.q_out + ((size_t)n * a.Hq + r.h) * a.Dk + r.d;
      *reinterpret_cast<uint4*>(o) = ap_pack(x);
      if (r.pair) *reinterpret_cast<uint4*>(o + half) = ap_pack(y);
    } else {
      put(a.k_pages, r.h, a.Dk, r.d, x, a.k_scale);
      if (r.pair) put(a.k_pages, r.h, a.Dk, r.d + half, y, a.k_scale);
    }
  }
}

int check_cache(const mimo_kv_cache* c, const char* what) {
  MIMO_REQUIRE(c && c->k && c->v, MIMO_ERR_ARG, "%s: null pointer", what);
  MIMO_REQUIRE(c->dtype == MIMO_KV_BF16 || c->dtype == MIMO_KV_E4M3, MIMO_ERR_ARG, "%s: cache dtype %d", what, c->dtype);
  MIMO_REQUIRE(c->dtype == MIMO_KV_BF16 || (c->k_scale && c->v_scale), MIMO_ERR_ARG, "%s: an E4M3 cache needs k_scale and v_scale", what);
  MIMO_REQUIRE((c->k_dim == 64 && c->v_dim == 64) || (c->k_dim == 128 && c->v_dim == 128) || (c->k_dim == 192 && c->v_dim == 128),
               MIMO_ERR_SHAPE, "%s: head dimensions %d / %d (64/64, 128/128 and 192/128 are supported)", what, c->k_dim, c->v_dim);
  MIMO_REQUIRE(c->page_size >= 16 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0, MIMO_ERR_SHAPE,
               "%s: page_size %d (a power of two from 16 to 1024)", what, c->page_size);
  MIMO_REQUIRE(c->kv_heads >= 1 && c->kv_heads <= 1024, MIMO_ERR_SHAPE, "%s: kv_heads %d", what, c->kv_heads);
  MIMO_REQUIRE(c->n_pages >= 1 && (int64_t)c->n_pages * c->page_size <= 0x7fffffff, MIMO_ERR_SHAPE,
               "%s: %d pages of %d (at most 2^31 - 1 slots)", what, c->n_pages, c->page_size);
  MIMO_REQUIRE(aligned16(c->k) && aligned16(c->v), MIMO_ERR_ALIGN, "%s: 16-byte alignment", what);
  return MIMO_OK;
}

}  // namespace mimo

using namespace mimo;

extern "C" {

int mimo_cache_step(const int32_t* lens, const int32_t* target, int B, int32_t* table, int max_pages, int32_t* free_pages,
                    const int32_t* n_free, int n_pages, int page_size, int N, int max_new, int32_t* lens_out,
                    int32_t* n_free_out, int32_t* starts, int32_t* slots, int32_t* positions, int32_t* commit_lens,
                    int32_t* commit_n_free, int32_t* status, void* stream) {
  MIMO_REQUIRE(lens && target && table && free_pages && n_free && lens_out && n_free_out && starts && status, MIMO_ERR_ARG,
               "cache_step: null pointer");
  MIMO_REQUIRE(N == 0 || (slots && positions), MIMO_ERR_ARG, "cache_step: null pointer");
  MIMO_REQUIRE(B >= 1 && B <= ST_MAX_REQS, MIMO_ERR_SHAPE, "cache_step: %d requests (1 to %d)", B, ST_MAX_REQS);
  MIMO_REQUIRE(N <= ST_MAX_TOKENS, MIMO_ERR_SHAPE, "cache_step: %d tokens (at most %d)", N, ST_MAX_TOKENS);
  MIMO_REQUIRE(N >= 0 && max_new >= 0 && max_pages >= 1 && n_pages >= 1, MIMO_ERR_SHAPE,
               "cache_step: need N, max_new >= 0 and max_pages, n_pages >= 1 (got %d, %d, %d, %d)", N, max_new, max_pages, n_pages);
  MIMO_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0, MIMO_ERR_SHAPE,
               "cache_step: page_size %d (a power of two from 16 to 1024)", page_size);
  MIMO_REQUIRE((int64_t)n_pages * page_size <= 0x7fffffff && (int64_t)max_pages * page_size <= kMaxTokens &&
                   (int64_t)max_pages * B <= 0x7fffffff, MIMO_ERR_SHAPE,
               "cache_step: at most 2^31 - 1 slots and table entries, 2^31 - 2^16 tokens of a request");
  MIMO_REQUIRE(lens_out != lens && n_free_out != n_free, MIMO_ERR_ARG, "cache_step: lens_out and n_free_out may not alias the state");
  MIMO_REQUIRE(!commit_lens == !commit_n_free, MIMO_ERR_ARG, "cache_step: commit_lens and commit_n_free go together");
  StepArgs a{lens, target, n_free, table, free_pages, B, max_pages, n_pages, __builtin_ctz(page_size), N, max_new,
             lens_out, n_free_out, starts, slots, positions, status, nullptr, nullptr};
  const int blocks = std::max(1, std::min(256, (N + ST_THREADS - 1) / ST_THREADS));
  if (blocks == 1) a.commit_lens = commit_lens, a.commit_n_free = commit_n_free;
  hipStream_t st = as_stream(stream);
  {
    ProfScope p(st, "cache_step");
    cache_step_kernel<<<blocks, ST_THREADS, 3 * (B + 1) * sizeof(int), st>>>(a);
  }
  if (int e = check_launch("cache_step")) return e;
  if (commit_lens && blocks > 1) {
    ProfScope p(st, "cache_commit");
    cache_commit_kernel<<<(B + 255) / 256, 256, 0, st>>>(lens_out, commit_lens, B, n_free_out, commit_n_free);
    return check_launch("cache_commit");
  }
  return MIMO_OK;
}

int mimo_cache_append(const uint16_t* q, int64_t q_stride, int heads, const uint16_t* k, int64_t k_stride, const uint16_t* v,
                      int64_t v_stride, int N, const int32_t* positions, const int32_t* slots, const mimo_kv_cache* cache,
                      int rotary_dim, const double* turns, uint16_t* q_out, int32_t* status, void* stream) {
  if (int e = check_cache(cache, "cache_append")) return e;
  MIMO_REQUIRE(N >= 0 && N <= kMaxBlocks, MIMO_ERR_SHAPE, "cache_append: %d tokens (0 to 2^24 - 1)", N);
  if (N == 0) return MIMO_OK;
  MIMO_REQUIRE(k && v && positions && slots, MIMO_ERR_ARG, "cache_append: null pointer");
  MIMO_REQUIRE(!q == !q_out, MIMO_ERR_ARG, "cache_append: q and q_out go together");
  MIMO_REQUIRE(!q || (heads >= 1 && heads <= 65536), MIMO_ERR_SHAPE, "cache_append: %d heads", heads);
  MIMO_REQUIRE(rotary_dim >= 0 && rotary_dim % 16 == 0 && rotary_dim <= cache->k_dim, MIMO_ERR_SHAPE,
               "cache_append: rotary_dim %d (a multiple of 16 up to k_dim)", rotary_dim);
  MIMO_REQUIRE(rotary_dim == 0 || turns, MIMO_ERR_ARG, "cache_append: null pointer");
  MIMO_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) &&
                   (q_stride | k_stride | v_stride) % 8 == 0, MIMO_ERR_ALIGN,
               "cache_append: 16-byte alignment of q, k, v and of their rows");
  const int64_t kn = (int64_t)cache->kv_heads * cache->k_dim, vn = (int64_t)cache->kv_heads * cache->v_dim;
  MIMO_REQUIRE(k_stride >= kn && v_stride >= vn && (!q || q_stride >= (int64_t)heads * cache->k_dim), MIMO_ERR_SHAPE,
               "cache_append: rows closer than their length");
  if (q) {
    const size_t out = (size_t)N * heads * cache->k_dim * 2;
    MIMO_REQUIRE(!overlap(q, ((size_t)(N - 1) * q_stride + (size_t)heads * cache->k_dim) * 2, q_out, out) &&
                     !overlap(k, ((size_t)(N - 1) * k_stride + kn) * 2, q_out, out) && !overlap(v, ((size_t)(N - 1) * v_stride + vn) * 2, q_out, out),
                 MIMO_ERR_ARG, "cache_append: q_out may not overlap q, k or v");
  }
  AppendArgs a{q, k, v, q_stride, k_stride, v_stride, heads, cache->kv_heads, cache->k_dim, cache->v_dim, N, rotary_dim, turns,
               positions, slots, q_out, cache->k, cache->v, cache->k_scale, cache->v_scale, __builtin_ctz(cache->page_size),
               cache->n_pages * cache->page_size, status};
  hipStream_t st = as_stream(stream);
  {
    ProfScope p(st, "cache_append");
    // few tokens are spread over several blocks each
    const int units = ((q ? heads : 0) * (cache->k_dim - rotary_dim / 2) + cache->kv_heads * (cache->k_dim - rotary_dim / 2 + cache->v_dim)) / 8;
    const dim3 grid(N, std::max(1, std::min((units + 255) / 256, AP_BLOCKS / N)));
    if (cache->dtype == MIMO_KV_E4M3) cache_append_kernel<true><<<grid, 256, 0, st>>>(a);
    else cache_append_kernel<false><<<grid, 256, 0, st>>>(a);
  }
  return check_launch("cache_append");
}

}  // extern "C"
