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
// us (4 TB/s: 7 blocks on a CU in all, the start counts); 64 tokens 3.5 us.  One pass: q, k and v are read and written once,
// in 16-byte pieces (a pair of them where they rotate).
//
// Angles are pos * turn_i turns in 64 bits (a position of 131072 times a first frequency of 1 / 2 pi leaves 32 bits with
// no useful fraction), reduced to a fraction of a turn before the 32-bit sine and cosine; one rotation is
// (x_i cos - x_{i + r/2} sin, x_{i + r/2} cos + x_i sin) in 32 bits, rounded once to what is stored.
struct AppendArgs {
  const uint16_t *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;             // elements between two tokens
  int Hq, Hkv, Dk, Dv, N, rot;
  const double* turns;
  float magnitude;
  const int32_t *positions, *slots;
  uint16_t* q_out;
  void *k_pages, *v_pages;
  const void *k_scale, *v_scale;                    // fp32 [Hkv], or the bytes of a cache with block scales
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

// one rotation of eight pairs (x_i, y_i), of four pairs (x_2i, x_2i+1)
__device__ __forceinline__ void ap_turn(float* x, float* y, const float* cs, const float* sn) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float p = x[i], q = y[i];
    x[i] = p * cs[i] - q * sn[i];
    y[i] = q * cs[i] + p * sn[i];
  }
}
__device__ __forceinline__ void ap_turn_side(float* x, const float* cs, const float* sn) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float p = x[2 * i], q = x[2 * i + 1];
    x[2 * i] = p * cs[i] - q * sn[i];
    x[2 * i + 1] = q * cs[i] + p * sn[i];
  }
}

// Part `part` of `parts` of token n (its q alone where KIND is AP_Q): 256 threads, a thread one unit of 8 values (of a pair of
// units, two) at a time; the first unit is on its way while the token's angles are worked out.  SIDE: the rotated pairs lie
// side by side (2 i, 2 i + 1), so that a unit holds four of them; else unit d is turned with unit d + rot / 2.
enum { AP_BF16, AP_E4M3, AP_Q };
template <int KIND, bool SIDE>
__device__ __forceinline__ void ap_token(const AppendArgs& a, int n, int part, int parts, float* s_cos, float* s_sin) {
#pragma clang fp contract(off)
  const int half = a.rot >> 1;
  const int pos = a.positions[n], slot = KIND == AP_Q ? -1 : a.slots[n];
  const bool keep = slot >= 0 && slot < a.n_slots;
  if (slot >= a.n_slots && threadIdx.x == 0 && a.status) a.status[0] = MIMO_ERR_SLOT;
  // units of 8 values: per q and k head rot / 16 pairs of units and (Dk - rot) / 8 units that stay, then v
  const int pairs = SIDE ? 0 : a.rot >> 4, U = SIDE ? a.Dk >> 3 : pairs + ((a.Dk - a.rot) >> 3), Uv = a.Dv >> 3;
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
    r.d = SIDE || r.kind == 2 || r.pair ? 8 * c : a.rot + 8 * (c - pairs);
    const uint16_t* row = r.kind == 0 ? a.q + n * a.q_stride + r.h * a.Dk : (r.kind == 1 ? a.k + n * a.k_stride + r.h * a.Dk : a.v + n * a.v_stride + r.h * a.Dv);
    r.x = *reinterpret_cast<const uint4*>(row + r.d);
    r.y = make_uint4(0, 0, 0, 0);
    if (r.pair) r.y = *reinterpret_cast<const uint4*>(row + r.d + half);
    return r;
  };
  int u = part * 256 + threadIdx.x;
  Unit first{};
  if (u < all) first = load(u);
  for (int i = threadIdx.x; i < half; i += 256) {
    const double t = (double)pos * a.turns[i];
    const float f = (float)(t - floor(t));
    float sn, cs;
    sincospif(2.0f * f, &sn, &cs);
    s_cos[i] = cs * a.magnitude, s_sin[i] = sn * a.magnitude;
  }
  __syncthreads();
  const int mask = (1 << a.page_shift) - 1;
  const size_t prow = keep ? ((size_t)(slot >> a.page_shift) * a.Hkv << a.page_shift) + (slot & mask) : 0;
  auto put = [&](void* pages, int h, int D, int d, const float* f, const void* scale) {
    const size_t at = (prow + ((size_t)h << a.page_shift)) * D + d;
    if constexpr (KIND == AP_E4M3) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pages) + at) = ap_pack_e4m3(f, static_cast<const float*>(scale)[h]);
    else *reinterpret_cast<uint4*>(static_cast<uint16_t*>(pages) + at) = ap_pack(f);
  };
  for (bool again = false; u < all; u += parts * 256, again = true) {
    const Unit r = again ? load(u) : first;
    float x[8], y[8];
    ap_unpack(r.x, x);
    if (r.kind == 2) {
      put(a.v_pages, r.h, a.Dv, r.d, x, a.v_scale);
      continue;
    }
    if (SIDE && r.d < a.rot) ap_turn_side(x, s_cos + r.d / 2, s_sin + r.d / 2);
    if (r.pair) {
      ap_unpack(r.y, y);
      ap_turn(x, y, s_cos + r.d, s_sin + r.d);
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

template <int KIND, bool SIDE>
__global__ void __launch_bounds__(256) cache_append_kernel(AppendArgs a) {
  __shared__ float s_cos[AP_MAX_ROT / 2], s_sin[AP_MAX_ROT / 2];
  ap_token<KIND, SIDE>(a, blockIdx.x, blockIdx.y, gridDim.y, s_cos, s_sin);
}

// ------------------------------------------------------------------ append with block scales
// A cache with block scales holds code * 2^(s - 127), with one byte s for K and one for V of each 16 slots (a block) and head.
// With the largest magnitude M that a call writes to a block, need = the smallest s with M <= 448 * 2^(s - 127), from 1 to
// 246 (448 * 2^119 is the largest value; past it values saturate, and an infinity does, while a NaN stays one).  A block whose
// first slot is among the written begins anew with s = need; in any other s = max(s, need), and where it grows the codes of
// the rows that the call does not write are taken times 2^(old - new).  Powers of two make that exact but for codes that
// leave E4M3's normal range (2^-9 of the new scale at the coarsest), so a block holds the same whether it was written token by
// token or at once, and the reader's conversion to bf16 takes the scale for nothing.
//
// The rows of a call that belong to one block stand together (a request's tokens do): the first of them is found by looking at
// the row before, and the waves that look at it write the whole block: each head's K or V rotated in registers, M, the codes.
// One launch with the q rows, whose HBM time covers it: 4096 tokens of 64/8 heads (233 MB) 43.8 us, 5.3 TB/s, 37 without K and
// V and 12 without q.  1687 tokens in pieces of 24 prompts, 32/8 heads 14.1 us (8.2 and 12.6): 130 blocks of slots for each of
// 8 heads are a chain of round trips (slots, rows, stores), angles in 64 bits and the starts of 3400 blocks.  64 decoded tokens
// 4.5 us (these times are of the same tensors again and again; on three sets in turn 45.2, 15.4 and 5.2), also where every one of
// them raises its block's scales.
constexpr int SB_SHIFT = 4, SB_ROWS = 1 << SB_SHIFT;       // slots that share a scale
constexpr int SB_TOP = 246;
// Blocks that look for work: each is given as few rows as that leaves (1687 tokens in pieces of 24 prompts 14.1 us; 1024
// blocks 17.5, 4096 14.9; one of 4096 tokens 43.8, 42.6, 48.0: a block without work still costs its start).
constexpr int SB_BLOCKS = 2048;

// the byte that holds magnitudes up to M (an fp32's bits, finite)
__device__ __forceinline__ int sb_need(uint32_t M) {
  return min(max((int)(M >> 23) - ((M & 0x7FFFFFu) > 0x600000u ? 7 : 8), 1), SB_TOP);
}
// the largest magnitude of eight values and `most`: NaN left out; by bits, and only finite values
__device__ __forceinline__ float sb_size(const float* f, float most) {
#pragma unroll
  for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(f[i]));
  return most;
}
__device__ __forceinline__ uint32_t sb_finite_size(const float* f, uint32_t most) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(f[i]) & 0x7FFFFFFFu;
    most = max(most, u < 0x7F800000u ? u : 0u);
  }
  return most;
}
__device__ __forceinline__ float sb_power(int e) {         // 2^e, 2^-127 for less
  return exp2i(max(e, -127));
}
// E4M3 of f * inverse; `over`: some values may be past 448 and are clamped (the scale keeps the others below it)
__device__ __forceinline__ uint2 sb_pack(const float* f, float inverse, bool over) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = f[i] * inverse;
  if (over)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ap_clamp(x[i]);
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], r, true);
    w[i] = (uint32_t)r;
  }
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ uint32_t sb_rescale(uint32_t w, float by) {
  const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  const int r = __builtin_amdgcn_cvt_pk_fp8_f32(lo.x * by, lo.y * by, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hi.x * by, hi.y * by, r, true);
}

// The block that row n is the first of: part `part` of `parts` of its 2 Hkv units (a head's K or V).  Up to 4 rows are a wave's
// work, so that four units are in hand at once; more are shared by the four waves.  slots: lane l holds that of row n + l, 17
// of them.
constexpr int SB_HALF = 96;                                // pairs of a head of 192
struct RunRoom {
  float cos[SB_ROWS * SB_HALF], sin[SB_ROWS * SB_HALF];
  uint32_t most[2][4];
};
// A barrier for what is in LDS alone: loads and stores on their way to memory are not waited for.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
template <bool SIDE>
__device__ __forceinline__ void ap_run(const AppendArgs& a, int n, int slots, int part, int parts, RunRoom& room) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = a.rot >> 1;
  const int slot = __builtin_amdgcn_readfirstlane(slots);
  const uint64_t other = __ballot(lane > SB_ROWS || slots >> SB_SHIFT != slot >> SB_SHIFT);
  const int run = __builtin_ctzll(other), R = min(run, SB_ROWS);
  uint32_t used = lane < R ? 1u << (slots & (SB_ROWS - 1)) : 0u;
#pragma unroll
  for (int d = 1; d < SB_ROWS; d <<= 1) used |= __shfl_xor(used, d, 64);
  used = __builtin_amdgcn_readfirstlane(used);
  if ((run > SB_ROWS || __builtin_popcount(used) != R) && threadIdx.x == 0 && a.status) a.status[0] = MIMO_ERR_SLOT;   // a slot twice
  const bool anew = used & 1u, shared = R > 4;
  const int mask = (1 << a.page_shift) - 1;
  const size_t page = (size_t)(slot >> a.page_shift);
  const int me = shared ? threadIdx.x : lane, T = shared ? 256 : 64, per = shared ? 1 : 4;

  // The unit in hand: a head's K or V, and this thread's share of its rows, items of 8 values (of a pair of units, twice 8);
  // r, d: row of the run and first dimension of an item (-1: none), the same for all K and for all V.
  constexpr int ITEMS = 2;                                 // 16 rows of 192 over 256 threads, 4 over 64
  int kind = -1, D = 0, rot = 0, had = 0, r[ITEMS], d[ITEMS];
  uint8_t *codes, *scale;
  uint4 x[ITEMS], y[ITEMS];
  auto load = [&](int unit) __attribute__((always_inline)) {
    const bool is_v = unit >= a.Hkv;
    if (kind != (int)is_v) {
      kind = is_v;
      D = is_v ? a.Dv : a.Dk, rot = is_v ? 0 : a.rot;
      const int pairs = SIDE ? 0 : rot >> 4, P = (D >> 3) - pairs;   // P: items of a row
#pragma unroll
      for (int e = 0; e < ITEMS; ++e) {
        const int i = me + T * e, row = i / P, c = i - row * P;
        r[e] = i < R * P ? row : -1;
        d[e] = SIDE || c < pairs ? 8 * c : rot + 8 * (c - pairs);
      }
    }
    const int h = is_v ? unit - a.Hkv : unit;
    const size_t head = page * a.Hkv + h;
    codes = static_cast<uint8_t*>(is_v ? a.v_pages : a.k_pages) + ((head << a.page_shift) + (slot & mask & ~(SB_ROWS - 1))) * D;
    scale = static_cast<uint8_t*>(const_cast<void*>(is_v ? a.v_scale : a.k_scale)) + (head << (a.page_shift - SB_SHIFT)) + ((slot & mask) >> SB_SHIFT);
    const uint16_t* rows = is_v ? a.v + n * a.v_stride + h * D : a.k + n * a.k_stride + h * D;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    had = anew ? 0 : *scale;
#pragma unroll
    for (int e = 0; e < ITEMS; ++e) {
      if (r[e] < 0) continue;
      const uint16_t* p = rows + r[e] * stride + d[e];
      x[e] = *reinterpret_cast<const uint4*>(p);
      if (!SIDE && 2 * d[e] < rot) y[e] = *reinterpret_cast<const uint4*>(p + (rot >> 1));
    }
  };
  int unit = part * per + (shared ? 0 : wave);
  if (unit < 2 * a.Hkv) load(unit);
  if (part * per < a.Hkv) {                                // a K is among the units
    for (int i = threadIdx.x; i < R * half; i += 256) {
      const int r = i / half, j = i - r * half;
      const double t = (double)a.positions[n + r] * a.turns[j], f = t - rint(t);   // -1/2 .. 1/2 turns
      // sine and cosine of what 32 bits hold of the angle, and a first-order step for the rest
      const float hi = (float)f, lo = (float)((f - (double)hi) * 6.283185307179586);
      float sn, cs;
      sincospif(2.0f * hi, &sn, &cs);
      room.cos[i] = (cs - sn * lo) * a.magnitude, room.sin[i] = (sn + cs * lo) * a.magnitude;
    }
    lds_barrier();
  }

  int turn = 0;
  // the largest of a value over the unit's threads
  auto over_unit = [&](uint32_t most) __attribute__((always_inline)) {
    most = dpp_max_u32(most);
    if (shared) {
      if (lane == 0) room.most[turn][wave] = most;
      lds_barrier();
      most = max(max(room.most[turn][0], room.most[turn][1]), max(room.most[turn][2], room.most[turn][3]));
      turn ^= 1;                                           // what it is written to next has been read by then
    }
    return (uint32_t)__builtin_amdgcn_readfirstlane(most);
  };
#pragma unroll 1
  for (; unit < 2 * a.Hkv; unit += per * parts) {          // all waves of the block alike where units are shared
    float f[ITEMS][8], g[ITEMS][8];
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < ITEMS; ++e) {
      if (r[e] < 0) continue;
      ap_unpack(x[e], f[e]);
      if (!SIDE && 2 * d[e] < rot) {
        ap_unpack(y[e], g[e]);
        ap_turn(f[e], g[e], room.cos + r[e] * half + d[e], room.sin + r[e] * half + d[e]);
        top = sb_size(g[e], top);
      } else if (SIDE && d[e] < rot) {
        ap_turn_side(f[e], room.cos + r[e] * half + d[e] / 2, room.sin + r[e] * half + d[e] / 2);
      }
      top = sb_size(f[e], top);
    }
    asm volatile("" : "+v"(had));                          // the byte has come to every thread before one may write it
    uint32_t most = over_unit(__float_as_uint(top) & 0x7FFFFFFFu);
    bool over = most > 0x7F600000u;                        // past 448 * 2^119
    if (most >= 0x7F800000u) {
      most = 0;
#pragma unroll
      for (int e = 0; e < ITEMS; ++e) {
        if (r[e] < 0) continue;
        most = sb_finite_size(f[e], most);
        if (!SIDE && 2 * d[e] < rot) most = sb_finite_size(g[e], most);
      }
      most = over_unit(most);
    }
    const int need = sb_need(most), now = anew ? need : max(had, need);
    if (!anew && now > had) {
      const float by = sb_power(had - now);
      const int cells = D >> 4;
      for (int i = me; i < SB_ROWS * cells; i += T) {
        if (used >> (i / cells) & 1u) continue;
        uint4* p = reinterpret_cast<uint4*>(codes + 16 * i);
        const uint4 w = *p;
        *p = make_uint4(sb_rescale(w.x, by), sb_rescale(w.y, by), sb_rescale(w.z, by), sb_rescale(w.w, by));
      }
    }
    if (me == 0 && (anew || now > had)) *scale = (uint8_t)now;
    const float inverse = sb_power(127 - now);
#pragma unroll
    for (int e = 0; e < ITEMS; ++e) {
      const int to = __shfl(slots, max(r[e], 0), 64) & (SB_ROWS - 1);
      if (r[e] < 0) continue;
      *reinterpret_cast<uint2*>(codes + to * D + d[e]) = sb_pack(f[e], inverse, over);
      if (!SIDE && 2 * d[e] < rot) *reinterpret_cast<uint2*>(codes + to * D + d[e] + (rot >> 1)) = sb_pack(g[e], inverse, over);
    }
    if (unit + per * parts < 2 * a.Hkv) load(unit + per * parts);
  }
}

// Blocks 0 .. kv - 1 look at W rows each (a power of two up to 16) for those that a block of slots begins at, consecutive
// blocks at rows 16 apart: a long chunk's begin every 16 rows, and in the order of the rows would fall on few XCDs.  The rest
// are the q rows'.
template <bool SIDE>
__global__ void __launch_bounds__(256, 4) cache_append_scaled_kernel(AppendArgs a, int W, int parts, int q_parts) {
  __shared__ RunRoom room;
  const int C = (a.N + SB_ROWS - 1) / SB_ROWS, kv = SB_ROWS / W * C * parts, b = blockIdx.x;
  if (b >= kv) {
    const int n = (b - kv) / q_parts;
    return ap_token<AP_Q, SIDE>(a, n, b - kv - n * q_parts, q_parts, room.cos, room.sin);
  }
  const int x = b / parts, n0 = x % C * SB_ROWS + x / C * W, lane = threadIdx.x & 63;
  if (n0 >= a.N) return;
  // lane l: row n0 - 1 + l, up to the 31 rows behind the last: a block's first piece (16 rows at most), up to 15 rows of others
  // and the next piece's first row
  const int at = n0 - 1 + lane;
  const int slot = lane <= W + 2 * SB_ROWS - 1 && at >= 0 && at < a.N ? a.slots[at] : -1, before = __shfl_up(slot, 1, 64);
  const bool mine = lane >= 1 && lane <= W;
  if (mine && slot >= a.n_slots && threadIdx.x < 64 && a.status) a.status[0] = MIMO_ERR_SLOT;
  uint64_t first = __ballot(mine && slot >= 0 && slot < a.n_slots && slot >> SB_SHIFT != before >> SB_SHIFT);
  for (bool again = false; first; first &= first - 1, again = true) {
    const int l = __builtin_ctzll(first);
    // rows of this block that other rows part from it are in somebody else's care at the same time
    const uint64_t all = __ballot(slot >> SB_SHIFT == __builtin_amdgcn_readlane(slot, l) >> SB_SHIFT);
    const bool parted = ((all >> l) & ((all >> l) + 1)) || (all & ((1ull << l) - 1));
    if (parted && threadIdx.x == 0 && a.status) a.status[0] = MIMO_ERR_SLOT;
    if (again) lds_barrier();                              // the last block's angles have been read
    ap_run<SIDE>(a, n0 - 1 + l, __shfl(slot, min(lane + l, 63), 64), b - x * parts, parts, room);
  }
}

// ------------------------------------------------------------------ read
// Cached tokens as bf16 rows: code times scale in 32 bits, rounded to bf16 (with block scales exact, but for products below bf16's
// least step of 2^-133, which bytes 1 and 2 have).  A thread turns 8 values; a block of 256 a few tokens one after another, whose
// rows of a head share cache lines.
//
// Bound by HBM: 32768 tokens of 4 heads of 192/128 with block scales (126 MB) 23.4 us a call, 5.4 TB/s; the rows are written past
// the caches (31.0 us through them, call after call into the same rows; into rows that are new each time 24.1 and 25.0).  The
// same for append's q would cost more in the attention that reads it than it saves (4096 tokens windowed: 126 us instead of
// 119).  137 tokens 2.7 us, a launch.
struct ReadArgs {
  const uint8_t *k, *v;
  const void *k_scale, *v_scale;
  const int32_t* slots;
  uint16_t *k_out, *v_out;
  int32_t* status;
  int N, Hkv, Dk, Dv, page_shift, n_slots, tokens;
};

template <int DTYPE>
__global__ void __launch_bounds__(256) cache_read_kernel(ReadArgs a) {
#pragma clang fp contract(off)
  const int Uk = a.Hkv * (a.Dk >> 3), U = Uk + a.Hkv * (a.Dv >> 3), mask = (1 << a.page_shift) - 1;
  const int first = blockIdx.x * a.tokens, count = min(a.tokens, a.N - first);
  for (int e = threadIdx.x; e < count * U; e += 256) {
    const int t = e / U, w = e - t * U, n = first + t;
    const bool is_v = w >= Uk;
    const int D = is_v ? a.Dv : a.Dk, c = is_v ? w - Uk : w, h = c / (D >> 3), d = 8 * (c - h * (D >> 3));
    const int slot = a.slots[n];
    if (slot >= a.n_slots && w == 0 && a.status) a.status[0] = MIMO_ERR_SLOT;
    uint4 out = make_uint4(0, 0, 0, 0);
    if (slot >= 0 && slot < a.n_slots) {
      const size_t head = (size_t)(slot >> a.page_shift) * a.Hkv + h, at = ((head << a.page_shift) + (slot & mask)) * D + d;
      const uint8_t* pages = is_v ? a.v : a.k;
      const void* scale = is_v ? a.v_scale : a.k_scale;
      if constexpr (DTYPE == MIMO_KV_BF16) {
        out = *reinterpret_cast<const uint4*>(pages + 2 * at);
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(pages + at);
        const float s = DTYPE == MIMO_KV_E4M3 ? static_cast<const float*>(scale)[h]
                                              : e8m0_f32(static_cast<const uint8_t*>(scale)[(head << (a.page_shift - SB_SHIFT)) + ((slot & mask) >> SB_SHIFT)]);
        float f[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t word = i ? x.y : x.x;
          const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
          f[4 * i] = lo.x * s, f[4 * i + 1] = lo.y * s, f[4 * i + 2] = hi.x * s, f[4 * i + 3] = hi.y * s;
        }
        out = ap_pack(f);
      }
    }
    uint16_t* to = is_v ? a.v_out + (size_t)n * a.Hkv * a.Dv : a.k_out + (size_t)n * a.Hkv * a.Dk;
    __builtin_nontemporal_store(__builtin_bit_cast(v4i, out), reinterpret_cast<v4i*>(to + h * D + d));
  }
}

int check_cache(const mimo_kv_cache* c, const char* what) {
  MIMO_REQUIRE(c && c->k && c->v, MIMO_ERR_ARG, "%s: null pointer", what);
  MIMO_REQUIRE(c->dtype == MIMO_KV_BF16 || c->dtype == MIMO_KV_E4M3 || c->dtype == MIMO_KV_E4M3_BLOCKS, MIMO_ERR_ARG, "%s: cache dtype %d", what, c->dtype);
  MIMO_REQUIRE(c->dtype == MIMO_KV_BF16 || (c->k_scale && c->v_scale), MIMO_ERR_ARG, "%s: an E4M3 cache needs k_scale and v_scale", what);
  MIMO_REQUIRE((c->k_dim == 64 && c->v_dim == 64) || (c->k_dim == 128 && c->v_dim == 128) || (c->k_dim == 192 && c->v_dim == 128),
               MIMO_ERR_SHAPE, "%s: head dimensions %d / %d (64/64, 128/128 and 192/128 are supported)", what, c->k_dim, c->v_dim);
  MIMO_REQUIRE(c->page_size >= 16 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0, MIMO_ERR_SHAPE,
               "%s: page_size %d (a power of two from 16 to 1024)", what, c->page_size);
  MIMO_REQUIRE(c->kv_heads >= 1 && c->kv_heads <= 1024, MIMO_ERR_SHAPE, "%s: kv_heads %d", what, c->kv_heads);
  MIMO_REQUIRE(c->n_pages >= 1 && (int64_t)c->n_pages * c->page_size <= 0x7fffffff, MIMO_ERR_SHAPE,
               "%s: %d pages of %d (at most 2^31 - 1 slots)", what, c->n_pages, c->page_size);
  MIMO_REQUIRE(aligned16(c->k) && aligned16(c->v), MIMO_ERR_ALIGN, "%s: 16-byte alignment", what);
  MIMO_REQUIRE(c->dtype != MIMO_KV_E4M3_BLOCKS || (aligned16(c->k_scale) && aligned16(c->v_scale)), MIMO_ERR_ALIGN,
               "%s: 16-byte alignment of the block scales", what);
  const size_t scales = (size_t)c->n_pages * c->kv_heads * (c->page_size / 16);
  MIMO_REQUIRE(c->dtype != MIMO_KV_E4M3_BLOCKS || !overlap(c->k_scale, scales, c->v_scale, scales), MIMO_ERR_ARG,
               "%s: k_scale and v_scale overlap: a block scale belongs to K or to V", what);
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
  const mimo_rotary rotary{turns, rotary_dim, 0, 1.0f};
  return mimo_cache_append_rotary(q, q_stride, heads, k, k_stride, v, v_stride, N, positions, slots, cache, &rotary, q_out, status, stream);
}

int mimo_cache_append_rotary(const uint16_t* q, int64_t q_stride, int heads, const uint16_t* k, int64_t k_stride, const uint16_t* v,
                             int64_t v_stride, int N, const int32_t* positions, const int32_t* slots, const mimo_kv_cache* cache,
                             const mimo_rotary* rotary, uint16_t* q_out, int32_t* status, void* stream) {
  if (int e = check_cache(cache, "cache_append")) return e;
  const bool scaled = cache->dtype == MIMO_KV_E4M3_BLOCKS;
  const int64_t most = scaled ? kMaxBlocks / 2 - SB_ROWS : kMaxBlocks;
  MIMO_REQUIRE(N >= 0 && N <= most, MIMO_ERR_SHAPE, "cache_append: %d tokens (0 to %s)", N, scaled ? "2^23 - 17" : "2^24 - 1");
  if (N == 0) return MIMO_OK;
  const mimo_rotary none{nullptr, 0, 0, 1.0f};
  const mimo_rotary& ro = rotary ? *rotary : none;
  MIMO_REQUIRE(k && v && positions && slots, MIMO_ERR_ARG, "cache_append: null pointer");
  MIMO_REQUIRE(!q == !q_out, MIMO_ERR_ARG, "cache_append: q and q_out go together");
  MIMO_REQUIRE(!q || (heads >= 1 && heads <= 65536), MIMO_ERR_SHAPE, "cache_append: %d heads", heads);
  MIMO_REQUIRE(ro.dim >= 0 && ro.dim % 16 == 0 && ro.dim <= cache->k_dim, MIMO_ERR_SHAPE,
               "cache_append: rotary_dim %d (a multiple of 16 up to k_dim)", ro.dim);
  MIMO_REQUIRE(ro.dim == 0 || ro.turns, MIMO_ERR_ARG, "cache_append: null pointer");
  MIMO_REQUIRE(ro.interleaved == 0 || ro.interleaved == 1, MIMO_ERR_ARG, "cache_append: interleaved must be 0 or 1");
  MIMO_REQUIRE(ro.magnitude - ro.magnitude == 0.0f, MIMO_ERR_ARG, "cache_append: magnitude must be finite");
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
  AppendArgs a{q, k, v, q_stride, k_stride, v_stride, heads, cache->kv_heads, cache->k_dim, cache->v_dim, N, ro.dim, ro.turns,
               ro.magnitude, positions, slots, q_out, cache->k, cache->v, cache->k_scale, cache->v_scale, __builtin_ctz(cache->page_size),
               cache->n_pages * cache->page_size, status};
  const bool side = ro.dim && ro.interleaved;
  hipStream_t st = as_stream(stream);
  // few tokens are spread over several blocks each
  const int per = cache->k_dim - (side ? 0 : ro.dim / 2);
  auto spread = [&](int units) { return std::max(1, std::min((units + 255) / 256, AP_BLOCKS / N)); };
  {
    ProfScope p(st, "cache_append");
    if (scaled) {
      // four units of a block of slots to a block (two: 15.3 us for the pieces, one 18.8); W rows to look at
      const int q_parts = spread(heads * per / 8);
      int parts = (cache->kv_heads + 1) / 2, W = 1;
      while (W < SB_ROWS && (int64_t)N * parts > (int64_t)W * SB_BLOCKS) W *= 2;
      parts = std::max(1, std::min(parts, SB_BLOCKS * SB_ROWS / N));
      const int64_t grid = (int64_t)((N + SB_ROWS - 1) / SB_ROWS) * (SB_ROWS / W) * parts + (q ? (int64_t)N * q_parts : 0);
      if (side) cache_append_scaled_kernel<true><<<(unsigned)grid, 256, 0, st>>>(a, W, parts, q_parts);
      else cache_append_scaled_kernel<false><<<(unsigned)grid, 256, 0, st>>>(a, W, parts, q_parts);
    } else {
      const int units = ((q ? heads : 0) * per + cache->kv_heads * (per + cache->v_dim)) / 8;
      const dim3 grid(N, spread(units));
      const bool f8 = cache->dtype == MIMO_KV_E4M3;
      if (side && f8) cache_append_kernel<AP_E4M3, true><<<grid, 256, 0, st>>>(a);
      else if (side) cache_append_kernel<AP_BF16, true><<<grid, 256, 0, st>>>(a);
      else if (f8) cache_append_kernel<AP_E4M3, false><<<grid, 256, 0, st>>>(a);
      else cache_append_kernel<AP_BF16, false><<<grid, 256, 0, st>>>(a);
    }
  }
  return check_launch("cache_append");
}

int mimo_cache_read(const mimo_kv_cache* cache, const int32_t* slots, int N, uint16_t* k_out, uint16_t* v_out, int32_t* status,
                    void* stream) {
  if (int e = check_cache(cache, "cache_read")) return e;
  MIMO_REQUIRE(N >= 0 && N <= kMaxBlocks, MIMO_ERR_SHAPE, "cache_read: %d tokens (0 to 2^24 - 1)", N);
  if (N == 0) return MIMO_OK;
  MIMO_REQUIRE(slots && k_out && v_out, MIMO_ERR_ARG, "cache_read: null pointer");
  MIMO_REQUIRE(aligned16(k_out) && aligned16(v_out), MIMO_ERR_ALIGN, "cache_read: 16-byte alignment of k_out and v_out");
  const size_t kn = (size_t)cache->kv_heads * cache->k_dim, vn = (size_t)cache->kv_heads * cache->v_dim;
  const size_t rows = (size_t)cache->n_pages * cache->page_size * (cache->dtype == MIMO_KV_BF16 ? 2 : 1);
  const void* outs[2] = {k_out, v_out};
  const size_t sizes[2] = {N * kn * 2, N * vn * 2};
  for (int i = 0; i < 2; ++i)
    MIMO_REQUIRE(!overlap(outs[i], sizes[i], cache->k, rows * kn) && !overlap(outs[i], sizes[i], cache->v, rows * vn) &&
                     !overlap(outs[i], sizes[i], slots, (size_t)N * 4),
                 MIMO_ERR_ARG, "cache_read: outputs may not overlap the cache or the slots");
  if (cache->dtype != MIMO_KV_BF16) {
    const size_t scales = cache->dtype == MIMO_KV_E4M3 ? (size_t)cache->kv_heads * 4 : (size_t)cache->n_pages * cache->kv_heads * (cache->page_size / 16);
    for (int i = 0; i < 2; ++i)
      MIMO_REQUIRE(!overlap(outs[i], sizes[i], cache->k_scale, scales) && !overlap(outs[i], sizes[i], cache->v_scale, scales), MIMO_ERR_ARG,
                   "cache_read: outputs may not overlap the scales");
  }
  MIMO_REQUIRE(!overlap(k_out, sizes[0], v_out, sizes[1]), MIMO_ERR_ARG, "cache_read: k_out may not overlap v_out");
  ReadArgs a{static_cast<const uint8_t*>(cache->k), static_cast<const uint8_t*>(cache->v), cache->k_scale, cache->v_scale, slots,
             k_out, v_out, status, N, cache->kv_heads, cache->k_dim, cache->v_dim, __builtin_ctz(cache->page_size),
             cache->n_pages * cache->page_size, 0};
  a.tokens = std::max(1, std::min(16, N / 2048));
  const unsigned grid = (N + a.tokens - 1) / a.tokens;
  hipStream_t st = as_stream(stream);
  {
    ProfScope p(st, "cache_read");
    if (cache->dtype == MIMO_KV_BF16) cache_read_kernel<MIMO_KV_BF16><<<grid, 256, 0, st>>>(a);
    else if (cache->dtype == MIMO_KV_E4M3) cache_read_kernel<MIMO_KV_E4M3><<<grid, 256, 0, st>>>(a);
    else cache_read_kernel<MIMO_KV_E4M3_BLOCKS><<<grid, 256, 0, st>>>(a);
  }
  return check_launch("cache_read");
}

}  // extern "C"
