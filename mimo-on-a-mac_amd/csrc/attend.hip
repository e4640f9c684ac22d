// Attention of a step's new tokens over the paged K/V cache (mimo_cache_attend; the reference's Attention,
// engine/mimo_stream/mimo_v2.py:110-150, on one request's cache).
//
// Rows.  The queries that share a K/V head (its G heads, one after another, of consecutive tokens) are the rows of a tile, so
// a key or value is read once for all of them: narrow tiles of 32 rows for requests with few rows (decode), wide tiles of 128.
//
// One pass over the keys with the running maximum m and sum l of each row (exp(x) = 2^(x log2 e) throughout):
//   S^T = K Q^T      v_mfma_f32_32x32x16_bf16, K rows as the A operand: lane (r, h) = (l % 32, l / 32) then holds, for
//                    query row r, the keys 8 (i / 4) + 4 h + i % 4 of a block of 32 in registers i = 0 .. 15
//   P = 2^(c S - m)  in registers; the row maximum needs one exchange between the lane halves
//   O^T += V^T P^T   the P registers 8 s .. 8 s + 7, rounded to bf16, are the B operand of keys 16 s .. as they stand: the
//                    order of keys inside a product is free, so V^T is read in the same order, by transposing LDS reads
// so neither S nor P leaves its lane, and m, l and the rescaling of O are per lane too.  V is bf16, so P has to be: wide tiles
// round it once (by up to 2^-8 of a weight; a second product for the rest would be 40% more matrix work), narrow ones, which
// wait for memory, multiply the rounded rest as well, which leaves 2^-17 of a weight.  l sums the unrounded values.
//
// K and V go from HBM to LDS without passing registers, 16 bytes a lane; in LDS a tile is [64-element column block][key][128
// bytes, E4M3 64] with the 16-byte cells of a row permuted by its number, which keeps the operand reads free of bank conflicts.
// E4M3 becomes bf16 (exactly) after the LDS read; the scales multiply c and the result.
//
// Masks.  A tile's loads touch only keys that some row of the tile sees: others (past the last position, between the first
// tokens and the window) read a visible row again, and their weights are set to 0.  A key that one row sees and another does
// not (of another wave's, too: all waves of a wide tile share its keys) still meets the other's weight 0 in the product, and
// 0 * NaN is NaN: a wave whose sums are not finite looks for such values in its tiles with masks, and if there are any takes
// its sums again key by key.
//
// Work is cut so that the card is full: a device-side count of all requests' tiles gives the number of key tiles per block
// (chunk); a row tile with more is split over several blocks, whose (O, m, l) a second kernel joins in a fixed order.
//
// What bounds it.  Wide: the matrix pipes next to the softmax, under a clock that the power limits.  4096 tokens at 8192, 64/4
// heads of 192/128 (1.72 TFLOP): 1540-1740 us on different cards, 1.0-1.1 PFLOP/s at 1.70-1.77 GHz, where a large bf16 product
// reaches 1.39; matrix pipes busy 55-59%, VALU 54-62%, no bank conflicts; 1.24 PFLOP/s without the softmax, and as much
// without the copies.  Two blocks of 4 waves on a CU fill each other's pauses: one block 0.86; 64 rows a wave, one wave a SIMD
// 0.97 (sums moved between the register files); the next tile's products woven into the softmax by hand 0.58 (spills; heads
// of 64, which have the room, 0.59 against 0.70); row sums by a matrix product, operands read further ahead, wave priorities:
// no change.  Heads of 64: the exponentials (16 cycles for 64 of them) and what is around them, 0.66-0.70 PFLOP/s.
// No vector register is spilled; 9 to 14 (wide) and 48 to 52 (narrow) scalar ones are, to lanes of a vector register.
// Narrow: HBM.  48 requests of 500 to 16384 keys (1.03 GB) 187 us, 5.5 TB/s; 32 of 1000 to 32768 in E4M3 (1.13 GB) 206 us, 5.4
// TB/s, above a large copy's 4.9 (read and written); a call of few keys 9 us, a chain of round trips (starts and lengths,
// the table, K and V, the waves' parts through LDS).
#include <algorithm>
#include <atomic>
#include <mutex>

#include "cache.h"
#include "device.h"
#include "parts.h"

namespace mimo {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));

struct AttendArgs {
  const uint16_t* q;
  int64_t q_stride;
  int N, Hq, Hkv, G, B, max_pages, n_pages, page_shift, window, sinks;
  const int32_t *starts, *lens, *table;
  const uint8_t *k, *v;
  const float *k_scale, *v_scale, *sink_logits;
  float scale;
  uint16_t* out;
  int32_t* status;
  // rows of a tile: TQ tokens of HT heads (HG groups of HT heads cover G), Hh = Hkv * HG
  int TQ, HT, HG, Hh, target;
  // split tiles: per slot TQ * HT rows of O (fp32 [Dv]) and (m, l); per (token, head group) the first part's slot and
  // parts | token's place in its tile << 16.  Part i > 0 is in slot (first & ~part_mask) + i part_step.  meta is null when no
  // tile can be split.
  float *part_o, *part_ml;
  int2* meta;
  int part_mask, part_step, slots;
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int AT_THREADS = 256;
// Blocks wanted: two per CU.  Wide: 512 tokens at 8192, 64/4 heads, 185 us; wanting 640 or 768 makes three parts of tiles that
// two fit: 215.  Narrow: 1024 makes one request of 32768 keys 27.7 us (25.6), 256 makes 128 windowed decodes 39.6 (27.9).
constexpr int AT_WIDE_TARGET = 512, AT_NARROW_TARGET = 512;
// Parts of wide tiles have at least 4 units of 64 keys: 40 tokens of 32/8 heads at 3000 21.7 us; 27.3 with 2, 24.9 with 8.
// Narrow tiles of up to 2 units of 128 keys (a window of 128) are not split, which saves the join's launch.
constexpr int AT_WIDE_MIN = 4, AT_NARROW_MIN = 2;
constexpr int AT_START = 8;                               // units that a wide block's start and a part's join cost

template <int DK_, int DV_, bool F8_, bool WIDE_> struct AtCfg {
  static constexpr int DK = DK_, DV = DV_;
  static constexpr bool F8 = F8_, WIDE = WIDE_;
  static constexpr int CBB = F8 ? 64 : 128;                // bytes of a row in one 64-element column block
  static constexpr int KCB = DK / 64, VCB = DV / 64;
  static constexpr int KEYS = WIDE ? 64 : 32;              // keys of one LDS tile (narrow: one wave's)
  static constexpr int NB = KEYS / 32;
  static constexpr int UNIT = WIDE ? 64 : 128;             // keys per iteration of the block
  static constexpr int ROWS = WIDE ? 128 : 32;
  static constexpr int KBYTES = KEYS * CBB * KCB, VBYTES = KEYS * CBB * VCB;
  static constexpr int STAGE = KBYTES + VBYTES;
  static constexpr int GR = 1024 / CBB;                    // rows of one copy instruction (64 lanes of 16 bytes)
  static constexpr int LR = (WIDE ? 16 : 32) / GR;         // row groups that a wave copies per tile
  static constexpr int MERGE = WIDE ? 0 : 4 * 32 * DV * 4 + 4 * 32 * 8;   // narrow: the waves' O, m, l joined at the end
  static constexpr int LDS = (WIDE ? 2 * STAGE : 4 * STAGE) > MERGE ? (WIDE ? 2 * STAGE : 4 * STAGE) : MERGE;
  static constexpr int WGS = 2;                            // blocks per CU
  static_assert(WGS * LDS <= 163840, "LDS of the blocks of a CU");
};

__device__ __forceinline__ void at_wait_vm(int n) {
  switch (n) {
    case 0: asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); break;
    case 2: asm volatile("s_waitcnt vmcnt(2)" ::: "memory"); break;
    case 4: asm volatile("s_waitcnt vmcnt(4)" ::: "memory"); break;
    case 6: asm volatile("s_waitcnt vmcnt(6)" ::: "memory"); break;
    case 8: asm volatile("s_waitcnt vmcnt(8)" ::: "memory"); break;
    case 12: asm volatile("s_waitcnt vmcnt(12)" ::: "memory"); break;
    default: asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); break;
  }
}
__device__ __forceinline__ void at_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes from every lane's address to lds + 16 * lane (lds: LDS byte offset, wave-uniform); the caller waits on vmcnt
__device__ __forceinline__ void at_copy16(const uint8_t* src, uint32_t lds) {
  const uint32_t m = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(m) : "memory", "m0");
}
#pragma clang diagnostic pop

__device__ __forceinline__ float at_swap_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float at_swap_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// four / two E4M3 codes of a dword to bf16, exact
__device__ __forceinline__ bf16x8 at_f8_bf16x8(uint32_t a, uint32_t b) {
  const bf16x2 x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false), y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
  const bf16x2 z = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false), w = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
  return bf16x8{x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}

// ------------------------------------------------------------------ the work of a block
// The keys a row tile sees: positions p_min .. p_max, keys lo .. p_max and the first `sinks`.  It walks them in groups of 16
// keys (which lie in one page): groups 0 .. sg - 1 hold the first tokens, group sg starts at org, gt groups in all; a unit is
// 4 (wide) or 8 groups, I units.
struct AtRange {
  int p_min, p_max, lo, sinks, sg, org, gt, I;
  __device__ __forceinline__ int key(int g) const { return g < sg ? 16 * g : org + 16 * (g - sg); }
};
__device__ __forceinline__ AtRange at_range(int p_min, int p_max, int window, int sinks, int unit) {
  AtRange r;
  r.p_min = p_min, r.p_max = p_max;
  r.lo = window && p_min >= window ? p_min - window + 1 : 0;
  r.sinks = r.lo ? min(sinks, r.lo) : 0;
  r.sg = (r.sinks + 15) >> 4;
  r.org = r.lo & ~15;
  if (16 * r.sg >= r.org) r.sg = r.org = 0;
  r.gt = r.sg + ((p_max - r.org) >> 4) + 1;
  r.I = (16 * r.gt + unit - 1) / unit;
  return r;
}
// the most units any row tile of a request of `len` tokens walks
__host__ __device__ __forceinline__ int at_most(int64_t len, int window, int sinks, int TQ, int unit) {
  if (len <= 0) return 0;
  const int64_t all = (len - 1) / unit + 1;
  if (!window) return (int)all;
  const int64_t groups = ((sinks < len ? sinks : len) + 15) / 16 + ((int64_t)window + TQ + 13) / 16 + 1;
  const int64_t w = (16 * groups + unit - 1) / unit;
  return (int)(w < all ? w : all);
}

// One row tile of one request and head group, units it0 .. it1 - 1 of its I: part `split` of ns, kept in `slot` when ns > 1.
struct AtItem {
  int b, s0, n, len, tt, hh, it0, it1, ns, slot;
};

// Request b's rows s0 .. s0 + n - 1 and length, clamped: whatever starts and lens hold, nothing is out of range.  false: its
// starts run backwards or are not among the rows.
__device__ __forceinline__ bool at_request(const AttendArgs& a, int b, int& s0, int& n, int& len) {
  const int from = a.starts[b], to = a.starts[b + 1];
  s0 = min(max(from, 0), a.N);
  n = min(max(to, s0), a.N) - s0;
  len = a.lens[b];
  if (n && (len < n || len > ((long long)a.max_pages << a.page_shift))) len = 0;   // refused: its rows are set to 0
  return s0 == from && s0 + n == to;
}
constexpr int AT_REFUSED = 1 << 22;                         // 64 lanes of this stay below 2^31
__device__ __forceinline__ int at_last(int v) { return __builtin_amdgcn_readlane(v, 63); }
// The list of work, which every wave makes for itself without a word to the others: lane l looks at requests l per ..,
// and the prefix sums of what they ask for are the places in the list.  Starts in order ask for at most N <= 2^20 tiles; a
// request whose starts are not counts as AT_REFUSED of them, which refuses the call.
// Wide tiles.  Block blockIdx.x's item: (request, part, row tile from the last to the first) x head group, head groups
// fastest: neighbouring blocks, on different XCDs, work on different heads, and an XCD keeps meeting the same ones.  Parts
// that a request's shorter tiles do not have stand together at its end (were a tile's parts neighbours, these blocks without
// work would all fall on the same XCDs: 320 tiles, half of them split, took 333 us instead of 185).  A tile is cut into parts
// of `chunk` units.  0: past the end of the list, or a part that this tile does not have; -1: the call is refused.
template <class C>
__device__ __forceinline__ int at_find(const AttendArgs& a, AtItem& it) {
  const int lane = threadIdx.x & 63;
  const int per = (a.B + 63) / 64, b0 = min(a.B, lane * per), b1 = min(a.B, b0 + per);
  int s0, n, len, tiles = 0, nt, ns, I, longest = 0;
  float load = 0.0f;                                       // units of all tiles; only their share per block is wanted
  auto read = [&](int b) {
    const bool sound = at_request(a, b, s0, n, len);
    nt = (n + a.TQ - 1) / a.TQ;
    I = at_most(len, a.window, a.sinks, a.TQ, C::UNIT);
    return sound;
  };
  // the lane's first request, as a rule its only one, is kept
  int first[5] = {0, 0, 0, 0, 0};
  auto size = [&](int b) {
    if (b == b0) s0 = first[0], n = first[1], len = first[2], nt = first[3], I = first[4];
    else read(b);
  };
  for (int b = b0; b < b1; ++b) {
    const bool sound = read(b);
    if (b == b0) first[0] = s0, first[1] = n, first[2] = len, first[3] = nt, first[4] = I;
    tiles = sound ? min(tiles + nt, AT_REFUSED) : AT_REFUSED;
    load += (float)nt * I;
    if (nt) longest = max(longest, I);
  }
  tiles = at_last(dpp_prefix_i32(tiles));
  load = dpp_sum_f32(load) * a.Hh;
  longest = (int)dpp_max_u32((uint32_t)longest);
  if (tiles >= AT_REFUSED) return -1;
  int chunk = 1 << 30, units = 0, parts = 0;
  auto count = [&](int c) {                                // this lane's blocks and those of split tiles; their units
    float cut = 0.0f;
    units = 0, parts = 0;
    for (int b = b0; b < b1; ++b) {
      size(b);
      ns = max(1, (I + c - 1) / c);
      units += nt * ns;
      if (ns > 1) parts += nt * ns, cut += (float)nt * I;
    }
    return cut;
  };
  // Parts that fit k rounds of `target` blocks: the fair share, rounded up by more than the sum's error (which leaves fewer
  // than target blocks more than tiles, and parts within twice the target), then larger while the split tiles' parts are more
  // than their share of the blocks.  One round, unless the card would stay half empty and two of smaller parts are sooner
  // done, a block's start and its part's join counted as AT_START units (32/8 heads at 8192: 640 tokens 150 us with the fair
  // share, 113 with one round; 1200 tokens 237 with one round, 209 with two.  AT_START 16 gains 5% on 800 tokens and makes a
  // chunk beside 32 long decodes 214 us instead of 160).
  float best = 0.0f;
#pragma unroll 1
  for (int k = 1; a.meta && k <= 2; ++k) {
    const float blocks = (float)(k * a.target);
    int c = max(AT_WIDE_MIN, (int)fminf(load * 1.0001f / blocks + 1.0f, 1.0e9f));
    bool more = false;
#pragma unroll 1
    for (int trial = 0; trial < 3; ++trial) {
      const float cut = dpp_sum_f32(count(c)) * a.Hh, over = dpp_sum_f32((float)parts) * a.Hh * load / (cut * blocks);
      if (!(over > 1.0f)) break;                           // also where nothing is split
      more = true;
      c = (int)fminf(c * over + 1.0f, 1.0e9f);
    }
    if (k == 1) {
      chunk = c, best = (float)(min(c, longest) + AT_START);
      if (!more) break;
    } else if (2.0f * (c + AT_START) < best) {
      count(c);
      const int64_t all = at_last(dpp_prefix_i32(min(parts, 1 << 22))), blk = at_last(dpp_prefix_i32(min(units, 1 << 22)));
      if (all * a.Hh <= a.slots && (blk - tiles) * a.Hh <= 2 * a.target) chunk = c;
    }
  }
  count(chunk);
  int ub = dpp_prefix_i32(units) - units, pb = dpp_prefix_i32(parts) - parts;
  const int u = blockIdx.x / a.Hh, hh = blockIdx.x % a.Hh;
  int f_b = 0, f_tt = 0, f_split = 0, f_slot = 0, f_ns = 0;
  const bool here = u >= ub && u < ub + units;
  if (here) {
    int b = b0;
    for (;; ++b) {
      size(b);
      ns = max(1, (I + chunk - 1) / chunk);
      if (u < ub + nt * ns) break;
      ub += nt * ns;
      pb += ns > 1 ? nt * ns : 0;
    }
    f_split = (u - ub) / nt;
    const int at = u - ub - f_split * nt;
    f_b = b, f_tt = nt - 1 - at, f_slot = (pb + at * ns + f_split) * a.Hh + hh, f_ns = ns;
  }
  const uint64_t who = __ballot(here);
  if (!who) return 0;
  const int src = __builtin_ctzll(who);
  auto from = [&](int v) { return __builtin_amdgcn_readlane(v, src); };
  it.b = from(f_b), it.tt = from(f_tt), it.slot = from(f_slot), it.hh = hh;
  it.s0 = from(s0), it.n = from(n), it.len = from(len);
  const int split = from(f_split);
  ns = from(f_ns);
  it.it0 = 0, it.it1 = 0x7fffffff, it.ns = 1;
  if (ns > 1) {
    const int p0 = it.len - it.n + it.tt * a.TQ, p1 = min(p0 + a.TQ, it.len) - 1;
    const int I = at_range(p0, p1, a.window, a.sinks, C::UNIT).I;
    it.ns = (I + chunk - 1) / chunk;                       // in parts of equal size
    if (split >= it.ns) return 0;
    it.it0 = part_begin(split, I, it.ns), it.it1 = part_begin(split + 1, I, it.ns);
  }
  return 1;
}

// 16 keys from a multiple of 16 on, of which a tile may load: their page and what hidden keys read instead
struct AtKeys {
  int g0, fb, id;
};
__device__ __forceinline__ AtKeys at_keys(const AttendArgs& a, const AtRange& r, int b, int g0) {
  AtKeys g;
  if (g0 > r.p_max || (g0 >= r.sinks && g0 + 15 < r.lo)) g0 = r.p_max & ~15;
  g.g0 = g0;
  g.fb = g0 >= r.lo || g0 < r.sinks ? g0 : r.lo;
  const int at = __builtin_amdgcn_readfirstlane(b * a.max_pages + (g0 >> a.page_shift));
  // the table is constant while the kernel runs: a scalar load, whose wait is not the vector loads'
  g.id = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(a.table))[at];
  return g;
}
__device__ __forceinline__ int at_page(const AttendArgs& a, int id) {
  if ((uint32_t)id < (uint32_t)a.n_pages) return id;
  if (a.status && (threadIdx.x & 63) == 0) a.status[0] = MIMO_ERR_SLOT;
  return 0;
}
// cache row (of [page, head, row in page]) of key g0 + r
__device__ __forceinline__ size_t at_row(const AttendArgs& a, const AtRange& r, const AtKeys& g, int page, int kv, int row) {
  const int j = g.g0 + row;
  const int key = j <= r.p_max && (j >= r.lo || j < r.sinks) ? j : g.fb;
  return (((size_t)page * a.Hkv + kv) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
}

// One query row (at q, position p) against the keys of units it0 .. it1 - 1, `count` groups from `first` on in each, in plain
// 32-bit arithmetic with the wave's lanes along the head: a hidden key is never touched.  For waves that met a NaN or an
// infinity in a value that not all of their rows see.  O: dimensions 64 e + lane.
template <class C>
__device__ __forceinline__ void at_slow(const AttendArgs& a, const AtRange& r, int b, int kv, int it0, int it1, int first, int count,
                                        const uint16_t* q, int p, float c, float (&O)[C::VCB], float& m, float& l) {
  const int lane = threadIdx.x & 63;
  float x[C::KCB];
#pragma unroll
  for (int e = 0; e < C::KCB; ++e) x[e] = bf16_to_f32(q[64 * e + lane]);
#pragma unroll
  for (int e = 0; e < C::VCB; ++e) O[e] = 0.0f;
  m = -INFINITY, l = 0.0f;
  auto load = [&](const uint8_t* base, size_t at) {
    return C::F8 ? e4m3_unpack2(base[at]).x : bf16_to_f32(reinterpret_cast<const uint16_t*>(base)[at]);
  };
#pragma unroll 1
  for (int g = it0 * (C::UNIT / 16); g < min(r.gt, it1 * (C::UNIT / 16)); ++g) {
    if (g % (C::UNIT / 16) < first || g % (C::UNIT / 16) >= first + count) continue;
    const int base = r.key(g);
#pragma unroll 1
    for (int j = base; j < base + 16 && j <= p; ++j) {
      if (a.window && j <= p - a.window && j >= a.sinks) continue;
      const int page = at_page(a, a.table[(size_t)b * a.max_pages + (j >> a.page_shift)]);
      const size_t row = (((size_t)page * a.Hkv + kv) << a.page_shift) + (j & ((1 << a.page_shift) - 1));
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < C::KCB; ++e) s += x[e] * load(a.k, row * C::DK + 64 * e + lane);
      s = dpp_sum_f32(s) * c;
      const float top = fmaxf(m, s), ref = top == -INFINITY ? 0.0f : top;
      const float was = at_exp2(m - ref), w = at_exp2(s - ref);
      m = top;
      l = l * was + w;
#pragma unroll
      for (int e = 0; e < C::VCB; ++e) O[e] = O[e] * was + (w == 0.0f ? 0.0f : w * load(a.v, row * C::DV + 64 * e + lane));
    }
  }
}

// One item.
template <class C>
__device__ __forceinline__ void at_tile(const AttendArgs& a, uint8_t* lds, const AtItem& item) {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));                              // nothing per lane is kept in registers from one item to the next
  const int lane = t & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int b = __builtin_amdgcn_readfirstlane(item.b), hg = item.hh % a.HG, kv = item.hh / a.HG, ns = item.ns;
  const int tok0 = item.tt * a.TQ, toks = min(a.TQ, item.n - tok0);
  const int heads = min(a.HT, a.G - hg * a.HT);
  const int qrow = (C::WIDE ? 32 * wave : 0) + r32;        // this lane's query row
  const int qt = qrow / a.HT, qh = qrow - qt * a.HT;
  const bool valid = qt < toks && qh < heads;
  const int head = kv * a.G + hg * a.HT + qh;
  const size_t out_at = ((size_t)(item.s0 + tok0 + qt) * a.Hq + head) * C::DV;
  const int base_pos = item.len - item.n + tok0;
  if (a.meta && item.it0 == 0 && t < toks)
    a.meta[(size_t)(item.s0 + tok0 + t) * a.Hh + item.hh] = make_int2(item.slot, ns | (t << 16));
  if (item.len == 0) {                                     // a refused request
    if (a.status && t == 0) a.status[0] = MIMO_ERR_SHAPE;
    if (valid && (C::WIDE || wave == 0))
      for (int d = 0; d < C::DV / 2; d += 8) *reinterpret_cast<uint4*>(a.out + out_at + h * (C::DV / 2) + d) = make_uint4(0, 0, 0, 0);
    return;
  }
  const AtRange rg = at_range(base_pos, base_pos + toks - 1, a.window, a.sinks, C::UNIT);
  const int it0 = item.it0, it1 = min(item.it1, rg.I);

  constexpr int UG = C::UNIT / 16, TG = C::KEYS / 16;      // groups of a unit, of an LDS tile
  const int wg = C::WIDE ? 0 : 2 * wave;                   // the tile's first group in its unit
  constexpr int NG = C::WIDE ? 1 : 2;                      // 16-key groups that the wave copies
  AtKeys kg[NG];
  auto look = [&](int it) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < NG; ++g) kg[g] = at_keys(a, rg, b, rg.key(it * UG + (C::WIDE ? wave : wg) + g));
  };
  look(it0);                                               // the table is read while the queries are asked for

  // queries as the B operand: row r32, dimensions 16 s + 8 h .. (E4M3: 32 (s / 2) + 16 h + 8 (s % 2) .., since a lane's 16
  // bytes of K are 16 dimensions, two products' worth); c = |scale| k_scale log2 e, a negative scale turns q round
  float c = a.scale * kLog2e * (C::F8 ? a.k_scale[kv] : 1.0f);
  const uint32_t flip = c < 0.0f ? 0x80008000u : 0u;
  const bool zero = c == 0.0f;
  c = zero ? 1.0f : fabsf(c);
  uint4 qraw[C::DK / 16];
  {
    const uint16_t* qp = a.q + (int64_t)(item.s0 + tok0 + qt) * a.q_stride + head * C::DK + (C::F8 ? 16 : 8) * h;
#pragma unroll
    for (int s = 0; s < C::DK / 16; ++s) {
      qraw[s] = make_uint4(0, 0, 0, 0);
      if (valid && !zero) qraw[s] = *reinterpret_cast<const uint4*>(qp + (C::F8 ? 32 * (s >> 1) + 8 * (s & 1) : 16 * s));
    }
  }
  bf16x8 Q[C::DK / 16];
  auto take_q = [&]() __attribute__((always_inline)) {     // once the first copies are on their way
#pragma unroll
    for (int s = 0; s < C::DK / 16; ++s)
      Q[s] = __builtin_bit_cast(bf16x8, make_uint4(qraw[s].x ^ flip, qraw[s].y ^ flip, qraw[s].z ^ flip, qraw[s].w ^ flip));
  };
  const int pos = base_pos + qt;                           // this lane's position
  const int w_first = C::WIDE ? 32 * wave / a.HT : 0, w_last = min(toks - 1, ((C::WIDE ? 32 * wave : 0) + 31) / a.HT);
  const bool busy = w_first <= w_last;                     // the wave has rows
  const int wp_min = base_pos + w_first, wp_max = base_pos + w_last;

  // copies: lane's row inside a row group and its 16-byte cell; the cell at place p of row x is p ^ swizzle(x).  bf16 K:
  // (x / 2) % 8, so that 16 rows' cells of one column differ in their banks; V: 4 ((x / 2) % 2), so that the 4 rows of 64 bytes
  // of a transposing read do; E4M3: (x / 4) % 4 for both.
  const int cr = lane / (C::CBB / 16);
  const int cell_k = C::F8 ? (lane & 3) ^ ((lane >> 4) & 3) : (lane & 7) ^ (lane >> 4);
  const int cell_v = C::F8 ? cell_k : (lane & 7) ^ (4 * ((lane >> 4) & 1));
  const uint32_t lds0 = lds_addr(lds) + (C::WIDE ? 0 : wave * C::STAGE);
  size_t crow[C::LR];
  auto rows_of = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < C::LR; ++x) {
      const int g = x * C::GR / 16;
      crow[x] = at_row(a, rg, kg[g], at_page(a, kg[g].id), kv, x * C::GR % 16 + cr);
    }
  };
  constexpr int ES = C::F8 ? 1 : 2;
  auto issue_k = [&](uint32_t stage) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < C::LR; ++x) {
      const uint8_t* p = a.k + crow[x] * (C::DK * ES) + 16 * (C::F8 ? cell_k : cell_k ^ (4 * (x & 1)));
#pragma unroll
      for (int cb = 0; cb < C::KCB; ++cb)
        at_copy16(p + cb * C::CBB, stage + cb * (C::KEYS * C::CBB) + ((C::WIDE ? wave * C::LR : 0) + x) * 1024);
    }
  };
  auto issue_v = [&](uint32_t stage) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < C::LR; ++x) {
      const uint8_t* p = a.v + crow[x] * (C::DV * ES) + 16 * cell_v;
#pragma unroll
      for (int cb = 0; cb < C::VCB; ++cb)
        at_copy16(p + cb * C::CBB, stage + C::KBYTES + cb * (C::KEYS * C::CBB) + ((C::WIDE ? wave * C::LR : 0) + x) * 1024);
    }
  };

  // operand addresses in a tile: K row r32, cell 2 s + h; V as the transposing reads want them
  const int i16 = lane & 15, d16 = (lane >> 4) & 1;
  const int k_at = C::F8 ? r32 * 64 + 16 * (h ^ ((r32 >> 2) & 3)) : r32 * 128 + 16 * (h ^ ((r32 >> 1) & 7));
  const int v_row = C::F8 ? 4 * h + ((i16 >> 1) & 3) + 8 * (i16 >> 3) : 4 * h + (i16 >> 2);
  const int v_at = C::F8 ? v_row * 64 + 16 * (d16 ^ ((v_row >> 2) & 3)) + 8 * (i16 & 1)
                         : v_row * 128 + 16 * ((2 * d16 + ((i16 >> 1) & 1)) ^ (4 * ((v_row >> 1) & 1))) + 8 * (i16 & 1);
  auto k_read = [&](const uint8_t* st, int kb, int s) __attribute__((always_inline)) {   // cell 2 s + h of key 32 kb + r32
    if constexpr (C::F8) return *reinterpret_cast<const uint4*>(st + (k_at ^ (32 * (s & 1))) + (s >> 1) * (C::KEYS * 64) + kb * 32 * 64);
    else return *reinterpret_cast<const uint4*>(st + (k_at ^ (32 * (s & 3))) + (s >> 2) * (C::KEYS * 128) + kb * 32 * 128);
  };
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"   // LDS pointers are 32 bits on the device
  auto v_frag = [&](const uint8_t* st, int kb, int s, int d) __attribute__((always_inline)) {
    typedef __attribute__((address_space(3))) v4s* lds4;
    typedef __attribute__((address_space(3))) v2i* lds2;
    if constexpr (C::F8) {
      const uint8_t* p = st + C::KBYTES + (v_at ^ (32 * (d & 1))) + (d >> 1) * (C::KEYS * 64) + (32 * kb + 16 * s) * 64;
      const v2i w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds2)(uint32_t)(uintptr_t)p);
      return at_f8_bf16x8(w[0], w[1]);
    } else {
      const uint8_t* p = st + C::KBYTES + (v_at ^ (64 * (d & 1))) + (d >> 1) * (C::KEYS * 128) + (32 * kb + 16 * s) * 128;
      const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uint32_t)(uintptr_t)p);
      const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uint32_t)((uintptr_t)p + 8 * 128));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
#pragma clang diagnostic pop

  v16f O[C::DV / 32];
#pragma unroll
  for (int d = 0; d < C::DV / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[d][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;                           // l: this lane half's keys

  v16f S[C::NB];
  bf16x8 P[C::NB][2], rest[C::WIDE ? 1 : C::NB][2];        // narrow: what the rounding of P leaves off, rounded
  // operands are read PX products ahead; the barriers keep the compiler from reading them all at once (spilled registers)
  constexpr int PX = 4;
  auto scores = [&](const uint8_t* st) __attribute__((always_inline)) {
    constexpr int PER = C::F8 ? 2 : 1, F = C::NB * C::DK / (16 * PER);   // products per read
    uint4 X[PX];
#pragma unroll
    for (int f = 0; f < PX && f < F; ++f) X[f] = k_read(st, f % C::NB, f / C::NB);
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int kb = f % C::NB, s = f / C::NB;
      __builtin_amdgcn_sched_barrier(0);
      const v16f none = {0.0f};
      const uint4 x = X[f % PX];
      if constexpr (C::F8) {
        S[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at_f8_bf16x8(x.x, x.y), Q[2 * s], s == 0 ? none : S[kb], 0, 0, 0);
        S[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at_f8_bf16x8(x.z, x.w), Q[2 * s + 1], S[kb], 0, 0, 0);
      } else {
        S[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), Q[s], s == 0 ? none : S[kb], 0, 0, 0);
      }
      if (f + PX < F) X[f % PX] = k_read(st, (f + PX) % C::NB, (f + PX) / C::NB);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // keys that a row does not see: unsigned(pos - j) < span for the causal order and the window together
  const uint32_t span = a.window ? (uint32_t)a.window : 0x80000000u;
  auto mask = [&](int g0) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < TG; ++x) {
      const int j0 = rg.key(g0 + x);
      const uint32_t back = (uint32_t)(pos - j0 - 4 * h);
      if (j0 >= a.sinks) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float s = S[x / 2][8 * (x % 2) + i];
          S[x / 2][8 * (x % 2) + i] = back - (uint32_t)(8 * (i / 4) + i % 4) < span ? s : -INFINITY;
        }
      } else {
        const int first = min(a.sinks, pos + 1) - j0 - 4 * h;   // first tokens that the row sees, from the lane's first key on
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int o = 8 * (i / 4) + i % 4;
          const float s = S[x / 2][8 * (x % 2) + i];
          S[x / 2][8 * (x % 2) + i] = back - (uint32_t)o < span || o < first ? s : -INFINITY;
        }
      }
    }
  };
  auto softmax = [&]() __attribute__((always_inline)) {
    float top = S[0][0];
#pragma unroll
    for (int kb = 0; kb < C::NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, S[kb][i]);
    top = at_swap_max(top) * c;
    // m may lag behind the maximum by 8 (weights of up to 2^8, exact as any others); past that O and l are rescaled
    if (__ballot(top > m + 8.0f || (m == -INFINITY && top > m))) {
      const float next = fmaxf(m, top), was = at_exp2(m - (next == -INFINITY ? 0.0f : next));
      m = next;
      l *= was;
#pragma unroll
      for (int d = 0; d < C::DV / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) O[d][i] *= was;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int kb = 0; kb < C::NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = at_exp2(__builtin_fmaf(S[kb][i], c, -ref));
        l += p;
        P[kb][i / 8][i % 8] = (__bf16)p;
        if constexpr (!C::WIDE) rest[kb][i / 8][i % 8] = (__bf16)(p - (float)P[kb][i / 8][i % 8]);
      }
  };
  auto values = [&](const uint8_t* st) __attribute__((always_inline)) {
    constexpr int ND = C::DV / 32, F = C::NB * 2 * ND;
    bf16x8 X[PX];
#pragma unroll
    for (int f = 0; f < PX; ++f) X[f] = v_frag(st, f / (2 * ND), f / ND % 2, f % ND);
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int kb = f / (2 * ND), s = f / ND % 2, d = f % ND;
      __builtin_amdgcn_sched_barrier(0);
      O[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(X[f % PX], P[kb][s], O[d], 0, 0, 0);
      if constexpr (!C::WIDE) O[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(X[f % PX], rest[kb][s], O[d], 0, 0, 0);
      if (f + PX < F) X[f % PX] = v_frag(st, (f + PX) / (2 * ND), (f + PX) / ND % 2, (f + PX) % ND);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // every row of the wave sees all keys of the tile from group g0 on
  auto open = [&](int g0) {
    const int j0 = rg.key(g0);
    return g0 >= rg.sg && j0 + C::KEYS - 1 <= wp_min && (!a.window || j0 > wp_max - a.window);
  };

  if constexpr (C::WIDE) {
    rows_of();
    issue_k(lds0);
    issue_v(lds0);
    take_q();
    for (int it = it0; it < it1; ++it) {
      const int cur = (it - it0) & 1, g0 = it * UG;
      if (it + 1 < it1) look(it + 1);
      at_wait_vm(0);
      __syncthreads();                                     // the tile has landed everywhere; the other one is free
      if (it + 1 < it1) {
        rows_of();
        issue_k(lds0 + (cur ^ 1) * C::STAGE);
        issue_v(lds0 + (cur ^ 1) * C::STAGE);
      }
      if (!busy || rg.key(g0) > wp_max) continue;
      const uint8_t* st = lds + cur * C::STAGE;
      scores(st);
      if (!open(g0)) mask(g0);
      softmax();
      values(st);
    }
  } else {
    const uint8_t* st = lds + wave * C::STAGE;
    constexpr int NK = C::LR * C::KCB, NV = C::LR * C::VCB;
    const int end = min(it1, (rg.gt - wg + UG - 1) / UG);  // of the units that hold groups of this wave
    if (it0 < end) {
      rows_of();
      issue_k(lds0);
      issue_v(lds0);
    }
    take_q();
    for (int it = it0; it < end; ++it) {
      const int g0 = it * UG + wg;
      const bool more = it + 1 < end;
      if (more) look(it + 1);
      at_wait_vm(NV);
      scores(st);
      at_wait_lds();                                       // K has been read: its room takes the next keys
      if (more) {
        rows_of();
        issue_k(lds0);
      }
      if (!open(g0)) mask(g0);
      softmax();
      if (more) at_wait_vm(NK);
      else at_wait_vm(0);
      values(st);
      at_wait_lds();
      if (more) issue_v(lds0);
    }
  }
  // Sums that are not finite.  What a row sees makes them so rightly; wrongly, a value that it does not see and another does
  // (through its weight of 0), or an infinity times a weight of 0 (a hidden key's copy, the rest of a weight) that makes it
  // a NaN.
  bool suspect = false;
  {
    float worst = 0.0f;
#pragma unroll
    for (int d = 0; d < C::DV / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) worst += O[d][i] - O[d][i];   // 0, or NaN
    // The tile's rows see different keys, the wave's own or another wave's: the keys in LDS are those that any of them sees.
    const bool apart = rg.p_min != rg.p_max;
    if ((apart || !C::F8) && __ballot(busy && worst != 0.0f)) {
      bool odd = false;
#pragma unroll 1
      for (int g = it0 * UG; g < min(rg.gt, it1 * UG); ++g) {
        const bool op = open(g / TG * TG);
        if (op && (C::WIDE || C::F8)) continue;
        const AtKeys k = at_keys(a, rg, b, rg.key(g));
        const int page = at_page(a, k.id);
#pragma unroll 1
        for (int x = 0; x < 16; ++x) {
          const size_t row = at_row(a, rg, k, page, kv, x) * C::DV;
          const uint32_t w = lane < C::DV * ES / 4 ? *reinterpret_cast<const uint32_t*>(a.v + row * ES + 4 * lane) : 0u;
          if (C::F8) odd |= (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
          else if (apart && !op) odd |= (((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u) != 0;
          else odd |= (w & 0x7FFFu) == 0x7F80u || (w >> 16 & 0x7FFFu) == 0x7F80u;
        }
      }
      suspect = __ballot(odd) != 0;
    }
  }
  const float vs = C::F8 ? a.v_scale[kv] : 1.0f;
  // the wave's rows once more, one by one; done(row, place of the row, its head, O, m, l)
  auto slow = [&](auto done) __attribute__((always_inline)) {
#pragma unroll 1
    for (int r = 0; r < 32; ++r) {
      const int row = __builtin_amdgcn_readfirstlane((C::WIDE ? 32 * wave : 0) + r), rt = row / a.HT, rh = row - rt * a.HT;
      if (rt >= toks || rh >= heads) continue;
      const int hd = kv * a.G + hg * a.HT + rh;
      float O[C::VCB], m, l;
      at_slow<C>(a, rg, b, kv, it0, it1, C::WIDE ? 0 : 2 * wave, C::WIDE ? 4 : 2,
                 a.q + (int64_t)(item.s0 + tok0 + rt) * a.q_stride + hd * C::DK, base_pos + rt,
                 a.scale * kLog2e * (C::F8 ? a.k_scale[kv] : 1.0f), O, m, l);
      done(r, rt, hd, O, m, l);
    }
  };

  if constexpr (C::WIDE) {
    if (suspect) {
      slow([&](int r, int rt, int hd, const float (&O)[C::VCB], float m, float l) __attribute__((always_inline)) {
        const size_t row = (size_t)item.slot * (a.TQ * a.HT) + 32 * wave + r;
        if (ns > 1 && lane == 0) a.part_ml[2 * row] = m, a.part_ml[2 * row + 1] = l;
        const float sink = a.sink_logits ? a.sink_logits[hd] * kLog2e : -INFINITY;
        const float top = fmaxf(m, sink), ref = top == -INFINITY ? 0.0f : top;
        const float f = at_exp2(m - ref), tot = l * f + at_exp2(sink - ref);
#pragma unroll
        for (int e = 0; e < C::VCB; ++e) {
          if (ns > 1) a.part_o[row * C::DV + 64 * e + lane] = O[e] * vs;
          else a.out[((size_t)(item.s0 + tok0 + rt) * a.Hq + hd) * C::DV + 64 * e + lane] = tot == 0.0f ? 0 : f32_to_bf16(O[e] * (vs * f / tot));
        }
      });
      return;
    }
    l = at_swap_sum(l);
    if (ns > 1) {
      if (!valid) return;
      const size_t row = (size_t)item.slot * (a.TQ * a.HT) + qt * a.HT + qh;
      if (h == 0) a.part_ml[2 * row] = m, a.part_ml[2 * row + 1] = l;
#pragma unroll
      for (int d = 0; d < C::DV / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4*>(a.part_o + row * C::DV + 32 * d + 2 * i + 4 * h) =
              make_float4(O[d][i] * vs, O[d][i + 1] * vs, O[d][i + 2] * vs, O[d][i + 3] * vs);
      return;
    }
    const float sink = a.sink_logits && valid ? a.sink_logits[head] * kLog2e : -INFINITY;
    const float top = fmaxf(m, sink), ref = top == -INFINITY ? 0.0f : top;
    const float f = at_exp2(m - ref), tot = l * f + at_exp2(sink - ref);
    const float w = tot == 0.0f ? 0.0f : vs * f / tot;
    // the halves of a row trade quads of values, so that a lane stores 16 bytes
#pragma unroll
    for (int d = 0; d < C::DV / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 8) {
        uint32_t x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = i + 2 * k;
          x[k] = tot == 0.0f ? 0u : (uint32_t)f32_to_bf16(O[d][e] * w) | ((uint32_t)f32_to_bf16(O[d][e + 1] * w) << 16);
        }
        const auto p = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false), q = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
        if (valid) *reinterpret_cast<uint4*>(a.out + out_at + 32 * d + 2 * i + 8 * h) = make_uint4(p[0], q[0], p[1], q[1]);
      }
  } else {
    // the waves' parts, joined over LDS in wave order: row r at [wave][r][DV], 16-byte pieces turned by the row
    float* po = reinterpret_cast<float*>(lds);
    float* pm = po + 4 * 32 * C::DV;
    at_wait_vm(0);
    __syncthreads();                                       // every wave is done with its tiles
    constexpr int NP = C::DV / 4;
    if (suspect) {
      slow([&](int r, int, int, const float (&O)[C::VCB], float m, float l) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < C::VCB; ++e) {
          const int piece = 16 * e + lane / 4;
          po[(wave * 32 + r) * C::DV + 4 * ((piece + r) & (NP - 1)) + (lane & 3)] = O[e];
        }
        if (lane == 0) pm[2 * (32 * wave + r)] = m, pm[2 * (32 * wave + r) + 1] = l;
      });
    } else {
      l = at_swap_sum(l);
#pragma unroll
      for (int d = 0; d < C::DV / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int piece = 8 * d + i / 2 + h;
          *reinterpret_cast<float4*>(po + (wave * 32 + r32) * C::DV + 4 * ((piece + r32) & (NP - 1))) =
              make_float4(O[d][i], O[d][i + 1], O[d][i + 2], O[d][i + 3]);
        }
      if (h == 0) pm[2 * (32 * wave + r32)] = m, pm[2 * (32 * wave + r32) + 1] = l;
    }
    __syncthreads();
    for (int e = t; e < 32 * NP; e += AT_THREADS) {
      const int row = e / NP, piece = e & (NP - 1), rt = row / a.HT, rh = row - rt * a.HT;
      if (rt >= toks || rh >= heads) continue;
      float mw[4], top = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) mw[w] = pm[2 * (32 * w + row)], top = fmaxf(top, mw[w]);
      const int hd = kv * a.G + hg * a.HT + rh;
      const float sink = ns == 1 && a.sink_logits ? a.sink_logits[hd] * kLog2e : -INFINITY;
      const float all = fmaxf(top, sink), ref = all == -INFINITY ? 0.0f : all;
      float tot = ns == 1 ? at_exp2(sink - ref) : 0.0f;
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = at_exp2(mw[w] - ref);
        const float4 o = *reinterpret_cast<const float4*>(po + (w * 32 + row) * C::DV + 4 * ((piece + row) & (NP - 1)));
        tot += pm[2 * (32 * w + row) + 1] * f;
        x[0] += o.x * f, x[1] += o.y * f, x[2] += o.z * f, x[3] += o.w * f;
      }
      if (ns > 1) {
        const size_t pr = (size_t)item.slot * (a.TQ * a.HT) + row;
        *reinterpret_cast<float4*>(a.part_o + pr * C::DV + 4 * piece) = make_float4(x[0] * vs, x[1] * vs, x[2] * vs, x[3] * vs);
        if (piece == 0) a.part_ml[2 * pr] = all, a.part_ml[2 * pr + 1] = tot;
      } else {
        const float w = tot == 0.0f ? 0.0f : vs / tot;
        uint2 y;
        y.x = (uint32_t)f32_to_bf16(x[0] * w) | ((uint32_t)f32_to_bf16(x[1] * w) << 16);
        y.y = (uint32_t)f32_to_bf16(x[2] * w) | ((uint32_t)f32_to_bf16(x[3] * w) << 16);
        if (tot == 0.0f) y = make_uint2(0, 0);
        *reinterpret_cast<uint2*>(a.out + ((size_t)(item.s0 + tok0 + rt) * a.Hq + hd) * C::DV + 4 * piece) = y;
      }
    }
    __syncthreads();                                       // the next item's copies may come
  }
}

// rows of no request
__device__ __forceinline__ void at_clear(const AttendArgs& a, int row) {
  const int first = a.starts[0], last = a.starts[a.B], gap = first + a.N - last;
  for (int i = blockIdx.x; i < gap; i += gridDim.x) {
    uint4* o = reinterpret_cast<uint4*>(a.out + (size_t)(i < first ? i : last + i - first) * row);
    for (int d = threadIdx.x; d < row / 8; d += AT_THREADS) o[d] = make_uint4(0, 0, 0, 0);
  }
}
// a refused call: all rows, and nothing is left for the join
__device__ __forceinline__ void at_refuse(const AttendArgs& a, int row) {
  const int64_t from = (int64_t)blockIdx.x * AT_THREADS + threadIdx.x, step = (int64_t)gridDim.x * AT_THREADS;
  for (int64_t i = from; i < (int64_t)a.N * row / 8; i += step) reinterpret_cast<uint4*>(a.out)[i] = make_uint4(0, 0, 0, 0);
  if (a.meta)
    for (int64_t i = from; i < (int64_t)a.N * a.Hh; i += step) a.meta[i] = make_int2(0, 0);
  if (from == 0 && a.status) a.status[0] = MIMO_ERR_SHAPE;
}

template <class C>
__global__ void __launch_bounds__(AT_THREADS, C::WGS) attend_wide_kernel(AttendArgs a) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  AtItem item;
  const int found = at_find<C>(a, item);
  if (found < 0) return at_refuse(a, a.Hq * C::DV);
  if (found) at_tile<C>(a, lds, item);
  at_clear(a, a.Hq * C::DV);
}

// Narrow tiles: all units of a head group, request after request, in equal shares for the blocks of the group, so that none
// ends late whatever the lengths (48 requests of 500 to 16384 keys 191 us; a list of parts as for wide tiles 209; wide tiles
// lose by it, 24 mixed requests 91 us instead of 52, for each cut costs them a start and 128 rows of a join).  A block
// walks its share tile by tile; a tile on the border of two shares is split.  Slot 2 (j Hh + hh) holds block j's part of a
// tile that began in an earlier share (or with this one), the slot behind it the part of one that goes on in the next.
template <class C>
__global__ void __launch_bounds__(AT_THREADS, C::WGS) attend_narrow_kernel(AttendArgs a) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, hh = blockIdx.x % a.Hh, j = blockIdx.x / a.Hh;
  const int per = (a.B + 63) / 64, b0 = min(a.B, lane * per), b1 = min(a.B, b0 + per);
  // without room for parts (no tile can have more than AT_NARROW_MIN units) a share is whole tiles, each counted as one
  int s0, n, len, nt, I;
  auto size = [&](int b) {
    const bool sound = at_request(a, b, s0, n, len);
    nt = (n + a.TQ - 1) / a.TQ;
    I = a.meta ? max(1, at_most(len, a.window, a.sinks, a.TQ, C::UNIT)) : 1;
    return sound;
  };
  int64_t mine = 0;
  int tiles = 0;
  for (int b = b0; b < b1; ++b) {
    const bool sound = size(b);
    mine += (int64_t)nt * I;
    tiles = sound ? min(tiles + nt, AT_REFUSED) : AT_REFUSED;
  }
  tiles = at_last(dpp_prefix_i32(tiles));
  if (tiles >= AT_REFUSED) return at_refuse(a, a.Hq * C::DV);
  int64_t before, total;
  if (!__ballot(mine >> 25)) {                             // 64 of them stay below 2^31
    const int p = dpp_prefix_i32((int)mine);
    before = p - mine, total = at_last(p);
  } else {
    before = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t p = __shfl_up(before, d, 64);
      if (lane >= d) before += p;
    }
    total = __shfl(before, 63, 64);
    before -= mine;
  }
  // blocks that share the work: a unit each at least, and one per CU while that leaves them no more than 8 units and the tiles
  // alone do not fill the card (one request of 32768 keys, 64/4 heads: 25.6 us with 256 blocks, 27.8 with 512; 8 of 4000: 24.1
  // and 25.5; a limit of 32 units changes neither)
  const bool few = total * a.Hh <= 8 * (a.target / 2) && (int64_t)tiles * a.Hh < a.target / 2;
  const int most = max(1, (few ? a.target / 2 : a.target) / a.Hh);
  const uint32_t shares = total >= most ? most : max(1, (int)total);
  // share x begins at unit (x coarse / shares) << sh, sh chosen so that 32 bits hold the products: no 64-bit division
  const int sh = max(0, 65 - __builtin_clzll(total | 1) - __builtin_clz(shares));
  const uint32_t coarse = (uint32_t)(total >> sh);
  auto begin = [&](uint32_t x) { return x == shares ? total : (int64_t)(x * coarse / shares) << sh; };
  auto holder = [&](int64_t x) { return (int)min(shares - 1, (((uint32_t)(x >> sh) + 1) * shares - 1) / max(1u, coarse)); };
  if (j < (int)shares) {
    const int64_t u0 = begin(j), u1 = begin(j + 1);
    for (int64_t u = u0; u < u1;) {
      int f_b = 0, f_tt = 0, f_off = 0;
      const bool here = u >= before && u < before + mine;
      if (here) {
        int64_t at = before;
        int b = b0;
        for (;; ++b) {
          size(b);
          if (u < at + (int64_t)nt * I) break;
          at += (int64_t)nt * I;
        }
        // tile of the request: the quotient by I, found bit by bit where 32 bits do not hold it
        int64_t x = u - at;
        for (int bit = 20; x >> 32; --bit)
          if (x >= (int64_t)I << bit) x -= (int64_t)I << bit, f_tt += 1 << bit;
        const uint32_t q = (uint32_t)x / (uint32_t)I;
        f_b = b, f_tt += q, f_off = (uint32_t)x - q * I;
      }
      const int src = __builtin_ctzll(__ballot(here));
      auto from = [&](int v) { return __builtin_amdgcn_readlane(v, src); };
      AtItem item;
      item.b = from(f_b), item.s0 = from(s0), item.n = from(n), item.len = from(len), item.tt = from(f_tt), item.hh = hh;
      const int bound = from(I), off = from(f_off);
      const int64_t start = u - off;
      const int p0 = item.len - item.n + item.tt * a.TQ, p1 = min(p0 + a.TQ, item.len) - 1;
      const int real = item.len ? at_range(p0, p1, a.window, a.sinks, C::UNIT).I : 1;
      item.ns = 1, item.slot = 0, item.it0 = 0, item.it1 = real;
      if (a.meta) {
        if (start < u0 || start + real > u1) item.ns = holder(start + real - 1) - holder(start) + 1;
        item.slot = 2 * (j * a.Hh + hh) + (start > u0 ? 1 : 0);
        item.it0 = off, item.it1 = (int)min((int64_t)real, u1 - start);
      }
      if (item.it0 < item.it1) at_tile<C>(a, lds, item);
      u = start + bound;
    }
  }
  at_clear(a, a.Hq * C::DV);
}

// The parts of a split row, joined in order by W waves: out = sum_j 2^(m_j - M) O_j / sum_j 2^(m_j - M) l_j, wave w parts w,
// w + W, ... (eight at once, asked for before the weights are known).  The sums of the other waves come through LDS.
template <int DV, int W>
__device__ __forceinline__ void at_join(const AttendArgs& a, int n, int hh, int qh, int2 mt, float (*so)[DV], float* sl) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  constexpr int E = DV / 64;
  const int ns = mt.y & 0xFFFF, hg = hh % a.HG, kv = hh / a.HG, head = kv * a.G + hg * a.HT + qh;
  const size_t rows = (size_t)a.TQ * a.HT, in = (size_t)(mt.y >> 16) * a.HT + qh;
  auto part = [&](int j) { return (size_t)(j ? (mt.x & ~a.part_mask) + j * a.part_step : mt.x) * rows + in; };
  float o[8][E];
  float2 ml[8];
  auto fetch = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (j0 + W * i >= ns) break;
      const size_t row = part(j0 + W * i);
      const float* p = a.part_o + row * DV + E * lane;
      ml[i] = *reinterpret_cast<const float2*>(a.part_ml + 2 * row);
#pragma unroll
      for (int k = 0; k < E; ++k) o[i][k] = p[k];
    }
  };
  if (wave < ns) fetch(wave);
  float top = -INFINITY;
  for (int j = lane; j < ns; j += 64) top = fmaxf(top, a.part_ml[2 * part(j)]);
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
  const float ref = top == -INFINITY ? 0.0f : top;
  float tot = 0.0f, x[E];
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = 0.0f;
  for (int j0 = wave; j0 < ns; j0 += 8 * W) {
    if (j0 != wave) fetch(j0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (j0 + W * i >= ns) break;
      const float f = at_exp2(ml[i].x - ref);
      tot += f * ml[i].y;
#pragma unroll
      for (int k = 0; k < E; ++k) x[k] += f * o[i][k];
    }
  }
#pragma unroll
  for (int k = 0; k < E; ++k) so[wave][E * lane + k] = x[k];
  if (lane == 0) sl[wave] = tot;
  __syncthreads();
  tot = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) tot += sl[w];
  const float sink = a.sink_logits ? a.sink_logits[head] * kLog2e : -INFINITY;
  const float all = fmaxf(top, sink), r2 = all == -INFINITY ? 0.0f : all, g = at_exp2(top - r2), sum = tot * g + at_exp2(sink - r2);
  uint16_t* out = a.out + ((size_t)n * a.Hq + head) * DV;
  for (int d = t; d < DV; d += 64 * W) {
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) y += so[w][d];
    out[d] = sum == 0.0f ? 0 : f32_to_bf16(y * g / sum);
  }
}
// The parts of an entry (a token and head group) that was split, or 0.  It is read whether or not the token belongs to a
// request (then nobody wrote it): what cannot be right is not followed.
__device__ __forceinline__ int2 at_meta(const AttendArgs& a, int entry) {
  const int2 mt = a.meta[entry];
  const int n = entry / a.Hh, first = min(max(a.starts[0], 0), a.N), last = min(max(a.starts[a.B], first), a.N);
  const int ns = mt.y & 0xFFFF, place = (uint32_t)mt.y >> 16;
  const bool ok = n >= first && n < last && ns > 1 && place < a.TQ && mt.x >= 0 && mt.x + (int64_t)(ns - 1) * a.part_step < a.slots;
  return ok ? mt : make_int2(0, 0);
}

// Few rows: a block for each, of W waves (few rows with many parts take 16, so that the parts arrive in one or two round
// trips).  Bound by the round trips: a launch, the entry, the parts; 4.3 us for 64 rows of 64 parts, 5.3 for 1024 of a few.
template <int DV, int W>
__global__ void __launch_bounds__(64 * W) attend_join_kernel(AttendArgs a) {
  __shared__ float sl[W], so[W][DV];
  const int entry = blockIdx.x / a.HT, qh = blockIdx.x - entry * a.HT;
  const int2 mt = at_meta(a, entry);
  if (!mt.y || entry % a.Hh % a.HG * a.HT + qh >= a.G) return;
  at_join<DV, W>(a, entry / a.Hh, entry % a.Hh, qh, mt, so, sl);
}
// Many rows: DV / 4 lanes for `per` heads of an entry, one after another; a row's parts come PB at a time, under a running
// maximum.  Round trips again, so many rows have to be on their way at once: 32768 rows of two parts, DV 128 (34 MB) 9.9 us,
// 21.3 with a wave a row; 20000 rows of four parts, DV 64 6.0 us (13.3).
template <int DV>
__global__ void __launch_bounds__(256, 8) attend_join_many_kernel(AttendArgs a, int per) {
  constexpr int LANES = DV / 4, PB = 4;
  const int d = 4 * (threadIdx.x & (LANES - 1)), cuts = (a.HT + per - 1) / per;
  const int item = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, entry = item / cuts;
  if (entry >= a.N * a.Hh) return;
  const int2 mt = at_meta(a, entry);
  const int ns = mt.y & 0xFFFF, n = entry / a.Hh, hh = entry - n * a.Hh, kv = hh / a.HG, hg = hh - kv * a.HG;
  const int q0 = (item - entry * cuts) * per, q1 = ns ? min(min(a.HT, a.G - hg * a.HT), q0 + per) : 0;
#pragma unroll 1
  for (int qh = q0; qh < q1; ++qh) {
    const int head = kv * a.G + hg * a.HT + qh;
    const size_t tile = (size_t)a.TQ * a.HT, in = (size_t)((uint32_t)mt.y >> 16) * a.HT + qh;
    float top = -INFINITY, tot = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j0 = 0; j0 < ns; j0 += PB) {
      float2 ml[PB];
      float4 o[PB];
#pragma unroll
      for (int i = 0; i < PB; ++i) {
        ml[i] = make_float2(-INFINITY, 0.0f);
        o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (j0 + i < ns) {
          const size_t at = (size_t)(j0 + i ? (mt.x & ~a.part_mask) + (j0 + i) * a.part_step : mt.x) * tile + in;
          ml[i] = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
          o[i] = *reinterpret_cast<const float4*>(a.part_o + at * DV + d);
        }
      }
      float next = top;
#pragma unroll
      for (int i = 0; i < PB; ++i) next = fmaxf(next, ml[i].x);
      const float ref = next == -INFINITY ? 0.0f : next, was = at_exp2(top - ref);
      top = next;
      tot *= was;
      x.x *= was, x.y *= was, x.z *= was, x.w *= was;
#pragma unroll
      for (int i = 0; i < PB; ++i) {
        const float f = at_exp2(ml[i].x - ref);
        tot += f * ml[i].y;
        x.x += f * o[i].x, x.y += f * o[i].y, x.z += f * o[i].z, x.w += f * o[i].w;
      }
    }
    const float sink = a.sink_logits ? a.sink_logits[head] * kLog2e : -INFINITY;
    const float all = fmaxf(top, sink), ref = all == -INFINITY ? 0.0f : all, g = at_exp2(top - ref), sum = tot * g + at_exp2(sink - ref);
    const float w = sum == 0.0f ? 0.0f : g / sum;
    uint2 y;
    y.x = (uint32_t)f32_to_bf16(x.x * w) | ((uint32_t)f32_to_bf16(x.y * w) << 16);
    y.y = (uint32_t)f32_to_bf16(x.z * w) | ((uint32_t)f32_to_bf16(x.w * w) << 16);
    if (sum == 0.0f) y = make_uint2(0, 0);
    *reinterpret_cast<uint2*>(a.out + ((size_t)n * a.Hq + head) * DV + d) = y;
  }
}

// ------------------------------------------------------------------ host
static void at_tiles(int rows, int N, int heads, int kv_heads, AttendArgs& a) {
  a.G = heads / kv_heads;
  a.HT = std::min(a.G, rows);
  a.HG = (a.G + a.HT - 1) / a.HT;
  a.Hh = kv_heads * a.HG;
  a.TQ = std::max(1, std::min(rows / a.HT, N));
}

struct AtRoom {
  size_t o, ml, meta;
};
static AtRoom at_room(int rows, int target, int N, int heads, int kv_heads, int v_dim) {
  AttendArgs a{};
  at_tiles(rows, N, heads, kv_heads, a);
  // wide: a request is split when its tiles walk more than chunk units, so its parts are at most twice its share of the
  // target; narrow: two slots a block
  const size_t pr = (size_t)2 * std::max(target, a.Hh) * a.TQ * a.HT;
  return {align256(pr * v_dim * 4), align256(pr * 8), align256((size_t)N * a.Hh * sizeof(int2))};
}

// Held while a call's kernel and its join are queued: threads that share a stream share its workspace, and a kernel of one
// between the two of another would write over the parts that are to be joined.
static std::mutex at_queue;

template <class C>
static int at_launch(AttendArgs a, bool join, hipStream_t st) {
  const auto kernel = [] {
    if constexpr (C::WIDE) return &attend_wide_kernel<C>;
    else return &attend_narrow_kernel<C>;
  }();
  // row tiles: at most sum ceil(n_b / TQ) over at most min(B, N) requests with rows; wide blocks: tiles plus splits
  const int64_t tiles = ((int64_t)a.N + (int64_t)std::min(a.B, a.N) * (a.TQ - 1)) / a.TQ;
  const int64_t grid = C::WIDE ? tiles * a.Hh + (join ? 2 * a.target : 0) : (int64_t)std::max(1, a.target / a.Hh) * a.Hh;
  MIMO_REQUIRE(grid <= kMaxBlocks, MIMO_ERR_SHAPE, "cache_attend: %lld row tiles of head groups", (long long)grid);
  // the join: a block for each of few rows; many (mostly rows that were not split: 262144 of them 4.8 us in eights, 15 more one
  // by one; fewer may all be split, and then have to be on their way together: 48 decodes 192 us in all, 202 in eights)
  const int64_t entries = (int64_t)a.N * a.Hh, rows = entries * a.HT;
  const int per = rows <= 65536 ? 1 : std::min(a.HT, 8);
  constexpr int IPB = 1024 / C::DV;
  const int64_t joins = (entries * ((a.HT + per - 1) / per) + IPB - 1) / IPB;
  MIMO_REQUIRE(!join || joins <= kMaxBlocks, MIMO_ERR_SHAPE, "cache_attend: %lld rows to join", (long long)rows);
  static std::atomic<uint64_t> allowed{0};                 // devices on which the kernel may use its LDS
  int dev = 0;
  MIMO_HIP(hipGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(allowed.load(std::memory_order_acquire) & bit)) {
    MIMO_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS));
    allowed.fetch_or(bit, std::memory_order_release);
  }
  a.part_mask = C::WIDE ? 0 : 1;
  a.part_step = C::WIDE ? a.Hh : 2 * a.Hh;
  a.slots = 2 * std::max(a.target, a.Hh);
  std::unique_lock<std::mutex> queue(at_queue, std::defer_lock);
  if (join) queue.lock();
  {
    ProfScope p(st, C::WIDE ? "attend_wide" : "attend_narrow");
    kernel<<<(unsigned)grid, AT_THREADS, C::LDS, st>>>(a);
  }
  if (int e = check_launch("attend")) return e;
  if (!join) return MIMO_OK;
  {
    ProfScope p(st, "attend_join");
    // rows of few tokens have many parts: at 64 rows of 64 parts 16 waves a row 4.3 us; at 512 rows (8 decodes of 4000 keys)
    // 4 waves 24.0 us in all, 16 25.1, a part of a wave 24.5
    if (rows <= 256) {
      attend_join_kernel<C::DV, 16><<<(unsigned)rows, 1024, 0, st>>>(a);
    } else if (rows <= 1024) {
      attend_join_kernel<C::DV, 4><<<(unsigned)rows, 256, 0, st>>>(a);
    } else {
      attend_join_many_kernel<C::DV><<<(unsigned)joins, 256, 0, st>>>(a, per);
    }
  }
  return check_launch("attend_join");
}

template <bool F8, bool WIDE>
static int at_dims(const AttendArgs& a, int dk, bool join, hipStream_t st) {
  switch (dk) {
    case 64: return at_launch<AtCfg<64, 64, F8, WIDE>>(a, join, st);
    case 128: return at_launch<AtCfg<128, 128, F8, WIDE>>(a, join, st);
    default: return at_launch<AtCfg<192, 128, F8, WIDE>>(a, join, st);
  }
}

}  // namespace mimo

using namespace mimo;

extern "C" {

size_t mimo_cache_attend_workspace_size(int N, int heads, int kv_heads, int v_dim) {
  if (N < 1 || heads < 1 || kv_heads < 1 || v_dim < 1 || heads % kv_heads) return 256;
  const AtRoom w = at_room(128, AT_WIDE_TARGET, N, heads, kv_heads, v_dim), n = at_room(32, AT_NARROW_TARGET, N, heads, kv_heads, v_dim);
  return std::max(w.o + w.ml + w.meta, n.o + n.ml + n.meta);
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
  MIMO_REQUIRE(B >= 1 && B <= (1 << 20) && max_pages >= 1 && max_new >= 0 && (int64_t)max_pages * cache->page_size <= kMaxTokens &&
                   (int64_t)max_pages * B <= 0x7fffffff, MIMO_ERR_SHAPE,
               "cache_attend: need 1 <= B <= 2^20, max_pages >= 1, max_new >= 0, at most 2^31 - 1 table entries, 2^31 - 2^16 tokens of a request "
               "(got %d, %d, %d)",
               B, max_pages, max_new);
  MIMO_REQUIRE(window >= 0 && sink_tokens >= 0, MIMO_ERR_SHAPE, "cache_attend: window and sink_tokens must be >= 0");
  MIMO_REQUIRE(scale == scale && scale - scale == 0.0f, MIMO_ERR_ARG, "cache_attend: scale must be finite");
  MIMO_REQUIRE(q_stride >= (int64_t)heads * cache->k_dim, MIMO_ERR_SHAPE, "cache_attend: rows closer than their length");
  MIMO_REQUIRE(aligned16(q) && aligned16(out) && q_stride % 8 == 0, MIMO_ERR_ALIGN,
               "cache_attend: 16-byte alignment of q, its rows and out");
  MIMO_REQUIRE(!overlap(q, ((size_t)(N - 1) * q_stride + (size_t)heads * cache->k_dim) * 2, out, (size_t)N * heads * cache->v_dim * 2),
               MIMO_ERR_ARG, "cache_attend: out may not overlap q");
  const size_t need = mimo_cache_attend_workspace_size(N, heads, cache->kv_heads, cache->v_dim);
  MIMO_REQUIRE(ws && ws_bytes >= need, MIMO_ERR_WORKSPACE, "cache_attend: workspace %zu < %zu", ws_bytes, need);
  MIMO_REQUIRE(aligned16(ws), MIMO_ERR_ALIGN, "cache_attend: 16-byte alignment of the workspace");
  AttendArgs a{};
  a.q = q, a.q_stride = q_stride, a.N = N, a.Hq = heads, a.Hkv = cache->kv_heads, a.B = B, a.max_pages = max_pages;
  a.n_pages = cache->n_pages, a.page_shift = __builtin_ctz(cache->page_size), a.window = window, a.sinks = window ? sink_tokens : 0;
  a.starts = starts, a.lens = lens, a.table = table;
  a.k = static_cast<const uint8_t*>(cache->k), a.v = static_cast<const uint8_t*>(cache->v);
  a.k_scale = cache->k_scale, a.v_scale = cache->v_scale, a.sink_logits = sink_logits;
  a.scale = scale, a.out = out, a.status = status;
  // narrow tiles hold the rows of a request in 32, wide ones are up to a quarter filled: at 5 to 8 rows of 8 heads the wide
  // ones take 132-136 us for 32 requests of 4000 keys, two and more narrow tiles 136-139, and at 12 143 against 356
  const bool wide = (int64_t)std::min(max_new, N) * (heads / cache->kv_heads) > 32;
  at_tiles(wide ? 128 : 32, N, heads, cache->kv_heads, a);
  a.target = wide ? AT_WIDE_TARGET : AT_NARROW_TARGET;
  // no tile can walk more units than the table or the window holds; where none has to be split there is no second launch
  const int most = at_most((int64_t)max_pages * cache->page_size, window, a.sinks, a.TQ, wide ? 64 : 128);
  const bool join = most > (wide ? AT_WIDE_MIN : AT_NARROW_MIN);
  const AtRoom room = at_room(wide ? 128 : 32, a.target, N, heads, cache->kv_heads, cache->v_dim);
  char* w = static_cast<char*>(ws);
  a.part_o = reinterpret_cast<float*>(w);
  a.part_ml = reinterpret_cast<float*>(w + room.o);
  a.meta = join ? reinterpret_cast<int2*>(w + room.o + room.ml) : nullptr;
  hipStream_t st = as_stream(stream);
  const bool f8 = cache->dtype == MIMO_KV_E4M3;
  if (wide) return f8 ? at_dims<true, true>(a, cache->k_dim, join, st) : at_dims<false, true>(a, cache->k_dim, join, st);
  return f8 ? at_dims<true, false>(a, cache->k_dim, join, st) : at_dims<false, false>(a, cache->k_dim, join, st);
}

}  // extern "C"
