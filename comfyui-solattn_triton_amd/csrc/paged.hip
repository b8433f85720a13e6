// Attention of one new token of each sequence over a key-value cache, paged or
// contiguous, of 16-bit values or of 8-bit codes: the visible keys are split over
// workgroups and waves, each with an online softmax of its own, and joined.
//
// Per sequence b the token sits at position len - 1 and sees the keys j < len,
// with a window those with j >= len - window or j < sinks. A query head shares its
// kv head with group - 1 others; these (up to 16) are the columns of the tiles.
// Sequences may have their first keys in common (`shared` of them, runs of `per`
// sequences): the heads of all of a run are then the columns of these keys, which
// are read once for 16 columns, for 32, or for 128 (paged_tiles.hpp), and what is
// behind them is attended as before, in the same launch; the join takes both. A column sees
// a part of the shared keys whole or not at all: of a sequence that ends inside a part, what it
// has of that part is with its own keys. (One product for all columns would take 0 times what
// is behind its end, and that may be a NaN or an infinity that another sequence does see.)
//
// Bound: HBM, 2 Hkv D values a visible key; the matrix instructions do 16 query
// columns whether they exist or not, 256 of their cycles for 16 KiB of a 16-bit cache.
//   bf16: four sequences of 32768 to 131072 tokens, 24 heads over 8 of 128 channels:
//     238-251 us, 5.3-5.6 TB/s (a large copy reaches 5.0-5.15); 32 of 512 to 16384, 16
//     heads of 64 over 4, pages of 16: 64 us; one sequence with a window of 4096: 10.2
//     us, two launches of the host's (kernels 6.5 and 4.5).
//   Codes: the four, e4m3: 138 us, 4.9 TB/s, kernel 135. The 32, int8: 39 us, 3.6 TB/s,
//     kernel 30-37 and join 5 (the vector units, 60% busy with a byte's way to a 16-bit
//     float, are not what it waits for: fewer of their instructions, or sequences of one
//     length, took as long). One with a window of 4096: 8.9 us, kernels 6.1 and 2.8.
//   Shared keys: 8 sequences of 24 heads over 8 behind 4096 bf16 keys: 13 us (22 as if
//     nothing was shared), latency: 10.6 of it the kernel, a chain of lengths, page ids,
//     keys and steps, and 2-4 the join. 64 in groups over int8: 19-21 us (48), latency
//     beside the conversions. 256 behind 32760 bf16 keys: 170-178 us, in some runs up to 192
//     (2600), products.
// A wave takes 32 keys at a time straight from HBM into operand registers, no LDS:
//   S^T = K Q^T (v_mfma_f32_16x16x32): row r of tile t is key 8 (r/4) + 4 t + r%4
//     of the 32, so lane (q, g) = (lane % 16, lane / 16) gets the scores of the
//     keys 8 g + 0..7: the order in which P is the B operand of the next product;
//   O^T += V^T P^T: a lane reads the same keys 8 g + 0..7, D / 16 channels each,
//     and transposes them in registers (v_perm_b32), one A operand per channel of
//     the D / 16: row i of operand j is channel (D / 16) i + j.
// The row's statistics need an exchange between the lanes g only. Codes become operands
// as they are (integers up to 127 and e4m3's values are exact in 16 bits); K's power of
// two multiplies the score, V's the weight.
#include "paged_tiles.hpp"

namespace solattn {
namespace {

constexpr int kWaves = 4;
constexpr int kStep = 32;       // keys of a wave's step
constexpr int kMaxSplits = 64;  // parts of a row over its own keys
constexpr int kMaxShared = 64;  // and over shared ones
constexpr int kGroups = 16;     // query columns of a tile

// What the cache holds: 16-bit values of the queries' type, or codes (cache8.hpp).
struct SameType {};
template <typename C>
constexpr bool kCodes = !__is_same(C, SameType);

struct PagedArgs {
  const uint16_t* q;
  int64_t sq_b, sq_h;
  const uint8_t* k;          // strides in bytes
  int64_t sk_p, sk_s, sk_h;
  const uint8_t* v;
  int64_t sv_p, sv_s, sv_h;
  const uint8_t* ks;         // codes: exponent bytes
  int64_t ks_p, ks_h;
  const uint8_t* vs;
  int64_t vs_p, vs_h;
  const int32_t* table;      // null: sequence b is page b
  int64_t table_b;
  const int32_t* lengths;    // with a table: each sequence's. Without: one shorter than `length` holds no token
                             // here, the others `length` keys (null: all of them)
  int length, pages, page, max_pages;
  Divisor by_page;
  int ranked;                // longest sequences first, where one has that many keys (0: never)
  int near;                  // pages' and slots' strides are within 32 bits
  uint16_t* o;
  int64_t so_b, so_h;
  float* part;               // parts > 1: [B][H][parts][D] sums, then [B][H][parts][2] max and sum
  int64_t part_ml;           // where the latter begin
  int B, H, Hkv, D, group, tiles, split;
  Divisor by_tiles, by_hkv, by_split, by_run;  // by_run: workgroups of the same own keys
  int window, sinks;         // window 0: none
  float c;                   // scale log2(e)
  // Keys in common: of `per` sequences each the first `shared`, cut into psplit parts, for
  // ptiles tiles of columns; the launch's first pitems workgroups. parts: psplit + split.
  int shared, per, psplit, ptiles, pitems, parts;
  Divisor by_ptiles, by_psplit, by_group;
};

__device__ __forceinline__ float over_groups_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float over_groups_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The same over all 64 lanes; within 16 by lane moves, in the order of a butterfly.
template <typename F>
__device__ __forceinline__ uint32_t over_row16(uint32_t x, F&& f) {
#define SOLATTN_DPP(ctrl) \
  x = f(x, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), ctrl, 0xf, 0xf, false)))
  SOLATTN_DPP(0xB1);   // quad_perm 1 0 3 2
  SOLATTN_DPP(0x4E);   // quad_perm 2 3 0 1
  SOLATTN_DPP(0x141);  // row_half_mirror
  SOLATTN_DPP(0x140);  // row_mirror
#undef SOLATTN_DPP
  return x;
}
template <typename F>
__device__ __forceinline__ uint32_t over_wave(uint32_t x, F&& f) {
  x = over_row16(x, f);
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = f(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return f(r[0], r[1]);
}
__device__ __forceinline__ float wave_max(float x) {
  return __uint_as_float(over_wave(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ float wave_sum(float x) {
  return __uint_as_float(over_wave(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// exp2 of the distance to a maximum; a row without keys has the maximum -inf and weight 0.
__device__ __forceinline__ float weight_of(float m, float top) {
  return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
}

__device__ __forceinline__ int sequence_length(const PagedArgs& a, int b) {
  const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
  int n = a.lengths ? a.lengths[b] : a.length;
  if (!a.table) n = n < a.length ? 0 : a.length;
  return static_cast<int>(min(static_cast<int64_t>(max(n, 0)), cap));
}

// The sequence with the r-th largest length of up to 256 (of as many times 128 keys: the
// first), r from 0: built bit by bit from what lanes with up to four sequences each say. Where
// none has `ranked` keys, or the longest is not a quarter above the mean, sequence r: there is
// nothing to gain, and the search takes its own time. Its length comes out of the lane that has
// it: another round of memory would be most of a short sequence's time.
constexpr int kRanked = 256;
__device__ __forceinline__ int by_length(const PagedArgs& a, int r, int& length) {
  constexpr int U = kRanked / 64;
  const int lane = threadIdx.x & 63, cap = a.max_pages * a.page;
  int len[U];
  bool few = true;
#pragma unroll
  for (int u = 0; u < U; ++u) len[u] = 64 * u < a.B ? a.lengths[min(lane + 64 * u, a.B - 1)] : 0;
#pragma unroll
  for (int u = 0; u < U; ++u) few = few && !__any(len[u] >= a.ranked);
  const auto found = [&](int b) __attribute__((always_inline)) {
    int n = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) n = b >> 6 == u ? __builtin_amdgcn_readlane(len[u], b & 63) : n;
    length = min(max(n, 0), cap);
    return b;
  };
  if (few) return found(r);
  uint32_t key[U], top = 0, total = 0;  // keys: unique; 0 is none (sequence 255 of length 0 is the last in any case)
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = lane + 64 * u;
    key[u] = i < a.B ? static_cast<uint32_t>(min(max(len[u], 0), cap)) / 128 << 8 | (kRanked - 1 - i) : 0u;
    top = max(top, key[u]), total += key[u] >> 8;
  }
  top = __builtin_amdgcn_readfirstlane(over_wave(top, [](uint32_t x, uint32_t y) { return max(x, y); }));
  total = __builtin_amdgcn_readfirstlane(over_wave(total, [](uint32_t x, uint32_t y) { return x + y; }));
  if (4ull * a.B * (top >> 8) <= 5ull * total) return found(r);
  uint32_t nth = 0;
  for (int bit = 31 - __builtin_clz(top | 1); bit >= 0; --bit) {
    const uint32_t with = nth | 1u << bit;
    int n = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (64 * u < a.B) n += __popcll(__ballot(key[u] >= with));
    if (n > r) nth = with;
  }
  return found(kRanked - 1 - static_cast<int>(nth & (kRanked - 1)));
}

// The visible keys as steps: first those of the sinks below the window, then the window's.
struct Visible {
  int len, low;        // keys [low, len) and [0, sinks_end)
  int sinks_end;       // <= low
  int sink_steps, first, steps;  // the window's steps begin at key `first`
};
__device__ __forceinline__ Visible visible(int len, int low, int sinks) {
  constexpr int S = kStep;
  Visible s;
  s.len = len, s.low = min(low, len);
  s.sinks_end = min(sinks, s.low);
  s.sink_steps = (s.sinks_end + S - 1) / S;
  s.first = s.low & ~(S - 1);
  s.steps = s.sink_steps + (len - s.first + S - 1) / S;
  return s;
}

// The longest sequence of a run of `per` (the first of these) and its length.
__device__ __forceinline__ void longest(const PagedArgs& a, int first, int& b, int& len) {
  const int lane = threadIdx.x & 63;
  int n = -1, at = 0;
  for (int i = lane; i < a.per; i += 64) {
    const int x = sequence_length(a, first + i);
    if (x > n) n = x, at = i;
  }
  const auto larger = [](uint32_t x, uint32_t y) { return static_cast<uint32_t>(max(static_cast<int>(x), static_cast<int>(y))); };
  const int top = static_cast<int>(over_wave(static_cast<uint32_t>(n), larger));
  const uint32_t best = over_wave(n == top ? static_cast<uint32_t>(at) : ~0u, [](uint32_t x, uint32_t y) { return min(x, y); });
  b = first + __builtin_amdgcn_readfirstlane(static_cast<int>(best));
  len = __builtin_amdgcn_readfirstlane(top);
}

// Steps of a part of `keys` shared ones.
template <bool TILED>
__device__ __forceinline__ int shared_part(const PagedArgs& a, int keys) {
  constexpr int S = TILED ? kKeys : kStep;
  return a.by_psplit.of((keys + S - 1) / S + a.psplit - 1);
}
// Of a column with `len` keys: how many of the keys that the part ends with (`end`) it may see, all or none.
__device__ __forceinline__ int sees(int len, int end) { return len >= end ? INT32_MAX : 0; }

// A workgroup's keys and columns. The columns of own keys are the heads of one sequence
// that share a kv head, those of shared keys the heads of all its sequences.
struct Work {
  Visible vis;
  int step0, step1, part;
  int b, seq;          // whose pages; the first column's sequence
  int hk, col0, ncol;  // columns col0 .. col0 + ncol - 1 of the kv head
  __device__ __forceinline__ void row(const PagedArgs& a, int c, bool many, int& b, int& h) const {
    uint32_t n = col0 + min(c, ncol - 1);
    const uint32_t g = many ? a.by_group.split(n) : n;
    b = many ? seq + static_cast<int>(n) : seq;
    h = hk * a.group + static_cast<int>(g);
  }
};

// The part's steps of `keys` shared ones, on sequence b's pages.
template <bool TILED>
__device__ __forceinline__ void shared_steps(const PagedArgs& a, Work& w, int b, int keys) {
  w.b = b;
  w.vis = visible(keys, 0, 0);
  if constexpr (TILED) w.vis.steps = (keys + kKeys - 1) / kKeys;
  const int per = shared_part<TILED>(a, keys);
  w.step0 = w.part * per, w.step1 = min(w.step0 + per, w.vis.steps);
}
// What shared keys mostly are: all of them, on the first sequence's pages. The first page
// ids are asked for as if they were, beside the lengths that tell.
__device__ __forceinline__ int all_shared(const PagedArgs& a) {
  return static_cast<int>(min(static_cast<int64_t>(a.shared), static_cast<int64_t>(a.max_pages) * a.page));
}

template <int DP>
struct __align__(16) PagedLds {
  float o[kWaves][kGroups][DP + 4];
  float m[kWaves][kGroups], l[kWaves][kGroups];
};

// Nothing in this part: the join passes over a sum of 0.
template <bool MANY>
__device__ __forceinline__ void no_keys(const PagedArgs& a, const Work& w) {
  for (int c = threadIdx.x; c < w.ncol; c += kWaves * 64) {
    int b, h;
    w.row(a, c, MANY, b, h);
    reinterpret_cast<float2*>(a.part + a.part_ml)[(static_cast<int64_t>(b) * a.H + h) * a.parts + w.part] =
        make_float2(-INFINITY, 0.f);
  }
}

// DP: the head dim that the registers hold; D < DP (kFull false) leaves the rest zero.
// NT: tiles of 16 columns. MANY: the columns are of several sequences; found: w has the longest
// one's pages and steps already.
template <typename E, typename C, int DP, bool kFull, int NT, bool MANY>
__device__ __forceinline__ void attend(const PagedArgs& a, PagedLds<DP>& lds, Work& w, bool found = false) {
  constexpr bool Q8 = kCodes<C>;
  constexpr int S = kStep;
  constexpr int NC = DP / 32;           // products of a score tile
  constexpr int KL = Q8 ? NC / 2 : NC;  // 16-byte pieces of a key that a lane reads
  constexpr int CH = DP / 16;           // channels of a lane's V piece = operands of the second product
  constexpr int VW = Q8 ? CH / 4 : CH / 2;  // their registers
  constexpr int ES = Q8 ? 1 : 2;        // bytes of a value
  constexpr int NP = Q8 ? 2 : 1;        // roundings of P (below)

  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const Visible& vis = w.vis;
  const int hk = w.hk;

  // Channels of product cc that this lane holds of q and of a key: eight from
  // 32 cc + 8 g on, of codes, read 16 bytes at a time, from 64 (cc / 2) + 16 g + 8 (cc % 2).
  bf16x8 q[NT][NC];
  int hi[NT];  // MANY: the sequence's length, then keys of the part that the column sees
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    int b, h;
    w.row(a, 16 * t + col, MANY, b, h);
    const uint16_t* qp = a.q + b * a.sq_b + h * a.sq_h;
    hi[t] = MANY ? sequence_length(a, b) : 0;
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      const int ch = Q8 ? 64 * (cc >> 1) + 16 * g + 8 * (cc & 1) : 32 * cc + 8 * g;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (kFull || ch < a.D) x = *reinterpret_cast<const uint4*>(qp + ch);
      q[t][cc] = __builtin_bit_cast(bf16x8, x);
    }
  }
  f32x4 acc[NT][CH];
  float m[NT], l[NT];  // l: this lane's keys
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int j = 0; j < CH; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[t] = -INFINITY, l[t] = 0.f;
  }

  const int vch = kFull || CH * col < a.D ? CH * col : 0;
  const auto base_of = [&](int st) __attribute__((always_inline)) {
    return st < vis.sink_steps ? st * S : vis.first + (st - vis.sink_steps) * S;
  };
  // Where the eight consecutive keys from j8 on are: they share a page (its size is a
  // multiple of 8, or the page is a whole sequence). Page ids are read a step ahead, so
  // that a step waits for one round of memory, not two.
  const auto slot_of = [&](int j8, int& slot) __attribute__((always_inline)) {
    const uint32_t j = static_cast<uint32_t>(min(j8, max(vis.len - 1, 0) & ~7));
    const uint32_t pg = a.by_page.of(j);
    slot = static_cast<int>(j - pg * a.page);
    return a.table ? a.table[w.b * a.table_b + pg] : w.b;
  };
  const uint8_t* const khead = a.k + hk * a.sk_h;
  const uint8_t* const vhead = a.v + hk * a.sv_h + ES * vch;
  int kslot, vslot, kid, vid;
  const auto find = [&](int st) __attribute__((always_inline)) {
    const int base = base_of(st);
    kid = slot_of(base + 8 * (col >> 2), kslot);
    vid = slot_of(base + 8 * g, vslot);
  };
  if (w.step0 + wave < w.step1) find(w.step0 + wave);
  int safe = 0;  // MANY: keys that every column sees
  if constexpr (MANY) {
    if (!found) {
      int b, len;
      longest(a, w.seq, b, len);
      if (b != w.seq || len < vis.len) {
        shared_steps<false>(a, w, b, min(len, vis.len));
        if (w.step0 >= w.step1) return no_keys<true>(a, w);
        if (w.step0 + wave < w.step1) find(w.step0 + wave);
      }
    }
    safe = vis.len;
    const int end = min(w.step1 * S, vis.len);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      hi[t] = sees(hi[t], end);
      safe = min(safe, hi[t]);
    }
    safe = __builtin_amdgcn_readfirstlane(static_cast<int>(
        over_row16(static_cast<uint32_t>(safe), [](uint32_t x, uint32_t y) { return min(x, y); })));
  }
  for (int st = w.step0 + wave; st < w.step1; st += kWaves) {
    const bool sink = st < vis.sink_steps;
    const int base = base_of(st);
    const int lo = sink ? 0 : vis.low, end = sink ? vis.sinks_end : vis.len;  // visible: lo <= j < end
    // Keys of page ids outside the cache are not visible (a key's score lane holds its V piece too).
    uint4 kr[2][KL];
    uint32_t vr[8][VW];
    uint2 ke, ve;  // exponents of the keys 8 g + 0..7
    const auto load_k = [&](int t, const uint8_t* at) __attribute__((always_inline)) {
#pragma unroll
      for (int cc = 0; cc < KL; ++cc) {
        const int ch = Q8 ? 64 * cc + 16 * g : 32 * cc + 8 * g;
        kr[t][cc] = *reinterpret_cast<const uint4*>(at + (kFull || ch < a.D ? ES * ch : 0));
      }
    };
    const auto load_v = [&](int i, const uint8_t* at) __attribute__((always_inline)) {
      if constexpr (VW == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(at);
        vr[i][0] = x.x, vr[i][1] = x.y, vr[i][2] = x.z, vr[i][3] = x.w;
      } else if constexpr (VW == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(at);
        vr[i][0] = x.x, vr[i][1] = x.y;
      } else {
        vr[i][0] = *reinterpret_cast<const uint32_t*>(at);
      }
    };
    // A lane's rows of K are those at col % 4 and 4 further, of V eight: a slot apart, but where a
    // whole-sequence page ends among them, whose last row is read again. (Every row's place by
    // itself, in 64 bits: 82 multiplications a step, more time than all the rest of it.)
    const bool vok = vid >= 0 && vid < a.pages;
    const uint32_t kpage = kid >= 0 && kid < a.pages ? kid : 0, vpage = vok ? vid : 0;
    const int kleft = a.page - 1 - kslot, vleft = a.page - 1 - vslot;
    const auto times = [](uint32_t x, int64_t stride) { return static_cast<uint64_t>(x) * static_cast<uint32_t>(stride); };
    if (a.near && (Q8 || !__any(min(kleft, vleft) < 7))) {
      const uint8_t* kp = khead + times(kpage, a.sk_p) + times(kslot + (col & 3), a.sk_s);
      load_k(0, kp);
      load_k(1, kp + 4 * a.sk_s);
      const uint8_t* vp = vhead + times(vpage, a.sv_p) + times(vslot, a.sv_s);
#pragma unroll
      for (int i = 0; i < 8; ++i, vp += a.sv_s) load_v(i, vp);
    } else {
      const uint8_t* kp = khead + static_cast<uint64_t>(kpage) * a.sk_p;
      const uint8_t* vp = vhead + static_cast<uint64_t>(vpage) * a.sv_p;
#pragma unroll
      for (int t = 0; t < 2; ++t) load_k(t, kp + (kslot + min(4 * t + (col & 3), kleft)) * a.sk_s);
#pragma unroll
      for (int i = 0; i < 8; ++i) load_v(i, vp + (vslot + min(i, vleft)) * a.sv_s);
    }
    if constexpr (Q8) {
      ke = *reinterpret_cast<const uint2*>(a.ks + hk * a.ks_h + times(vpage, a.ks_p) + vslot);
      ve = *reinterpret_cast<const uint2*>(a.vs + hk * a.vs_h + times(vpage, a.vs_p) + vslot);
    }
    if (st + kWaves < w.step1) find(st + kWaves);
    // scores of this lane: key base + 8 g + i in element i % 4 of tile i / 4
    f32x4 s[NT][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) {
        bf16x8 kop;
        if constexpr (Q8) {
          const uint4 x = kr[i][cc >> 1];
          const uint32_t lo2 = cc & 1 ? x.z : x.x, hi2 = cc & 1 ? x.w : x.y;
          kop = __builtin_bit_cast(bf16x8, make_uint4(C::template pair<E>(lo2, 0), C::template pair<E>(lo2, 2),
                                                      C::template pair<E>(hi2, 0), C::template pair<E>(hi2, 2)));
        } else {
          kop = __builtin_bit_cast(bf16x8, kr[i][cc]);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (cc == 0) s[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
          s[t][i] = E::mfma16(kop, q[t][cc], s[t][i]);
        }
      }
    const float c = Q8 ? 1.f : a.c;  // codes: the factor is the key's
    if constexpr (Q8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = power_at(i < 4 ? ke.x : ke.y, i & 3) * a.c;
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][i >> 2][i & 3] *= f;
      }
    }
    if (base < lo || base + S > (MANY ? safe : end) || __any(!vok)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = base + 8 * g + i;
        const bool on = vok && j >= lo && j < end;
#pragma unroll
        for (int t = 0; t < NT; ++t)
          s[t][i >> 2][i & 3] = on && (!MANY || j < hi[t]) ? s[t][i >> 2][i & 3] : -INFINITY;
#pragma unroll
        for (int r = 0; r < VW; ++r) vr[i][r] = on ? vr[i][r] : 0u;  // 0 P of a value that may be anything
        if constexpr (Q8) {
          uint32_t& e = i < 4 ? ve.x : ve.y;
          e = on ? e : e & ~(0xFFu << (8 * (i & 3)));
        }
      }
    }
    float neg[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, s[t][i >> 2][i & 3]);
      const float m_new = fmaxf(m[t], over_groups_max(mx) * c);
      if (__any(m_new != m[t])) {
        const float alpha = weight_of(m[t], m_new);
        l[t] *= alpha;
#pragma unroll
        for (int j = 0; j < CH; ++j) acc[t][j] *= alpha;
        m[t] = m_new;
      }
      neg[t] = m[t] == -INFINITY ? 0.f : -m[t];
    }
    // P, of codes times V's powers in two bf16 parts: fp16 does not have their range, and
    // the sums are as near as in fp16.
    bf16x8 pb[NT][NP];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(s[t][i >> 2][i & 3], c, neg[t]));
        l[t] += p[i];
        if constexpr (Q8) p[i] *= power_at(i < 4 ? ve.x : ve.y, i & 3);
      }
      uint32_t x[4], y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = Q8 ? Bf16::pack(p[2 * r], p[2 * r + 1]) : E::pack(p[2 * r], p[2 * r + 1]);
        if constexpr (NP == 2) y[r] = Bf16::pack(p[2 * r] - Bf16::lo(x[r]), p[2 * r + 1] - Bf16::hi(x[r]));
      }
      pb[t][0] = __builtin_bit_cast(bf16x8, make_uint4(x[0], x[1], x[2], x[3]));
      if constexpr (NP == 2) pb[t][1] = __builtin_bit_cast(bf16x8, make_uint4(y[0], y[1], y[2], y[3]));
    }
#pragma unroll
    for (int j = 0; j < CH; ++j) {  // channel j of the lane's piece, its eight keys
      uint32_t x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (Q8)
          x[r] = C::across(vr[2 * r][j >> 2], vr[2 * r + 1][j >> 2], j & 3);
        else
          x[r] = __builtin_amdgcn_perm(vr[2 * r + 1][j >> 1], vr[2 * r][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
      }
      const bf16x8 vop = __builtin_bit_cast(bf16x8, make_uint4(x[0], x[1], x[2], x[3]));
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int n = 0; n < NP; ++n)
          acc[t][j] = Q8 ? Bf16::mfma16(vop, pb[t][n], acc[t][j]) : E::mfma16(vop, pb[t][n], acc[t][j]);
    }
  }

  // Join the waves, a tile of columns at a time: O[q][channel], channel CH (4 g + i) + j in
  // acc[j][i]. A thread takes four channels of a column.
  constexpr int L = DP / 4;
  const int ch = 4 * (threadIdx.x % L);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t) __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < CH; j += 4)
        *reinterpret_cast<float4*>(&lds.o[wave][col][CH * (4 * g + i) + j]) =
            make_float4(acc[t][j][i], acc[t][j + 1][i], acc[t][j + 2][i], acc[t][j + 3][i]);
    const float sum_l = over_groups_sum(l[t]);
    if (g == 0) {
      lds.m[wave][col] = m[t];
      lds.l[wave][col] = sum_l;
    }
    __syncthreads();
    if (!kFull && ch >= a.D) continue;
    for (int qc = threadIdx.x / L; qc < min(kGroups, w.ncol - 16 * t); qc += kWaves * 64 / L) {
      float top = lds.m[0][qc];
#pragma unroll
      for (int i = 1; i < kWaves; ++i) top = fmaxf(top, lds.m[i][qc]);
      float o[4] = {}, sum = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        const float f = weight_of(lds.m[i][qc], top);
        const float4 x = *reinterpret_cast<const float4*>(&lds.o[i][qc][ch]);
        o[0] = fmaf(x.x, f, o[0]), o[1] = fmaf(x.y, f, o[1]), o[2] = fmaf(x.z, f, o[2]), o[3] = fmaf(x.w, f, o[3]);
        sum = fmaf(lds.l[i][qc], f, sum);
      }
      int b, h;
      w.row(a, 16 * t + qc, MANY, b, h);
      if (a.parts > 1) {
        const int64_t at = (static_cast<int64_t>(b) * a.H + h) * a.parts + w.part;
        *reinterpret_cast<float4*>(a.part + at * a.D + ch) = make_float4(o[0], o[1], o[2], o[3]);
        if (ch == 0) *reinterpret_cast<float2*>(a.part + a.part_ml + 2 * at) = make_float2(top, sum);
      } else {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no visible key: zeros
        *reinterpret_cast<uint2*>(a.o + b * a.so_b + h * a.so_h + ch) =
            make_uint2(E::pack(o[0] * inv, o[1] * inv), E::pack(o[2] * inv, o[3] * inv));
      }
    }
  }
}

// Whether fp16 holds the largest values of codes of a part's keys [first, end). Two bytes a key
// and two rounds of memory in front of the first tile: 256 fp16 sequences of 24 heads behind
// 32760 int8 keys 204 -> 197 us, of 16 heads of 64 behind 8000 of e4m3 42.1 -> 42.5. Where one
// page of these is beyond fp16 they take 307 and 55.
template <typename C>
__device__ __forceinline__ bool fp16_holds(const PagedArgs& a, const Work& w, uint32_t* any, int first, int end) {
  bool over = false;
  for (int j = first + 8 * static_cast<int>(threadIdx.x); j < end; j += 8 * kWaves * 64) {
    const uint32_t pg = a.by_page.of(static_cast<uint32_t>(j));
    const int64_t slot = j - static_cast<int64_t>(pg) * a.page, id = a.table[w.b * a.table_b + pg];
    if (id < 0 || id >= a.pages) continue;
    const uint2 k = *reinterpret_cast<const uint2*>(a.ks + w.hk * a.ks_h + id * a.ks_p + slot);
    const uint2 v = *reinterpret_cast<const uint2*>(a.vs + w.hk * a.vs_h + id * a.vs_p + slot);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t kb = (i < 4 ? k.x : k.y) >> (8 * (i & 3)) & 0xFFu, vb = (i < 4 ? v.x : v.y) >> (8 * (i & 3)) & 0xFFu;
      over = over || (j + i < end && max(kb, vb) > C::kFp16Byte);
    }
  }
  any[wave_id()] = __any(over);
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) all |= any[i];
  __syncthreads();  // (the LDS is the tiles')
  return all == 0;
}

// The same for 128 columns of several sequences, by tiles in LDS: steps of 64 keys. Codes
// become values of the queries' type there, which fp16 may not hold: a part that has such keys
// goes as fewer columns do, where the powers stay apart, 32 columns at a time.
constexpr int kTiled = kTileRows / kGroups;  // its tiles of columns
template <typename E, typename C, int D>
__device__ __forceinline__ void attend_many(const PagedArgs& a, uint8_t* lds, Work& w) {
  static_assert(kWaves * 64 == kTileThreads, "a wave for 32 rows");
  const int lane = threadIdx.x & 63, half = lane >> 5, row = 32 * wave_id() + (lane & 31);
  int b, h;
  w.row(a, row, true, b, h);
  bf16x8 q[D / 16];
  load_row<D>(q, a.q + b * a.sq_b + h * a.sq_h, half);
  int hi = sequence_length(a, b);
  const auto near = [&](int64_t slot) { return a.near && slot < (1 << 28); };
  const TileSource ks{a.k + w.hk * a.sk_h, a.sk_p, a.sk_s, a.ks + w.hk * a.ks_h, a.ks_p, near(a.sk_s)};
  const TileSource vs{a.v + w.hk * a.sv_h, a.sv_p, a.sv_s, a.vs + w.hk * a.vs_h, a.vs_p, near(a.sv_s)};
  TilePages pg{a.table + w.b * a.table_b, a.by_page, a.pages, w.vis.len};
  TileLds<D>& ring = *reinterpret_cast<TileLds<D>*>(lds);
  if constexpr (!kCodes<C>) pg.fetch_ids(ring.ids, w.step0 * kKeys, 0);
  {
    int best, len;
    longest(a, w.seq, best, len);
    if (best != w.seq || len < w.vis.len) {
      shared_steps<true>(a, w, best, min(len, w.vis.len));
      if (w.step0 >= w.step1) return no_keys<true>(a, w);
      pg.table = a.table + w.b * a.table_b, pg.end = w.vis.len;
      if constexpr (!kCodes<C>) pg.fetch_ids(ring.ids, w.step0 * kKeys, 0);
    }
  }
  if constexpr (kCodes<C> && __is_same(E, Fp16)) {
    if (!fp16_holds<C>(a, w, reinterpret_cast<uint32_t*>(lds), w.step0 * kKeys, min(w.step1 * kKeys, w.vis.len))) {
      const int col0 = w.col0, ncol = w.ncol;
      w.vis = visible(w.vis.len, 0, 0);
      w.step0 *= kKeys / kStep, w.step1 = min(w.step1 * (kKeys / kStep), w.vis.steps);
#pragma unroll 1
      for (int c = 0; c < ncol; c += 2 * kGroups) {
        if (c) __syncthreads();  // (the last columns' sums are read from LDS)
        w.col0 = col0 + c, w.ncol = min(2 * kGroups, ncol - c);
        attend<E, C, D, true, 2, true>(a, *reinterpret_cast<PagedLds<D>*>(lds), w, true);
      }
      return;
    }
  }
  hi = sees(hi, min(w.step1 * kKeys, w.vis.len));
  const int safe = __builtin_amdgcn_readfirstlane(static_cast<int>(
      over_wave(static_cast<uint32_t>(hi), [](uint32_t x, uint32_t y) { return min(x, y); })));
  RowState<D / 32> st;
  if constexpr (kCodes<C>) {
    const uint32_t kb = lds_addr(lds), vb = kb + 2 * kKeys * D;
    attend_codes<E, C, D>(st, q, kb, vb, ks, vs, pg, w.step0, w.step1 - w.step0, hi, safe, a.c);
  } else {
    attend_ring<E, D>(st, q, ring, ks, vs, pg, w.step0, w.step1 - w.step0, hi, safe, a.c);
  }
  const float l = xhalf_sum(st.l);
  if (row >= w.ncol) return;
  const int64_t at = (static_cast<int64_t>(b) * a.H + h) * a.parts + w.part;
  float* p = a.part + at * D + 4 * half;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x16& x = st.acc[dt];
      *reinterpret_cast<float4*>(p + 32 * dt + 8 * i) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
  if (half == 0)
    *reinterpret_cast<float2*>(a.part + a.part_ml + 2 * at) = make_float2(l == 0.f ? -INFINITY : st.m, l);
}

// PT: tiles of 16 columns over shared keys (0: a launch without any; kTiled: by tiles in LDS).
template <typename E, typename C, int DP, bool kFull, int PT>
__global__ void __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
paged_kernel(const PagedArgs a) {
  constexpr bool TILED = PT == kTiled;
  constexpr size_t kTileLds = !TILED ? 0 : kCodes<C> ? 4 * kKeys * DP : sizeof(TileLds<DP>);
  constexpr size_t kLds = kTileLds > sizeof(PagedLds<DP>) ? kTileLds : sizeof(PagedLds<DP>);
  __shared__ __align__(256) uint8_t lds_bytes[kLds];
  PagedLds<DP>& lds = *reinterpret_cast<PagedLds<DP>*>(lds_bytes);
  // (over 16-bit pages the compiler's own loads are sooner done, 128 sequences of 128 keys 14.9 ->
  // 14.5 us; over codes and behind shared keys they are not, 39.4 -> 39.0)
  if constexpr (PT > 0 || kCodes<C>) fetch_arguments(a);
  uint32_t n = blockIdx.x;
  Work w;
  if constexpr (PT > 0) {
    if (n < static_cast<uint32_t>(a.pitems)) {
      // an XCD (they are dealt round robin) takes a run of items: the tiles over the same keys side by side
      const uint32_t x = n & 7u, q8 = a.pitems >> 3, rem = a.pitems & 7u;
      n = x * q8 + min(x, rem) + (n >> 3);
      const int tile = a.by_ptiles.split(n);
      w.hk = a.by_hkv.split(n);
      w.part = a.by_psplit.split(n);
      w.seq = static_cast<int>(n) * a.per;
      w.col0 = tile * 16 * PT;
      w.ncol = min(16 * PT, a.per * a.group - w.col0);
      // (a part that the longest sequence may have keys for; whether it does is found out there)
      shared_steps<TILED>(a, w, w.seq, all_shared(a));
      if (w.step0 >= w.step1)
        no_keys<true>(a, w);
      else if constexpr (TILED)
        attend_many<E, C, DP>(a, lds_bytes, w);
      else
        attend<E, C, DP, kFull, PT, true>(a, lds, w);
      return;
    }
    n -= a.pitems;
  }
  if constexpr (kCodes<C>) {
    // kv heads of the same keys on one XCD, side by side: their rows and exponents share
    // lines (32 ragged sequences of 4 heads of 64 channels, pages of 16: 54.6 -> 45.5 us).
    const uint32_t x = n & 7u;
    uint32_t i = n >> 3;
    const uint32_t in_run = a.by_run.split(i), run = 8 * i + x;  // runs of the kv heads, dealt round robin
    if (run < (static_cast<uint32_t>(a.B * a.split) & ~7u)) n = run * a.by_run.d + in_run;
  }
  const int tile = a.by_tiles.split(n);
  w.hk = a.by_hkv.split(n);
  const int split = a.by_split.split(n);
  w.part = a.psplit + split;
  int len;
  if (a.ranked)
    w.b = by_length(a, n, len);
  else
    w.b = static_cast<int>(n), len = sequence_length(a, w.b);
  w.seq = w.b;
  w.col0 = tile * kGroups;
  w.ncol = min(kGroups, a.group - w.col0);
  int low = PT > 0 ? a.shared : a.window ? max(len - a.window, 0) : 0;
  if constexpr (PT > 0) {
    if (len > 0 && len < all_shared(a)) {  // from where the part begins that it ends in, on the pages of the longest
      int best, top;
      longest(a, w.seq - w.seq % a.per, best, top);
      const int keys = min(top, all_shared(a)), part = shared_part<TILED>(a, keys) * (TILED ? kKeys : kStep);
      low = len < keys ? len - len % part : len;
      w.b = best;
    }
  }
  w.vis = visible(len, low, PT > 0 ? 0 : a.sinks);
  const int per = a.by_split.of(w.vis.steps + a.split - 1);
  w.step0 = split * per, w.step1 = min(w.step0 + per, w.vis.steps);
  if (w.step0 >= w.step1 && a.parts > 1)
    no_keys<false>(a, w);
  else
    attend<E, C, DP, kFull, 1, false>(a, lds, w);
}

// Joins the parts of a row: a wave per (b, head), two channels a lane.
template <typename E>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedArgs a) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= static_cast<int64_t>(a.B) * a.H) return;
  const int lane = threadIdx.x & 63, ch = 2 * lane;
  const float2* ml = reinterpret_cast<const float2*>(a.part + a.part_ml) + row * a.parts;
  const float2 mine = lane < a.parts ? ml[lane] : make_float2(-INFINITY, 0.f);  // (parts <= 64)
  const float top = wave_max(mine.x), f = weight_of(mine.x, top), sum = wave_sum(mine.y * f);
  const bool on = ch < a.D;
  const float* p = a.part + row * a.parts * a.D + (on ? ch : 0);
  float o0 = 0.f, o1 = 0.f;
  // Splits behind the last that saw a key are not read (one without steps wrote no sums);
  // eight loads in flight, those past the last read it again and weigh 0.
  const uint64_t seen = __ballot(mine.x != -INFINITY);
  const int used = seen ? 64 - __clzll(seen) : 0;
  for (int i0 = 0; i0 < used; i0 += 8) {
    float2 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      x[u] = *reinterpret_cast<const float2*>(p + static_cast<int64_t>(min(i0 + u, used - 1)) * a.D);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float fi = i0 + u < used ? __shfl(f, i0 + u) : 0.f;  // (parts <= 64, so i0 + u < 64)
      o0 = fmaf(x[u].x, fi, o0);
      o1 = fmaf(x[u].y, fi, o1);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (on)
    *reinterpret_cast<uint32_t*>(a.o + (row / a.H) * a.so_b + (row % a.H) * a.so_h + ch) = E::pack(o0 * inv, o1 * inv);
}

// The same in one round of memory: a workgroup per row, a thread asks for every
// kJoinThreads / (D / 4)-th part at once, four channels of each, and LDS adds them up.
constexpr int kMaxParts = kMaxSplits + kMaxShared, kJoinThreads = 256;
template <typename E, int L, int N>  // L: threads of a part; N: parts of a thread
__global__ void __launch_bounds__(kJoinThreads) paged_wide_join_kernel(const PagedArgs a) {
  constexpr int G = kJoinThreads / L;
  __shared__ float f[kMaxParts];
  __shared__ __align__(16) float sums[G][4 * L];
  const uint32_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, g = threadIdx.x / L, ch = 4 * (threadIdx.x % L);
  const float2* ml = reinterpret_cast<const float2*>(a.part + a.part_ml) + static_cast<int64_t>(row) * a.parts;
  const float* p = a.part + static_cast<int64_t>(row) * a.parts * a.D + min(ch, a.D - 4);
  const float2 m0 = lane < a.parts ? ml[lane] : make_float2(-INFINITY, 0.f);
  const float2 m1 = lane + 64 < a.parts ? ml[lane + 64] : make_float2(-INFINITY, 0.f);  // (parts <= 128)
  float4 x[N];
#pragma unroll
  for (int n = 0; n < N; ++n)
    x[n] = *reinterpret_cast<const float4*>(p + static_cast<int64_t>(min(g + G * n, a.parts - 1)) * a.D);
  const float top = wave_max(fmaxf(m0.x, m1.x)), f0 = weight_of(m0.x, top), f1 = weight_of(m1.x, top);
  const float sum = wave_sum(fmaf(m0.y, f0, m1.y * f1));
  if (threadIdx.x < 64) f[lane] = f0, f[lane + 64] = f1;
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const float fi = g + G * n < a.parts ? f[g + G * n] : 0.f;
    // (a part without keys of this row is passed over: it may hold anything)
    if (fi != 0.f) o.x = fmaf(x[n].x, fi, o.x), o.y = fmaf(x[n].y, fi, o.y), o.z = fmaf(x[n].z, fi, o.z), o.w = fmaf(x[n].w, fi, o.w);
  }
  *reinterpret_cast<float4*>(&sums[g][ch]) = o;
  __syncthreads();
  if (g || ch >= a.D) return;
#pragma unroll
  for (int i = 1; i < G; ++i) {
    const float4 y = *reinterpret_cast<const float4*>(&sums[i][ch]);
    o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(a.o + static_cast<int64_t>(row / a.H) * a.so_b + (row % a.H) * a.so_h + ch) =
      make_uint2(E::pack(o.x * inv, o.y * inv), E::pack(o.z * inv, o.w * inv));
}

// Splits of a sequence: as many as leave the launch within four workgroups a CU, eight
// in a batch of sixteen or more, whose sequences are rarely of one length; of at least a
// step a wave as long as the longest sequence allows. (Within four against one more
// split: three sequences of 32768 keys 84 -> 81 us, five 138 -> 127. Within eight against four: 32
// ragged sequences of up to 16384 keys 61 -> 56, 72 of up to 4096 156 -> 134; 96 of
// 4096 each 275 -> 284. Four of 32768 to 131072: within two 281, four 250, eight 258.)
// No split is longer than 4096 keys as far as there may be 64 of them: one long sequence
// in a large batch is not left to one workgroup a head.
// Over codes eight in any batch: a split of as many keys is half the bytes (eight sequences
// of up to 32760 keys 80 -> 73 us, four of 131072 148 -> 143; more than eight, 32 of up to
// 16384 39 -> 41, fewer 46).
int splits(int64_t B, int64_t Hkv, int64_t tiles, int64_t most, int64_t window, int64_t sinks, bool codes) {
  const int64_t keys = window && window < most && sinks < most - window ? window + sinks : most;
  const int64_t steps = cdiv(keys, kStep) + 1;
  int64_t n = (B < 16 && !codes ? 1024 : 2048) / (B * Hkv * tiles);
  if (n < cdiv(keys, 4096)) n = cdiv(keys, 4096);
  if (n > steps / kWaves) n = steps / kWaves;
  if (n > kMaxSplits) n = kMaxSplits;
  return n < 1 ? 1 : static_cast<int>(n);
}

// How a call is cut.
struct Cut {
  int64_t tiles, split;
  int64_t ctiles, ptiles, psplit;  // shared keys (0: none): tiles of 16 columns in a workgroup, tiles of columns, splits
  int64_t parts() const { return psplit + split; }
  int64_t part_bytes(int64_t B, int64_t H, int64_t D) const { return parts() > 1 ? B * H * parts() * (D + 2) * 4 : 0; }
};
// Shared keys: up to 16 columns are one tile, up to 64 tiles of 32, whose keys come straight
// from HBM; more are tiles of 128 in LDS (of 64 or 128 channels). Splits end with a round of
// a workgroup's steps (four waves; a tile): a wave with a step more than the others is
// waited for.
Cut cut(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t keys, int64_t window, int64_t sinks, int64_t shared,
        int64_t groups, int cache_type) {
  Cut c{};
  c.tiles = cdiv(H / Hkv, kGroups);
  if (shared > keys) shared = keys;
  if (shared > 0) keys -= shared;
  c.split = splits(B, Hkv, c.tiles, keys, window, sinks, cache_type != 0);
  if (shared <= 0) return c;
  const int64_t cols = B / groups * (H / Hkv);
  const bool tiled = cols > 4 * kGroups && (D == 64 || D == 128);
  c.ctiles = tiled ? kTiled : cols > kGroups ? 2 : 1;
  c.ptiles = cdiv(cols, kGroups * c.ctiles);
  const int64_t steps = cdiv(shared, tiled ? kKeys : kStep), round = tiled ? 1 : kWaves, items = groups * Hkv * c.ptiles;
  const auto within = [&](int64_t most) {
    int64_t n = most / items;
    n = n < 1 ? 1 : n > kMaxShared ? kMaxShared : n;
    return cdiv(steps, round * cdiv(steps, round * n));
  };
  // One workgroup a CU where two would leave a wave less than some four steps: 8 sequences of
  // 24 heads behind 4100 keys 13.2 us, within two 15. Else two: 64 in four runs of 16 heads of
  // 64 behind 8000 int8 / e4m3 / fp16 keys 22.5 / 21.4 / 22.4 us, within two 20.4 / 19.4 / 19.1;
  // 16 behind 32760 int8 / bf16 keys 38 / 43 and 35 / 43; 64 in eight runs behind 4100 31 and
  // 32. One again for more columns of other head dims than 64 and 128 (192 of 96 channels
  // behind 8000 35 us, within two 38). Tiles: two where that leaves each twelve tiles (64 sequences of 24 heads
  // behind 32760 keys 62 against 70; 32 behind 4100 21 against 18), one and a half where
  // enough own keys take the other places meanwhile. That is by what both take, own bytes
  // against products: 256 sequences behind 32760 with up to 250 / 500 / 1000 of their own 163 /
  // 171 / 219 us, within two 163 / 187 / 245; behind 131071 with 500 / 2000 564 / 616 and 522 /
  // 645; over e4m3 with 500 196 and 190; 512 of 16 heads of 64 over 4 with 240 148 and 122.
  const int64_t two = within(512);
  if (!tiled)
    c.psplit = cols <= 4 * kGroups && steps > 3 * kWaves * two ? two : within(256);
  else if (steps < 12 * two)
    c.psplit = within(256);
  else
    c.psplit = 150 * keys * (cache_type ? 1 : 2) > shared * (H / Hkv) ? within(384) : two;
  return c;
}

// The kernel of a head dim: <channels of the registers, all of them used>.
template <typename E, typename C, int PT>
auto kernel_of(int64_t D) {
  if constexpr (PT == kTiled)
    return D == 128 ? paged_kernel<E, C, 128, true, PT> : paged_kernel<E, C, 64, true, PT>;
  else
    return D == 128  ? paged_kernel<E, C, 128, true, PT>
           : D == 64 ? paged_kernel<E, C, 64, true, PT>
           : D > 64  ? paged_kernel<E, C, 128, false, PT>
                     : paged_kernel<E, C, 64, false, PT>;
}
template <typename E, typename C>
auto kernel_of(int64_t D, int64_t ctiles) {
  return ctiles == 0   ? kernel_of<E, C, 0>(D)
         : ctiles == 1 ? kernel_of<E, C, 1>(D)
         : ctiles == 2 ? kernel_of<E, C, 2>(D)
                       : kernel_of<E, C, kTiled>(D);
}
template <typename E>
auto wide_join_of(int64_t D, int64_t parts) {
  return D > 64 ? (parts <= 32 ? paged_wide_join_kernel<E, 32, 4> : paged_wide_join_kernel<E, 32, 16>)
                : (parts <= 64 ? paged_wide_join_kernel<E, 16, 4> : paged_wide_join_kernel<E, 16, 8>);
}
template <typename E>
auto kernel_of(int64_t D, int64_t ctiles, int cache_type) {
  return cache_type == 0              ? kernel_of<E, SameType>(D, ctiles)
         : cache_type == SOLATTN_INT8 ? kernel_of<E, Int8Codes>(D, ctiles)
                                      : kernel_of<E, Fp8Codes>(D, ctiles);
}

}  // namespace

int paged_attn(const PagedCall& p, hipStream_t s, const char* what) {
  const int64_t B = p.B, H = p.H, Hkv = p.Hkv, D = p.D;
  SOLATTN_REQUIRE(p.dtype == SOLATTN_BF16 || p.dtype == SOLATTN_FP16, SOLATTN_EINVAL, "%s: dtype %d", what, p.dtype);
  SOLATTN_REQUIRE(p.cache_type == 0 || p.cache_type == SOLATTN_INT8 || p.cache_type == SOLATTN_E4M3, SOLATTN_EINVAL,
                  "%s: cache type %d", what, p.cache_type);
  SOLATTN_REQUIRE(B > 0 && H > 0 && Hkv > 0 && H % Hkv == 0, SOLATTN_EINVAL,
                  "%s: %lld query heads over %lld kv heads", what, (long long)H, (long long)Hkv);
  SOLATTN_REQUIRE(B < (1ll << 31) && H < (1ll << 31) && B * H < (1ll << 31), SOLATTN_EUNSUPPORTED, "%s: grid too large",
                  what);
  const int64_t whole = p.cache_type ? 16 : 8;
  SOLATTN_REQUIRE(D >= whole && D <= 128 && D % whole == 0, SOLATTN_EUNSUPPORTED,
                  "%s: head_dim %lld (multiples of %lld up to 128)", what, (long long)D, (long long)whole);
  SOLATTN_REQUIRE(p.window >= 0 && p.sinks >= 0 && p.window < (1ll << 31) && p.sinks < (1ll << 31), SOLATTN_EINVAL,
                  "%s: window %lld, sinks %lld", what, (long long)p.window, (long long)p.sinks);
  SOLATTN_REQUIRE(p.pages > 0 && p.pages < (1ll << 31) && p.page_size > 0 && p.max_pages >= 0 &&
                      (!p.table || p.page_size % 8 == 0),
                  SOLATTN_EINVAL, "%s: %lld pages of %lld (a multiple of 8)", what, (long long)p.pages,
                  (long long)p.page_size);
  // (what is counted past the last key: the rest of a step; of shared keys a tile's, or the next of 256 threads' eight)
  const int64_t past = p.shared ? 8 * kWaves * 64 : kStep;
  SOLATTN_REQUIRE(p.page_size < (1ll << 31) && p.max_pages < (1ll << 31) && p.max_pages * p.page_size < (1ll << 31) - past,
                  SOLATTN_EUNSUPPORTED, "%s: sequences beyond 2^31 keys", what);
  SOLATTN_REQUIRE(p.shared >= 0 && p.shared < (1ll << 31), SOLATTN_EINVAL, "%s: %lld shared keys", what, (long long)p.shared);
  SOLATTN_REQUIRE(p.shared == 0 || (p.window == 0 && p.sinks == 0), SOLATTN_EINVAL, "%s: shared keys and a window", what);
  SOLATTN_REQUIRE(p.shared == 0 || (p.groups > 0 && B % p.groups == 0), SOLATTN_EINVAL,
                  "%s: %lld sequences in %lld groups", what, (long long)B, (long long)p.groups);
  SOLATTN_REQUIRE(p.scale > 0.f, SOLATTN_EINVAL, "%s: scale %g", what, static_cast<double>(p.scale));
  SOLATTN_REQUIRE(p.q && p.k && p.v && p.o, SOLATTN_EINVAL, "%s: null pointer", what);
  const auto rows = [](const void* at, int64_t x, int64_t y, int64_t z, int64_t m) {
    return reinterpret_cast<uintptr_t>(at) % 16 == 0 && x % m == 0 && y % m == 0 && z % m == 0;
  };
  SOLATTN_REQUIRE(rows(p.q, p.sq_b, p.sq_h, 0, 8) && rows(p.k, p.sk_p, p.sk_s, p.sk_h, whole) &&
                      rows(p.v, p.sv_p, p.sv_s, p.sv_h, whole) && rows(p.o, p.so_b, p.so_h, 0, 8),
                  SOLATTN_EINVAL, "%s: rows must be 16-byte aligned with strides multiple of %lld", what, (long long)whole);
  const auto scales = [](const void* at, int64_t x, int64_t y) {
    return at && reinterpret_cast<uintptr_t>(at) % 8 == 0 && x % 8 == 0 && y % 8 == 0;
  };
  SOLATTN_REQUIRE(!p.cache_type || (scales(p.ks, p.ks_p, p.ks_h) && scales(p.vs, p.vs_p, p.vs_h)), SOLATTN_EINVAL,
                  "%s: scales must be 8-byte aligned with strides multiple of 8", what);
  PagedArgs a{};
  const int64_t es = p.cache_type ? 1 : 2;
  a.q = p.q, a.sq_b = p.sq_b, a.sq_h = p.sq_h;
  a.k = static_cast<const uint8_t*>(p.k), a.sk_p = es * p.sk_p, a.sk_s = es * p.sk_s, a.sk_h = es * p.sk_h;
  a.v = static_cast<const uint8_t*>(p.v), a.sv_p = es * p.sv_p, a.sv_s = es * p.sv_s, a.sv_h = es * p.sv_h;
  a.ks = p.ks, a.ks_p = p.ks_p, a.ks_h = p.ks_h;
  a.vs = p.vs, a.vs_p = p.vs_p, a.vs_h = p.vs_h;
  a.table = p.table, a.table_b = p.table_stride;
  a.lengths = p.lengths, a.length = static_cast<int>(p.length);
  a.pages = static_cast<int>(p.pages), a.page = static_cast<int>(p.page_size), a.max_pages = static_cast<int>(p.max_pages);
  a.by_page = divisor(p.page_size);
  const auto u32 = [](int64_t x) { return x >= 0 && x < (1ll << 32); };
  a.near = u32(a.sk_p) && u32(a.sk_s) && u32(a.sv_p) && u32(a.sv_s);
  SOLATTN_REQUIRE(!p.cache_type || (u32(p.ks_p) && u32(p.vs_p)), SOLATTN_EUNSUPPORTED,
                  "%s: pages' scales 2^32 bytes apart", what);
  a.o = p.o, a.so_b = p.so_b, a.so_h = p.so_h;
  a.B = static_cast<int>(B), a.H = static_cast<int>(H), a.Hkv = static_cast<int>(Hkv), a.D = static_cast<int>(D);
  a.group = static_cast<int>(H / Hkv);
  a.window = static_cast<int>(p.window), a.sinks = static_cast<int>(p.sinks);
  a.c = p.scale * kLog2e;
  const Cut c = cut(B, H, Hkv, D, p.max_pages * p.page_size, p.window, p.sinks, p.shared, p.groups, p.cache_type);
  a.tiles = static_cast<int>(c.tiles), a.split = static_cast<int>(c.split);
  a.by_tiles = divisor(c.tiles), a.by_hkv = divisor(Hkv), a.by_split = divisor(c.split), a.by_run = divisor(Hkv * c.tiles);
  a.parts = static_cast<int>(c.parts());
  const int64_t need = c.part_bytes(B, H, D);
  SOLATTN_REQUIRE(need == 0 || (p.workspace && p.workspace_bytes >= need), SOLATTN_ESIZE,
                  "%s: workspace %lld < %lld bytes", what, (long long)p.workspace_bytes, (long long)need);
  SOLATTN_REQUIRE(reinterpret_cast<uintptr_t>(p.workspace) % 256 == 0, SOLATTN_EINVAL,
                  "%s: workspace must be 256-byte aligned", what);
  a.part = static_cast<float*>(p.workspace);
  a.part_ml = B * H * c.parts() * D;
  int64_t grid = B * Hkv * c.tiles * c.split;
  if (c.psplit > 0) {
    const int64_t items = p.groups * Hkv * c.ptiles * c.psplit;
    grid += items;
    SOLATTN_REQUIRE(grid < (1ll << 31), SOLATTN_EUNSUPPORTED, "%s: grid too large", what);
    a.shared = static_cast<int>(p.shared), a.per = static_cast<int>(B / p.groups);
    a.psplit = static_cast<int>(c.psplit), a.ptiles = static_cast<int>(c.ptiles), a.pitems = static_cast<int>(items);
    a.by_ptiles = divisor(c.ptiles), a.by_psplit = divisor(c.psplit), a.by_group = divisor(a.group);
  }
  const bool wide = p.cache_type != 0 || p.shared != 0;  // (the others keep their order of sums)
  const int64_t join_grid = a.parts == 1 ? 0 : wide ? B * H : cdiv(B * H, 4);
  static_assert(kJoinThreads == kLaunchThreads && kWaves * 64 == kLaunchThreads, "one bound");
  SOLATTN_REQUIRE(grid < kMostBlocks && join_grid < kMostBlocks, SOLATTN_EUNSUPPORTED, "%s: grid too large", what);
  // More workgroups than are there at once: those of the longest sequences first, so that none
  // of theirs begin when the others end (32 ragged sequences of bf16 keys 69 -> 63 us, eight
  // over e4m3 72 -> 66, four of up to 131072 144 -> 138). Only where a sequence is long enough
  // that the batch holds some 2^26 values of k, and the longer the more sequences there are to
  // search: 128 ragged ones of up to 4096 bf16 keys of 8 heads 223 -> 199, of up to 512 29 -> 32.
  // Nor in a launch of 8192 or more, which one workgroup's keys are too little of (256 of up to
  // 1024 keys of 32 heads 391 -> 394) and which a wide table makes of short sequences (256 of 64
  // keys behind tables of 32768: 41 us, 48 where their lengths are only looked at).
  int64_t from = cdiv(1ll << 27, B * Hkv * D);
  if (from < 4 * B) from = 4 * B;
  const bool ranked = p.table && c.psplit == 0 && B > 1 && B <= kRanked && grid > 1024 && grid < 8192 &&
                      from <= p.max_pages * p.page_size;
  a.ranked = ranked ? static_cast<int>(from) : 0;
  const bool bf = p.dtype == SOLATTN_BF16;
  const auto kern = bf ? kernel_of<Bf16>(D, c.ctiles, p.cache_type) : kernel_of<Fp16>(D, c.ctiles, p.cache_type);
  hipLaunchKernelGGL(kern, dim3(static_cast<uint32_t>(grid)), dim3(kWaves * 64), 0, s, a);
  if (int rc = check_launch(what)) return rc;
  if (a.parts == 1) return SOLATTN_OK;
  if (!wide) {
    hipLaunchKernelGGL(bf ? paged_join_kernel<Bf16> : paged_join_kernel<Fp16>,
                       dim3(static_cast<uint32_t>(join_grid)), dim3(256), 0, s, a);
    return check_launch(what);
  }
  const auto join = bf ? wide_join_of<Bf16>(D, a.parts) : wide_join_of<Fp16>(D, a.parts);
  hipLaunchKernelGGL(join, dim3(static_cast<uint32_t>(join_grid)), dim3(kJoinThreads), 0, s, a);
  return check_launch(what);
}

int64_t paged_attn_workspace(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t keys, int64_t window,
                             int64_t sinks, int64_t shared, int64_t groups, int cache_type) {
  constexpr int64_t top = 1ll << 31;  // (what the call takes: nothing passes 64 bits)
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || keys < 0 || window < 0 || sinks < 0) return 0;
  if (B >= top || H >= top || B * H >= top || D > 128 || keys >= top) return 0;
  if (shared < 0 || shared >= top || (shared && (groups <= 0 || B % groups))) return 0;
  return cut(B, H, Hkv, D, keys, window, sinks, shared, groups, cache_type).part_bytes(B, H, D);
}

}  // namespace solattn

using namespace solattn;

extern "C" int64_t solattn_paged_attn_shared_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D,
                                                             int64_t max_pages, int64_t page_size, int64_t window,
                                                             int64_t sinks, int cache_type, int64_t shared,
                                                             int64_t groups) {
  const bool fit = max_pages >= 0 && page_size >= 0 && max_pages < (1ll << 31) && page_size < (1ll << 31);
  return fit ? paged_attn_workspace(B, H, Hkv, D, max_pages * page_size, window, sinks, shared, groups, cache_type) : 0;
}

extern "C" int64_t solattn_paged_attn_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t max_pages,
                                                      int64_t page_size, int64_t window, int64_t sinks) {
  return solattn_paged_attn_shared_workspace_bytes(B, H, Hkv, D, max_pages, page_size, window, sinks, 0, 0, 1);
}

extern "C" int solattn_paged_attn_shared(const uint16_t* q, int64_t sq_b, int64_t sq_h, const void* k_cache, int64_t sk_p,
                                         int64_t sk_s, int64_t sk_h, const void* v_cache, int64_t sv_p, int64_t sv_s,
                                         int64_t sv_h, int64_t pages, int64_t page_size, int cache_type,
                                         const uint8_t* k_scale, int64_t sks_p, int64_t sks_h, const uint8_t* v_scale,
                                         int64_t svs_p, int64_t svs_h, const int32_t* page_table, int64_t table_stride,
                                         int64_t max_pages, const int32_t* lengths, int64_t B, int64_t H, int64_t Hkv,
                                         int64_t D, int dtype, int64_t window, int64_t sinks, int64_t shared,
                                         int64_t groups, float scale, void* workspace, int64_t workspace_bytes,
                                         uint16_t* o, int64_t so_b, int64_t so_h, solattn_stream_t stream) {
  clear_error();
  const char* what = "paged_attn";
  SOLATTN_REQUIRE(page_table && lengths, SOLATTN_EINVAL, "%s: null page table or lengths", what);
  PagedCall p{};
  p.q = q, p.sq_b = sq_b, p.sq_h = sq_h;
  p.k = k_cache, p.sk_p = sk_p, p.sk_s = sk_s, p.sk_h = sk_h;
  p.v = v_cache, p.sv_p = sv_p, p.sv_s = sv_s, p.sv_h = sv_h;
  p.ks = k_scale, p.ks_p = sks_p, p.ks_h = sks_h, p.vs = v_scale, p.vs_p = svs_p, p.vs_h = svs_h;
  p.cache_type = cache_type, p.pages = pages, p.page_size = page_size;
  p.table = page_table, p.table_stride = table_stride, p.max_pages = max_pages, p.lengths = lengths;
  p.B = B, p.H = H, p.Hkv = Hkv, p.D = D, p.dtype = dtype;
  p.window = window, p.sinks = sinks, p.shared = shared, p.groups = groups, p.scale = scale;
  p.workspace = workspace, p.workspace_bytes = workspace_bytes, p.o = o, p.so_b = so_b, p.so_h = so_h;
  return paged_attn(p, reinterpret_cast<hipStream_t>(stream), what);
}

extern "C" int solattn_paged_attn(const uint16_t* q, int64_t sq_b, int64_t sq_h, const uint16_t* k_cache,
                                  int64_t sk_p, int64_t sk_s, int64_t sk_h, const uint16_t* v_cache, int64_t sv_p,
                                  int64_t sv_s, int64_t sv_h, int64_t pages, int64_t page_size,
                                  const int32_t* page_table, int64_t table_stride, int64_t max_pages,
                                  const int32_t* lengths, int64_t B, int64_t H, int64_t Hkv, int64_t D, int dtype,
                                  int64_t window, int64_t sinks, float scale, void* workspace,
                                  int64_t workspace_bytes, uint16_t* o, int64_t so_b, int64_t so_h,
                                  solattn_stream_t stream) {
  return solattn_paged_attn_shared(q, sq_b, sq_h, k_cache, sk_p, sk_s, sk_h, v_cache, sv_p, sv_s, sv_h, pages, page_size,
                                   0, nullptr, 0, 0, nullptr, 0, 0, page_table, table_stride, max_pages, lengths, B, H,
                                   Hkv, D, dtype, window, sinks, 0, 1, scale, workspace, workspace_bytes, o, so_b, so_h,
                                   stream);
}
