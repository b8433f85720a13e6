// What the sliding-window kernels share: which keys a row sees, the 64-key tiles
// of a block of rows, their copies into LDS and the 16-bit MFMA products.
//
// Row i sits at position p = q_start + i. With a window of W keys and S sinks it
// sees, of the keys j < len, those of
//   causal:    j <= p and (p - j < W or j < S)
//   symmetric: |p - j| < W or j < S
// and none when p >= len. Seen from a row the keys are the interval [jl, jh] and
// those below sk; seen from a key the rows are one interval [pl, ph].
#pragma once

#include "elem.hpp"
#include "fwd_common.hpp"

namespace solattn {

struct Mat {  // a BTHD tensor of 16-bit values, strides in elements
  const uint16_t* p;
  int64_t b, t, h;
};

struct WindowArgs {
  Mat q, k, v, o, d_o;       // (o, d_o: backward's inputs)
  uint16_t* out;             // forward: o; backward: dq
  int64_t out_b, out_t, out_h;
  uint16_t* dk;
  int64_t dk_b, dk_t, dk_h;
  uint16_t* dv;
  int64_t dv_b, dv_t, dv_h;
  float* lse;                // [B][H][Tq], log2 domain; +inf for a row that sees nothing
  uint16_t* o_lo;            // [B][Tq][H][D], what rounding o took away (null: not kept)
  float* delta;              // [B][H][Tq]
  float* lse_p;              // fp16's backward: [B][H][Tq], lse less kPScale
  float2* mag;               // fp16's backward: [B][H][4 nqb], of 32 rows: the largest |do_i| and |D_i|
  const int32_t* lengths;    // null: Tk
  int B, H, Hkv, group, Tq, Tk, q_start;
  int window, sinks, causal; // window <= 2^30
  int nqb, nkb;              // blocks of rows and of keys
  int split;                 // forward: parts of a block's key tiles
  int nsb, ks, kn, slots;    // backward: blocks with sinks; parts of these and of the others; cut blocks' slots a head
  Divisor by_split, by_group, by_nqb, by_hkv, by_items, by_ks, by_kn;  // by_items: parts of a head in the dk, dv launch
  float* part;               // backward: [B Hkv][slots][dk, dv][128][D]; forward: [B H][Tq][split][D]
  float* part_ml;            // forward: [B H][Tq][split][max, sum]
  float c, scale;            // c = scale log2(e)
};

__device__ __forceinline__ int sequence_length(const WindowArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
}

// The keys of one row (see above): j in [jl, jh] or j < sk.
struct RowKeys {
  int jl, jh, sk;
};
__device__ __forceinline__ RowKeys row_keys(const WindowArgs& a, int p, int len) {
  RowKeys r;
  r.jl = p - a.window + 1;
  r.jh = a.causal ? p : p + a.window - 1;
  r.sk = a.causal ? min(a.sinks, p + 1) : a.sinks;
  r.jh = min(r.jh, len - 1);
  r.sk = min(r.sk, len);
  if (p >= len) r.jl = 0, r.jh = -1, r.sk = 0;
  return r;
}

// The rows of one key: p in [pl, ph]; none when pl > ph.
struct KeyRows {
  int pl, ph;
};
__device__ __forceinline__ KeyRows key_rows(const WindowArgs& a, int j, int len) {
  KeyRows r;
  const int end = min(len, a.q_start + a.Tq) - 1;
  r.pl = a.causal ? j : j < a.sinks ? 0 : j - a.window + 1;
  r.ph = j < a.sinks ? end : min(j + a.window - 1, end);
  r.pl = max(r.pl, a.q_start);
  if (j >= len) r.pl = 1, r.ph = 0;
  return r;
}

// Of consecutive rows at p0 to p1: the keys that every one of them sees, j in [all_lo,
// all_hi] or j < all_sk, and bounds of those that any does.
struct RowsKeys {
  int all_lo, all_hi, all_sk, any_lo, any_hi, any_sk;
  __device__ __forceinline__ bool all(int first, int keys) const {
    return (first >= all_lo && first + keys - 1 <= all_hi) || first + keys <= all_sk;
  }
  __device__ __forceinline__ bool none(int first, int keys) const {
    return (first > any_hi || first + keys - 1 < any_lo) && first >= any_sk;
  }
};
__device__ __forceinline__ RowsKeys rows_keys(const WindowArgs& a, int p0, int p1, int len) {
  const RowKeys lo = row_keys(a, p0, len), hi = row_keys(a, min(p1, len - 1), len);
  RowsKeys r;
  r.any_lo = lo.jl, r.any_hi = hi.jh, r.any_sk = hi.sk;
  r.all_lo = hi.jl, r.all_hi = lo.jh, r.all_sk = lo.sk;
  if (p1 >= len) r.all_hi = -1, r.all_sk = 0;  // a row that sees nothing
  if (p0 >= len) r.any_lo = 0, r.any_hi = -1, r.any_sk = 0;
  return r;
}

// Of consecutive keys j0 to j1: the rows that see every one of them, p in [all_lo,
// all_hi], and bounds of those that see any.
struct KeysRows {
  int all_lo, all_hi, any_lo, any_hi;
};
__device__ __forceinline__ KeysRows keys_rows(const WindowArgs& a, int j0, int j1, int len) {
  // intervals move up with the key, but that those of sinks end with the sequence and,
  // symmetric, begin with it
  const KeyRows first = key_rows(a, j0, len), last = key_rows(a, min(j1, len - 1), len);
  const KeyRows past_sinks = key_rows(a, min(max(j0, a.sinks), j1), len);
  KeysRows r;
  r.any_lo = first.pl, r.any_hi = j0 < a.sinks ? first.ph : last.ph;
  r.all_lo = last.pl, r.all_hi = past_sinks.ph;
  if (j1 >= len) r.all_hi = -1;  // a key that no row sees
  if (j0 >= len) r.any_lo = 1, r.any_hi = -1;
  return r;
}

// The 64-key tiles that rows [p0, p1] see: those of the sinks below the window,
// then the window's. Keys of a tile that none of these rows sees are not read:
// safe(j) is a key that is.
struct KeyTiles {
  int lo, hi;     // window keys of the rows, [lo, hi)
  int s_end;      // sink keys below them
  int ns, n, w0;  // sink tiles, tiles, first key of the first window tile
  __device__ __forceinline__ int first(int t) const { return t < ns ? kKeys * t : w0 + kKeys * (t - ns); }
  __device__ __forceinline__ int safe(int j) const { return j < s_end ? j : min(max(j, lo), hi - 1); }
  __device__ __forceinline__ bool whole(int t) const {  // every key of the tile is some row's
    const int j = first(t);
    return j + kKeys <= s_end || (j >= lo && j + kKeys <= hi);
  }
};
__device__ __forceinline__ KeyTiles key_tiles(const WindowArgs& a, int p0, int p1, int len) {
  KeyTiles k;
  if (p0 >= len) {
    k.lo = k.hi = k.s_end = k.ns = k.n = k.w0 = 0;
    return k;
  }
  p0 = __builtin_amdgcn_readfirstlane(p0);  // (kept scalar: copies take scalar bases)
  len = __builtin_amdgcn_readfirstlane(len);
  p1 = min(__builtin_amdgcn_readfirstlane(p1), len - 1);
  k.lo = max(p0 - a.window + 1, 0);
  k.hi = min(a.causal ? p1 + 1 : max(p1 + a.window, a.sinks), len);
  k.s_end = min(a.sinks, k.lo);
  k.w0 = k.lo & ~(kKeys - 1);
  k.ns = min((k.s_end + kKeys - 1) / kKeys, k.w0 / kKeys);
  k.n = k.ns + (k.hi - k.w0 + kKeys - 1) / kKeys;
  return k;
}

// Workgroup id -> item of the launch, so that each of the 8 XCDs (dealt round robin)
// walks contiguous runs of items: neighbours share their keys in its L2. Without
// lengths an XCD has one run; a padded batch, whose sequences may be short or empty,
// is dealt out in runs of 32 items: in one run each, some XCDs have nothing to do (four
// prompts of 16000, 9000, 5000 and 1000 tokens: 1160 against 2540 us; gradients of four of
// 2000, 1500, 900 and 300: 300 against 395), and where every sequence is whole the runs
// cost a little (four of 16000: 2500 against 2470; gradients of two of 8000: 1108 against 1019).
__device__ __forceinline__ uint32_t xcd_item(const WindowArgs& a, uint32_t w, uint32_t total) {
  if (a.lengths) {
    constexpr uint32_t R = 32;
    if (w >= total / (8 * R) * (8 * R)) return w;
    const uint32_t x = w & 7u, i = w >> 3;
    return (i / R * 8 + x) * R + i % R;
  }
  const uint32_t x = w & 7u, q8 = total >> 3, rem = total & 7u;
  return x * q8 + min(x, rem) + (w >> 3);
}

// Item of the dk, dv launch -> (batch, kv head), block of keys and part; slot: its
// place in the workspace, when its block is cut.
struct KeyPart {
  int bh, block, part, parts;
  int64_t slot;
};
__device__ __forceinline__ KeyPart key_part(const WindowArgs& a, uint32_t w) {
  const int sink_items = a.nsb * a.ks;
  KeyPart k;
  uint32_t n = a.by_items.split(w);
  k.bh = static_cast<int>(w);
  const int i = static_cast<int>(n) - (static_cast<int>(a.by_items.d) - sink_items);
  if (i >= 0) {  // sinks' parts last: the shorter ones, unless there are very many sinks
    k.slot = static_cast<int64_t>(k.bh) * a.slots + i;
    n = i;
    k.part = a.by_ks.split(n), k.block = n, k.parts = a.ks;
  } else {
    k.slot = static_cast<int64_t>(k.bh) * a.slots + sink_items + n;
    k.part = a.by_kn.split(n), k.block = a.nsb + n, k.parts = a.kn;
  }
  return k;
}

// ------------------------------------------------------------------- LDS tiles
// Tiles that are read both by rows (16-byte pieces of 16 rows) and transposed
// (ds_read_b64_tr_b16: 4 rows x 4 consecutive pieces) need one swizzle that keeps
// both free of conflicts: the row's low bits pick a quarter of the row for the
// transposed read, the next ones a place within it.
template <int D>
__device__ __forceinline__ int swz_both(int row, int chunk) {
  const int r = D == 128 ? row : row >> 1;
  return D == 128 ? chunk ^ (((r & 3) << 2) | ((r >> 2) & 3)) : chunk ^ (((r & 1) << 2) | ((r >> 1) & 3));
}

// How a tile is read: by rows (K of the forward), transposed (its V) or both.
enum { kByRow, kTransposed, kBoth };
template <int D, int HOW>
__device__ __forceinline__ int swz(int row, int chunk) {
  return HOW == kByRow ? swz_k<D>(row, chunk) : HOW == kTransposed ? swz_v<D>(row, chunk) : swz_both<D>(row, chunk);
}

// 64 rows of D values into the LDS tile at dst, row i from base + row_of(i) stride.
template <int NTHREADS, int D, int HOW, typename RowOf>
__device__ __forceinline__ void copy_tile(uint32_t dst, const uint16_t* base, int64_t stride, RowOf&& row_of) {
  constexpr int C = D / 8, U = kKeys * C / NTHREADS;
  const uint32_t l0 = dst + wave_id() * 64 * 16;
  uint32_t tid = threadIdx.x;  // (hidden: the addresses are made at each copy, not held through a loop)
  asm volatile("" : "+v"(tid));
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int e = tid + NTHREADS * u, row = e / C, pc = e % C;
    g2l16(base + static_cast<int64_t>(row_of(row)) * stride + swz<D, HOW>(row, pc) * 8, l0 + NTHREADS * u * 16);
  }
}

// Whole tiles of consecutive rows need one lane offset: a copy of all threads is
// NTHREADS / (D / 8) rows, after which a lane's swizzle repeats.
template <int NTHREADS, int D, int HOW>
__device__ __forceinline__ uint32_t copy_offset(int64_t stride) {
  constexpr int C = D / 8;
  static_assert(NTHREADS / C % 16 == 0, "a lane keeps its piece");
  const int row = threadIdx.x / C, pc = threadIdx.x % C;
  return static_cast<uint32_t>((row * stride + swz<D, HOW>(row, pc) * 8) * 2);
}
template <int NTHREADS, int D>
__device__ __forceinline__ void copy_whole(uint32_t dst, const uint16_t* first, int64_t stride, uint32_t off) {
  constexpr int R = NTHREADS / (D / 8), U = kKeys / R;
  const uint32_t l0 = dst + wave_id() * 64 * 16;
#pragma unroll
  for (int u = 0; u < U; ++u) g2l16_s(first + u * R * stride, off, l0 + NTHREADS * u * 16);
}

// Half a tile (rows [32 hh, 32 hh + 32) of it) for the forward's pipeline: row i from
// base + row_of(32 hh + i) stride, or consecutive rows from `first` on (issue_half).
template <int NTHREADS, int D, int HOW, typename RowOf>
__device__ __forceinline__ void copy_half(uint32_t dst, int hh, const uint16_t* base, int64_t stride, RowOf&& row_of) {
  constexpr int C = D / 8, U = kKeys / 2 * C / NTHREADS;
  const uint32_t l0 = dst + wave_id() * 64 * 16;
  uint32_t tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int e = tid + NTHREADS * u, row = 32 * hh + e / C, pc = e % C;
    g2l16(base + static_cast<int64_t>(row_of(row)) * stride + swz<D, HOW>(row, pc) * 8, l0 + NTHREADS * u * 16);
  }
}

// Operands of an LDS tile (256-byte aligned): the row operand (m, cc) is rows
// 32 m + lane % 32, channels 16 cc + 8 (lane / 32) ..; the transposed operand
// (ks, dt) is channel 32 dt + lane % 32 of rows 16 ks + 8 (e / 4) + 4 (lane / 32)
// + e % 4. A lane keeps one address for the first and two for the second.
template <int D, int HOW>
struct TileAddr {
  uint32_t row, tr0, tr1;
  __device__ __forceinline__ TileAddr(uint32_t tile, int lane) {
    const int col = lane & 31, half = lane >> 5;
    row = tile + col * (2 * D) + 16 * swz<D, HOW>(col, half);
    const int g = lane >> 4, sl = lane & 15, r0 = 4 * (g >> 1) + (sl >> 2), cp = 2 * (g & 1) + ((sl & 3) >> 1);
    tr0 = tile + r0 * (2 * D) + 16 * swz<D, HOW>(r0, cp) + 8 * (sl & 1);
    tr1 = tile + (r0 + 8) * (2 * D) + 16 * swz<D, HOW>(r0 + 8, cp) + 8 * (sl & 1);
  }
  // Hides the addresses from the optimiser: what is derived from them afterwards is
  // derived there, not hoisted out of the loop into registers of its own.
  __device__ __forceinline__ void remade() { asm volatile("" : "+v"(row), "+v"(tr0), "+v"(tr1)); }
  __device__ __forceinline__ bf16x8 by_row(int m, int cc, uint32_t at = 0) const {  // at: bytes to another buffer
    const uint32_t x = (row ^ static_cast<uint32_t>(cc << 5)) + m * (64 * D) + at;
    return *reinterpret_cast<const __attribute__((address_space(3))) bf16x8*>(static_cast<uintptr_t>(x));
  }
  __device__ __forceinline__ bf16x8 transposed(int ks, int dt, uint32_t at = 0) const {
    typedef short v4i16 __attribute__((ext_vector_type(4)));
    const uint32_t x0 = (tr0 ^ static_cast<uint32_t>(dt << 6)) + ks * (32 * D) + at;
    const uint32_t x1 = (tr1 ^ static_cast<uint32_t>(dt << 6)) + ks * (32 * D) + at;
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        reinterpret_cast<__attribute__((address_space(3))) v4i16*>(static_cast<uintptr_t>(x0)));
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        reinterpret_cast<__attribute__((address_space(3))) v4i16*>(static_cast<uintptr_t>(x1)));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// This lane's row of a B operand straight from memory: channels 16 cc + 8 (lane / 32) ...
template <int D>
__device__ __forceinline__ void load_row(bf16x8 (&x)[D / 16], const uint16_t* row, int half) {
#pragma unroll
  for (int cc = 0; cc < D / 16; ++cc)
    x[cc] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(row + 16 * cc + 8 * half));
}

// Rows of 32 columns of an accumulator pair-packed into a B operand: elements 8 ks .. 8 ks + 7.
template <typename E>
__device__ __forceinline__ bf16x8 pack8(const f32x16& s, int ks) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = E::pack(s[8 * ks + 2 * i], s[8 * ks + 2 * i + 1]);
  return __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
}

// Elements of an accumulator as B operands: in one rounding, or in two that add up to
// the value but for some 2^-17 of it (bf16; fp16: 2^-22).
template <typename E, int NW>
__device__ __forceinline__ void pack_all(bf16x8 (&w)[NW][2], const f32x16& s) {
  if constexpr (NW == 1) {
    w[0][0] = pack8<E>(s, 0);
    w[0][1] = pack8<E>(s, 1);
  } else {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      uint32_t u[4], v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = s[8 * ks + 2 * i], y = s[8 * ks + 2 * i + 1];
        u[i] = E::pack(x, y);
        v[i] = E::pack(x - E::lo(u[i]), y - E::hi(u[i]));
      }
      w[0][ks] = __builtin_bit_cast(bf16x8, make_uint4(u[0], u[1], u[2], u[3]));
      w[1][ks] = __builtin_bit_cast(bf16x8, make_uint4(v[0], v[1], v[2], v[3]));
    }
  }
}

// acc^T (channel 32 dt + 8 (r / 4) + 4 half + r % 4 of row `lane % 32`) times f into a row of D values.
template <typename E, int ND>
__device__ __forceinline__ void store_row(const f32x16 (&acc)[ND], float f, uint16_t* row, bool on, int half) {
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int ip = 0; ip < 2; ++ip) {
      uint32_t w[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i = 4 * (2 * ip + u);
        w[u][0] = E::pack(acc[dt][i] * f, acc[dt][i + 1] * f);
        w[u][1] = E::pack(acc[dt][i + 2] * f, acc[dt][i + 3] * f);
      }
      uint32_t y[2];  // the two lanes of a row swap halves, so each writes 16 contiguous bytes
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t x = half ? w[0][e] : w[1][e];
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        y[e] = half ? r[0] : r[1];
      }
      const uint4 v = half ? make_uint4(y[0], y[1], w[1][0], w[1][1]) : make_uint4(w[0][0], w[0][1], y[0], y[1]);
      if (on) *reinterpret_cast<uint4*>(row + 32 * dt + 16 * ip + 8 * half) = v;
    }
}

// acc f becomes what is left of it when it is rounded to the type.
template <typename E, int ND>
__device__ __forceinline__ void rounded_off(f32x16 (&acc)[ND], float f) {
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const float x = acc[dt][r] * f, y = acc[dt][r + 1] * f;
      const uint32_t w = E::pack(x, y);
      acc[dt][r] = x - E::lo(w);
      acc[dt][r + 1] = y - E::hi(w);
    }
}

// Which of the 32 x 32 tile's elements of this lane count, as bits k (element r is k =
// 8 (r / 4) + r % 4, so below 28): those of an interval are two shifts, and an element's
// bit drawn out to a word keeps or clears it without a compare.
__device__ __forceinline__ uint32_t bits_from(int k) { return ~0u << min(max(k, 0), 28); }
__device__ __forceinline__ uint32_t bit_word(uint32_t bits, int r) {
  uint32_t w;  // (hidden from the optimiser, which would go back to compares)
  asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(w) : "v"(bits), "i"(8 * (r >> 2) + (r & 3)));
  return w;
}
__device__ __forceinline__ float keep(float x, uint32_t word) { return __uint_as_float(__float_as_uint(x) & word); }

// Bits of the keys first + 4 half + k that the row sees.
__device__ __forceinline__ uint32_t key_bits(const RowKeys& rk, int first, int half) {
  const int base = first + 4 * half;
  return (bits_from(rk.jl - base) & ~bits_from(rk.jh + 1 - base)) | ~bits_from(rk.sk - base);
}
// Bits of the rows first + 4 half + k that see the key.
__device__ __forceinline__ uint32_t row_bits(const KeyRows& kr, int first, int half) {
  const int base = first + 4 * half;
  return bits_from(kr.pl - base) & ~bits_from(kr.ph + 1 - base);
}

// Scores of 32 keys (first + the key of element r) for this lane's row: those it does not see become -inf.
__device__ __forceinline__ void mask_keys(f32x16& s, const RowKeys& rk, int first, int half) {
  const uint32_t bits = key_bits(rk, first, half);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const uint32_t w = bit_word(bits, r);
    s[r] = __uint_as_float((__float_as_uint(s[r]) & w) | (__float_as_uint(-INFINITY) & ~w));
  }
}

}  // namespace solattn
