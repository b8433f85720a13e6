// Attention of many rows over the pages of one sequence: 128 query rows a workgroup, a
// wave for 32 of them, keys and values in LDS, the pipeline over halves of 32 keys that the
// windowed forward has (window_common.hpp). A row is a head of one of the sequences that
// share the keys.
//
// Bound: the matrix instructions, 4 D operations a row and key, beside the exponentials of
// the scores. 256 sequences of 24 heads over 8, of 128 channels, behind 32760 keys alone:
// 16-bit values 143 us, 0.72 PFLOP/s (0.95 between the first tile's latency and the parts'
// way out: behind 131071 keys 467 us, matrix instructions in 39% of the cycles, vector ones
// in 43%, either in 63%); e4m3 some 10% more, whose conversions stand between the products.
//
// What differs from the windowed forward is where keys come from: a lane finds the place of
// one key of a tile of 64 well ahead of its copy, and the copies of a half (rows of eight
// consecutive keys a wave at most, so of one page) take their scalar bases from these lanes.
// (Bases found by each copy in scalar arithmetic: some 40 scalar instructions a copy, 160 a
// step of 16 matrix instructions.) Keys past the end or on pages that are none of the
// cache's are rows of zeros, and masked. 16-bit values are copied straight into LDS
// (attend_ring); codes go through registers and become 16-bit values there, once for all
// the rows that read the tile (attend_codes). P is rounded once to the queries' type, as in
// the windowed forward: a second part would double the products with V, half of what bounds
// a tile.
#pragma once

#include "cache8.hpp"
#include "window_common.hpp"

namespace solattn {

constexpr int kTileRows = 128, kTileThreads = 2 * kTileRows;

static __device__ uint4 zero_row[16];  // (never written)

// The cache as the tiles read it; strides in bytes.
struct TileSource {
  const uint8_t* p;  // this kv head
  int64_t page, slot;
  const uint8_t* e;  // codes: exponents
  int64_t e_page;
  bool near;         // strides are within 32 bits, and a few slots
};

// Where a tile's keys are, a lane each: rows' addresses and, of codes, their powers of two.
struct TileRows {
  uint32_t lo, hi;
  float power;
  __device__ __forceinline__ const uint8_t* of_lane(int lane) const {  // (another for every lane)
    const uint64_t x = static_cast<uint32_t>(__shfl(lo, lane)) | static_cast<uint64_t>(static_cast<uint32_t>(__shfl(hi, lane))) << 32;
    return reinterpret_cast<const uint8_t*>(x);
  }
  __device__ __forceinline__ const uint8_t* of_group(int lane) const {  // (the same for all)
    const uint64_t x = static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, lane)) |
                       static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(hi, lane))) << 32;
    return reinterpret_cast<const uint8_t*>(x);
  }
};

// Page ids that are kept in LDS: of 64 tiles, twice.
constexpr int kIdTiles = 64, kIds = kIdTiles * kKeys / 8 + 1;  // (pages have 8 slots at least)

struct TilePages {
  const int32_t* table;  // the sequence's row
  Divisor by_page;
  int pages, end;        // keys [0, end) are visible
  // The page of this lane's key of the 64 from j0 on; -1: not visible.
  __device__ __forceinline__ int ids(int j0) const {
    const int j = j0 + (static_cast<int>(threadIdx.x) & 63);
    const int id = table[by_page.of(static_cast<uint32_t>(min(j, end - 1)))];
    return j < end && id >= 0 && id < pages ? id : -1;
  }
  // The ids of segment s (64 tiles) of the keys from `first` on, into LDS.
  __device__ __forceinline__ int page0(int first, int s) const {
    return static_cast<int>(by_page.of(static_cast<uint32_t>(first + s * kIdTiles * kKeys)));
  }
  __device__ __forceinline__ void fetch_ids(int32_t (&to)[2][kIds + 3], int first, int s) const {
    const int p0 = page0(first, s), n = static_cast<int>(by_page.of(static_cast<uint32_t>(end - 1))) - p0 + 1;
    for (int i = threadIdx.x; i < min(n, kIds); i += kTileThreads) {
      const int id = table[p0 + i];
      to[s & 1][i] = id >= 0 && id < pages ? id : -1;
    }
  }
};

// A key's row, of page `id` (-1: a row of zeros).
__device__ __forceinline__ TileRows row_at(const TileSource& s, int id, uint32_t slot) {
  uint64_t at = reinterpret_cast<uint64_t>(s.p);
  if (s.near)
    at += static_cast<uint64_t>(static_cast<uint32_t>(id)) * static_cast<uint32_t>(s.page) +
          static_cast<uint64_t>(slot) * static_cast<uint32_t>(s.slot);
  else
    at += id * s.page + slot * s.slot;
  at = id >= 0 ? at : reinterpret_cast<uint64_t>(zero_row);
  return {static_cast<uint32_t>(at), static_cast<uint32_t>(at >> 32), 0.f};
}

// Scores of a half from key j0 on: keys that are not visible (`seen` has a bit for each) or
// not below `hi` become -inf; every row sees the keys below `safe`.
__device__ __forceinline__ void mask_half(f32x16& s, int j0, uint32_t seen, int hi, int safe) {
  if (seen == ~0u && j0 + 32 <= safe) return;
  const int half = (threadIdx.x & 63) >> 5;
  const uint32_t bits = (seen >> (4 * half)) & ~bits_from(hi - j0 - 4 * half);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const uint32_t w = bit_word(bits, r);
    s[r] = __uint_as_float((__float_as_uint(s[r]) & w) | (__float_as_uint(-INFINITY) & ~w));
  }
}

// Copies half `hf` of a tile of 16-bit values into the half buffer at dst.
template <int D, int HOW>
struct HalfCopy {
  static constexpr int C = D / 8, R = 64 / C, U = 32 / (kTileThreads / C);  // pieces of a row; rows of a wave's copy; copies
  uint32_t off;
  __device__ __forceinline__ void init(const TileSource& s) {
    off = static_cast<uint32_t>((threadIdx.x & 63) / C * s.slot) + piece();
  }
  __device__ __forceinline__ uint32_t piece() const {
    const int lane = threadIdx.x & 63;
    return swz<D, HOW>(R * wave_id() + lane / C, lane % C) * 16;
  }
  __device__ __forceinline__ void start(uint32_t dst, int hf, uint64_t seen, const TileRows& rows, const TileSource& s) {
    const bool plain = static_cast<uint32_t>(seen >> (32 * hf)) == ~0u && s.near;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int g0 = u * (kTileThreads / C) + R * wave_id();
      if (plain)
        g2l16_s(rows.of_group(32 * hf + g0), off, dst + g0 * 2 * D);
      else
        g2l16(rows.of_lane(32 * hf + g0 + (threadIdx.x & 63) / C) + piece(), dst + g0 * 2 * D);
    }
  }
};

// The same of codes, 16 of a row a thread: start() asks for them, finish() has their values
// in LDS.
template <typename E, typename CODES, int D, int HOW>
struct HalfDecode {
  static constexpr int C = D / 16;
  uint4 w;
  float power;
  uint32_t to0, to1;  // where the piece's two halves go
  bool mine;
  __device__ __forceinline__ void init() {
    const int e = threadIdx.x, row = e / C % 32, pc = e % C;
    mine = D == 128 || (e < 32 * C) == (HOW == kByRow);  // 64 channels: half the threads for K, half for V
    to0 = row * 2 * D + swz<D, HOW>(row, 2 * pc) * 16;
    to1 = row * 2 * D + swz<D, HOW>(row, 2 * pc + 1) * 16;
  }
  __device__ __forceinline__ void start(int hf, const TileRows& rows) {
    const int e = threadIdx.x, row = 32 * hf + e / C % 32;
    power = __shfl(rows.power, row);
    const uint8_t* at = rows.of_lane(row);
    if (mine) w = *reinterpret_cast<const uint4*>(at + e % C * 16);
  }
  __device__ __forceinline__ void finish(uint32_t dst) const {
    if (!mine) return;
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    uint32_t y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = CODES::template scaled<E>(x[i], 0, power);
      y[2 * i + 1] = CODES::template scaled<E>(x[i], 2, power);
    }
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) u32x4* lds4;
    *reinterpret_cast<lds4>(static_cast<uintptr_t>(dst + to0)) = u32x4{y[0], y[1], y[2], y[3]};
    *reinterpret_cast<lds4>(static_cast<uintptr_t>(dst + to1)) = u32x4{y[4], y[5], y[6], y[7]};
  }
};

// The keys of tiles tile0 .. tile0 + ntiles - 1 (64 each, the last may end early) for this
// lane's row (32 wave + lane % 32 of the workgroup's), which sees those below `hi`; every
// row of the workgroup sees those below `safe`. st: the row's O^T, maximum and sum.
template <typename E, typename CODES, int D>
__device__ __forceinline__ void attend_codes(RowState<D / 32>& st, const bf16x8 (&q)[D / 16], uint32_t kb, uint32_t vb,
                                             const TileSource& ks, const TileSource& vs, const TilePages& pg,
                                             int tile0, int ntiles, int hi, int safe, float c) {
  constexpr int ND = D / 32, NC = D / 16;
  constexpr uint32_t kHalf = kKeys * D;  // bytes of half a tile
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const uint32_t kl = k_lane<D>(kb, lane & 31, half), vl = v_lane<D>(vb, lane);
  const int first = tile0 * kKeys;
  HalfDecode<E, CODES, D, kByRow> kc;
  HalfDecode<E, CODES, D, kTransposed> vc;
  kc.init();
  vc.init();
  st.m = kNoMax;
  st.l = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) st.acc[dt] = f32x16{};
  const auto key0 = [&](int t) __attribute__((always_inline)) { return first + kKeys * min(t, ntiles - 1); };
  const auto ids_of = [&](int t) __attribute__((always_inline)) { return pg.ids(key0(t)); };
  const auto rows = [&](int id, int t, const TileSource& s) __attribute__((always_inline)) {
    const uint32_t j = static_cast<uint32_t>(key0(t) + lane), slot = j - pg.by_page.of(j) * pg.by_page.d;
    TileRows r = row_at(s, id, slot);
    if (id >= 0) r.power = power_of(s.e[id * s.e_page + slot]);
    return r;
  };
  const auto mask = [&](f32x16& s, int t, int hf, uint64_t seen) __attribute__((always_inline)) {
    mask_half(s, first + kKeys * t + 32 * hf, static_cast<uint32_t>(seen >> (32 * hf)), hi, safe);
  };
  // In round t: K's rows of the tiles t + 1 and t + 2, V's of t and t + 1; those of a tile
  // further on are found here, the ids of t + 4 asked for.
  int i2, i3, i4;
  uint64_t s0w, s1w, s2w, s3w;  // which keys of the tiles t, t + 1, t + 2, t + 3 are visible
  TileRows k1, k2, v0, v1;
  {
    const int i0 = ids_of(0), i1 = ids_of(1);
    i2 = ids_of(2), i3 = ids_of(3);
    const TileRows k0 = rows(i0, 0, ks);
    v0 = rows(i0, 0, vs);
    s0w = __ballot(i0 >= 0), s1w = __ballot(i1 >= 0), s2w = __ballot(i2 >= 0), s3w = __ballot(i3 >= 0);
    kc.start(0, k0);
    kc.finish(kb);
    kc.start(1, k0);
    kc.finish(kb + kHalf);
    vc.start(0, v0);
    vc.finish(vb);
    k1 = rows(i1, 1, ks), v1 = rows(i1, 1, vs), k2 = rows(i2, 2, ks);
  }
  f32x16 sa, sb;  // scores of even and odd halves
  bf16x8 pa[2], pb[2];
  __syncthreads();
  {  // step 0, without a stream: both halves are scored, the running max is the whole tile's
    f32x16 x0 = {}, x1 = {};
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) x0 = E::mfma32(k_op_x<D>(kl, 0, cc), q[cc], x0);
    __syncthreads();  // every wave is done with K(0)
    if (ntiles > 1) kc.start(0, k1);
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) x1 = E::mfma32(k_op_x<D>(kl + kHalf, 0, cc), q[cc], x1);
    mask(x0, 0, 0, s0w);
    mask(x1, 0, 1, s0w);
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fmaxf(x0[r], x1[r]));
    st.m = fmaxf(kNoMax, xhalf_max(mx) * c);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = E::exp_pair(x0[2 * i], x0[2 * i + 1], c, -st.m, st.l);
    pa[0] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
    pa[1] = __builtin_bit_cast(bf16x8, make_uint4(w[4], w[5], w[6], w[7]));
    sb = x1;
    if (ntiles > 1) kc.finish(kb);
  }
  mfma_fence(st.acc);  // O's zeros are in their registers before the asm MFMAs that add to them
  __syncthreads();
  int t = 0;
#pragma unroll 1
  for (; t < ntiles - 1; ++t) {
    i4 = ids_of(t + 4);
    const TileRows k3 = rows(i3, t + 3, ks), v2 = rows(i2, t + 2, vs);
    // step 2 t + 1: K of half 2 t + 3, V of 2 t + 1
    kc.start(1, k1);
    vc.start(1, v0);
    window_step<E, D>(st, sb, sa, pa, pb, kl, vl, q, c);
    kc.finish(kb + kHalf);
    vc.finish(vb + kHalf);
    __syncthreads();
    // step 2 t + 2: K of half 2 t + 4, V of 2 t + 2
    if (t + 2 < ntiles) kc.start(0, k2);
    vc.start(0, v1);
    mask(sa, t + 1, 0, s1w);
    window_step<E, D>(st, sa, sb, pb, pa, kl + kHalf, vl + kHalf, q, c);
    mask(sb, t + 1, 1, s1w);
    if (t + 2 < ntiles) kc.finish(kb);
    vc.finish(vb);
    __syncthreads();
    i2 = i3, i3 = i4;
    k1 = k2, k2 = k3, v0 = v1, v1 = v2;
    s0w = s1w, s1w = s2w, s2w = s3w, s3w = __ballot(i4 >= 0);
  }
  vc.start(1, v0);
  window_step<E, D>(st, sb, sa, pa, pb, kl, vl, q, c);
  vc.finish(vb + kHalf);
  __syncthreads();
  mfma_fence(st.acc);
#pragma unroll
  for (int i = 0; i < NC; ++i)  // P.V of the last half
    st.acc[i % ND] = E::mfma32(v_op_x<D>(vl + kHalf, i / ND, i % ND), pb[i / ND], st.acc[i % ND]);
}

// The same with 16-bit values, copied four halves ahead into rings of four: a copy has two
// steps to land, and the wait at a step's end leaves the newest two steps' copies in flight.
// Page ids are kept in LDS, so that no load of the loop but the copies counts.
template <int D>
struct TileLds {
  uint16_t k[4][32 * D], v[4][32 * D];
  int32_t ids[2][kIds + 3];
};

// Leaves N copies in flight.
template <int N>
__device__ __forceinline__ void wait_copies() {
  __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (N >> 4) << 14);
}
// Behind it no wave reads LDS any more: the compiler does not wait for its reads here by itself.
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <typename E, int D>
__device__ __forceinline__ void attend_ring(RowState<D / 32>& st, const bf16x8 (&q)[D / 16], TileLds<D>& lds,
                                            const TileSource& ks, const TileSource& vs, const TilePages& pg, int tile0,
                                            int ntiles, int hi, int safe, float c) {
  constexpr int ND = D / 32, NC = D / 16;
  constexpr uint32_t kHalf = kKeys * D;  // bytes of half a tile
  using KCopy = HalfCopy<D, kByRow>;
  using VCopy = HalfCopy<D, kTransposed>;
  constexpr int STEP = KCopy::U + VCopy::U;  // copies of a step
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const uint32_t kb = lds_addr(lds.k), vb = lds_addr(lds.v);
  const uint32_t kl = k_lane<D>(kb, lane & 31, half), vl = v_lane<D>(vb, lane);
  const int first = tile0 * kKeys;
  KCopy kc;
  VCopy vc;
  kc.init(ks);
  vc.init(vs);
  st.m = kNoMax;
  st.l = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) st.acc[dt] = f32x16{};
  // Where this lane's key of tile t is (t may pass the last tile: nothing is read there). The
  // ids come from LDS, so a tile's are asked for a round before its rows' places are needed.
  struct Key {
    int id;
    uint32_t slot;
  };
  const auto key_of = [&](int t) __attribute__((always_inline)) {
    const uint32_t j = min(static_cast<uint32_t>(first + lane) + kKeys * t, static_cast<uint32_t>(pg.end));
    const uint32_t page = pg.by_page.of(j);
    const int sg = t / kIdTiles;
    const uint32_t i = page - pg.page0(first, sg);
    return Key{lds.ids[sg & 1][min(i, static_cast<uint32_t>(kIds - 1))], j - page * pg.by_page.d};
  };
  const auto seen_of = [&](Key& k, int t) __attribute__((always_inline)) {
    k.id = static_cast<uint32_t>(first + lane) + kKeys * t < static_cast<uint32_t>(pg.end) ? k.id : -1;
    return __ballot(k.id >= 0);
  };
  const auto mask = [&](f32x16& s, int t, int hf, uint64_t seen) __attribute__((always_inline)) {
    mask_half(s, first + kKeys * t + 32 * hf, static_cast<uint32_t>(seen >> (32 * hf)), hi, safe);
  };
  wait_copies<0>();
  tile_barrier();
  // Round t copies the second half of tile t + 2 and the first of t + 3 for K, of t + 1 and
  // t + 2 for V.
  uint64_t s0w, s1w, s2w, s3w;  // visible keys of the tiles t, t + 1, t + 2, t + 3
  TileRows k2, k3, v1, v2;
  Key key2, key3;
  {
    Key key0 = key_of(0), key1 = key_of(1);
    key2 = key_of(2), key3 = key_of(3);
    s0w = seen_of(key0, 0), s1w = seen_of(key1, 1), s2w = seen_of(key2, 2);
    const TileRows k0 = row_at(ks, key0.id, key0.slot), k1 = row_at(ks, key1.id, key1.slot), v0 = row_at(vs, key0.id, key0.slot);
    kc.start(kb, 0, s0w, k0, ks);
    kc.start(kb + kHalf, 1, s0w, k0, ks);
    if (ntiles > 1) kc.start(kb + 2 * kHalf, 0, s1w, k1, ks);
    vc.start(vb, 0, s0w, v0, vs);
    if (ntiles > 1) kc.start(kb + 3 * kHalf, 1, s1w, k1, ks);
    vc.start(vb + kHalf, 1, s0w, v0, vs);
    k2 = row_at(ks, key2.id, key2.slot), v1 = row_at(vs, key1.id, key1.slot);
  }
  // All but the newest two steps' copies are there; near the end, where steps ask for
  // fewer, all are.
  const auto land = [&](int t) __attribute__((always_inline)) {
    if (t + 3 < ntiles)
      wait_copies<2 * STEP>();
    else
      wait_copies<0>();
    tile_barrier();
  };
  f32x16 sa, sb;  // scores of even and odd halves
  bf16x8 pa[2], pb[2];
  land(-1);
  {  // step 0, without a stream: both halves are scored, the running max is the whole tile's
    f32x16 x0 = {}, x1 = {};
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) x0 = E::mfma32(k_op_x<D>(kl, 0, cc), q[cc], x0);
    tile_barrier();  // every wave is done with K(0)
    if (ntiles > 2) kc.start(kb, 0, s2w, k2, ks);
    if (ntiles > 1) vc.start(vb + 2 * kHalf, 0, s1w, v1, vs);
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) x1 = E::mfma32(k_op_x<D>(kl + kHalf, 0, cc), q[cc], x1);
    mask(x0, 0, 0, s0w);
    mask(x1, 0, 1, s0w);
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fmaxf(x0[r], x1[r]));
    st.m = fmaxf(kNoMax, xhalf_max(mx) * c);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = E::exp_pair(x0[2 * i], x0[2 * i + 1], c, -st.m, st.l);
    pa[0] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
    pa[1] = __builtin_bit_cast(bf16x8, make_uint4(w[4], w[5], w[6], w[7]));
    sb = x1;
  }
  mfma_fence(st.acc);  // O's zeros are in their registers before the asm MFMAs that add to them
  land(-1);
  int t = 0;
#pragma unroll 1
  for (; t < ntiles - 1; ++t) {
    if (t % kIdTiles == kIdTiles / 2 && (t / kIdTiles + 1) * kIdTiles < ntiles) pg.fetch_ids(lds.ids, first, t / kIdTiles + 1);
    const uint32_t a0 = (t & 1) * 2 * kHalf, b0 = 2 * kHalf - a0;  // halves 2 t and 2 t + 2 of the rings
    const Key key4 = key_of(t + 4);
    s3w = seen_of(key3, t + 3);
    k3 = row_at(ks, key3.id, key3.slot), v2 = row_at(vs, key2.id, key2.slot);
    if (t + 2 < ntiles) kc.start(kb + a0 + kHalf, 1, s2w, k2, ks);  // step 2 t + 1
    vc.start(vb + b0 + kHalf, 1, s1w, v1, vs);
    window_step<E, D>(st, sb, sa, pa, pb, kl + b0, vl + a0, q, c);
    land(t);
    if (t + 3 < ntiles) kc.start(kb + b0, 0, s3w, k3, ks);  // step 2 t + 2
    if (t + 2 < ntiles) vc.start(vb + a0, 0, s2w, v2, vs);
    mask(sa, t + 1, 0, s1w);
    window_step<E, D>(st, sa, sb, pb, pa, kl + b0 + kHalf, vl + a0 + kHalf, q, c);
    mask(sb, t + 1, 1, s1w);
    land(t);
    k2 = k3, v1 = v2, key2 = key3, key3 = key4;
    s1w = s2w, s2w = s3w;
  }
  const uint32_t a0 = (t & 1) * 2 * kHalf;
  window_step<E, D>(st, sb, sa, pa, pb, kl + 2 * kHalf - a0, vl + a0, q, c);
  mfma_fence(st.acc);
#pragma unroll
  for (int i = 0; i < NC; ++i)  // P.V of the last half
    st.acc[i % ND] = E::mfma32(v_op_x<D>(vl + a0 + kHalf, i / ND, i % ND), pb[i / ND], st.acc[i % ND]);
}

}  // namespace solattn
