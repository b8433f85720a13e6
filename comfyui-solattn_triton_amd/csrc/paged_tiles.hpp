// Attention of many rows over the pages of one sequence: 128 query rows a workgroup, a
// wave for 32 of them, keys and values in LDS, the pipeline over halves of 32 keys that the
// windowed forward has (window_common.hpp). A row is a head of one of the sequences that
// share the keys.
//
// What differs is where a half comes from: a wave copies rows of eight consecutive keys at
// most, so of one page, whose id a lane has read two halves ahead; the copy's base is
// scalar. Keys past the end or on pages that are none of the cache's come from a row of
// zeros and are masked. Codes go through registers and become 16-bit values there, once
// for all the rows that read the tile.
#pragma once

#include "cache8.hpp"
#include "window_common.hpp"

namespace solattn {

constexpr int kTileRows = 128, kTileThreads = 2 * kTileRows;

static __device__ uint4 zero_row[16];  // (never written)

// The cache as the tiles read it; strides in bytes, slots' below 2^28.
struct TileSource {
  const uint8_t* p;  // this kv head
  int64_t page, slot;
  const uint8_t* e;  // codes: exponents
  int64_t e_page;
};

// The pages' ids of the 32 keys of a half, a lane each (twice); -1: not visible.
struct TilePages {
  const int32_t* table;  // the sequence's row
  Divisor by_page;
  int pages, end;        // keys [0, end) are visible
  __device__ __forceinline__ int ids(int j0) const {
    const int j = j0 + (static_cast<int>(threadIdx.x) & 31);
    const int id = table[by_page.of(static_cast<uint32_t>(min(j, end - 1)))];
    return j < end && id >= 0 && id < pages ? id : -1;
  }
  __device__ __forceinline__ int slot(int j) const {
    const uint32_t n = static_cast<uint32_t>(j);
    return static_cast<int>(n - by_page.of(n) * by_page.d);
  }
};

// Copies of one half (keys j0 .. j0 + 31) into the half buffer at dst.
template <int D, int HOW>
struct HalfCopy {  // 16-bit values, straight into LDS
  static constexpr int C = D / 8, R = 64 / C, U = 32 / (kTileThreads / C);  // pieces of a row; rows of a wave's copy; copies
  uint32_t off;
  __device__ __forceinline__ void init(const TileSource& s) {
    const int lane = threadIdx.x & 63, row = R * wave_id() + lane / C;
    off = static_cast<uint32_t>(lane / C * s.slot + swz<D, HOW>(row, lane % C) * 16);
  }
  __device__ __forceinline__ void start(uint32_t dst, int j0, int ids, const TileSource& s, const TilePages& pg) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int g0 = u * (kTileThreads / C) + R * wave_id(), j = j0 + g0;
      const uint32_t to = dst + g0 * 2 * D;
      const int id = __builtin_amdgcn_readlane(ids, g0);
      const uint8_t* base = s.p + max(id, 0) * s.page + pg.slot(j) * s.slot;
      if (id >= 0 && j + R <= pg.end) {
        g2l16_s(base, off, to);
      } else {
        const bool on = id >= 0 && j + lane / C < pg.end;
        g2l16(on ? base + off : reinterpret_cast<const uint8_t*>(zero_row) + lane % C * 16, to);
      }
    }
  }
  __device__ __forceinline__ void finish(uint32_t) const {}
};
template <typename E, typename CODES, int D, int HOW>
struct HalfDecode {  // codes, 16 of a row a thread, through registers
  static constexpr int C = D / 16;
  uint4 w;
  float power;
  uint32_t to0, to1;  // where the piece's two halves go
  bool mine;
  __device__ __forceinline__ void init(const TileSource&) {
    const int e = threadIdx.x, row = e / C % 32, pc = e % C;
    mine = D == 128 || (e < 32 * C) == (HOW == kByRow);  // 64 channels: half the threads for K, half for V
    to0 = row * 2 * D + swz<D, HOW>(row, 2 * pc) * 16;
    to1 = row * 2 * D + swz<D, HOW>(row, 2 * pc + 1) * 16;
  }
  __device__ __forceinline__ void start(uint32_t, int j0, int ids, const TileSource& s, const TilePages& pg) {
    const int e = threadIdx.x, row = e / C % 32, pc = e % C;
    const int id = __shfl(ids, row), slot = pg.slot(j0 + row);
    w = make_uint4(0, 0, 0, 0);
    power = 0.f;
    if (id >= 0 && mine) {
      w = *reinterpret_cast<const uint4*>(s.p + id * s.page + slot * s.slot + pc * 16);
      power = power_of(s.e[id * s.e_page + slot]);
    }
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
template <typename E, int D, typename KCopy, typename VCopy>
__device__ __forceinline__ void attend_tiles(RowState<D / 32>& st, const uint16_t* qrow, uint32_t kb, uint32_t vb,
                                             const TileSource& ks, const TileSource& vs, const TilePages& pg,
                                             int tile0, int ntiles, int hi, int safe, float c) {
  constexpr int ND = D / 32, NC = D / 16;
  constexpr uint32_t kHalf = kKeys * D;  // bytes of half a tile
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const uint32_t kl = k_lane<D>(kb, lane & 31, half), vl = v_lane<D>(vb, lane);
  const int first = tile0 * kKeys, last = 2 * ntiles - 1;
  KCopy kc;
  VCopy vc;
  kc.init(ks);
  vc.init(vs);
  st.m = kNoMax;
  st.l = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) st.acc[dt] = f32x16{};
  const auto ids_of = [&](int n) __attribute__((always_inline)) { return pg.ids(first + 32 * min(n, last)); };
  const auto land = [&]() __attribute__((always_inline)) {
    wait_tile_copies();
    __syncthreads();
  };
  // Scores of half n: keys that are not visible become -inf.
  const auto mask = [&](f32x16& s, int n, int ids) __attribute__((always_inline)) {
    const uint32_t seen = static_cast<uint32_t>(__ballot(ids >= 0));
    const int j0 = first + 32 * n;
    if (seen != ~0u || j0 + 32 > safe) {
      const uint32_t bits = (seen >> (4 * half)) & ~bits_from(hi - j0 - 4 * half);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t w = bit_word(bits, r);
        s[r] = __uint_as_float((__float_as_uint(s[r]) & w) | (__float_as_uint(-INFINITY) & ~w));
      }
    }
  };
  // ids of the halves n to n + 3 in step n
  int i0 = ids_of(0), i1 = ids_of(1), i2 = ids_of(2), i3 = ids_of(3);
  kc.start(kb, first, i0, ks, pg);
  kc.finish(kb);
  kc.start(kb + kHalf, first + 32, i1, ks, pg);
  kc.finish(kb + kHalf);
  vc.start(vb, first, i0, vs, pg);
  vc.finish(vb);
  bf16x8 q[NC];
  load_row<D>(q, qrow, half);
  f32x16 sa, sb;  // scores of even and odd halves
  bf16x8 pa[2], pb[2];
  land();
  {  // step 0, without a stream: both halves are scored, the running max is the whole tile's
    f32x16 s0 = {}, s1 = {};
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) s0 = E::mfma32(k_op_x<D>(kl, 0, cc), q[cc], s0);
    __syncthreads();  // every wave is done with K(0)
    if (last > 1) kc.start(kb, first + 64, i2, ks, pg);
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) s1 = E::mfma32(k_op_x<D>(kl + kHalf, 0, cc), q[cc], s1);
    mask(s0, 0, i0);
    mask(s1, 1, i1);
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fmaxf(s0[r], s1[r]));
    st.m = fmaxf(kNoMax, xhalf_max(mx) * c);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = E::exp_pair(s0[2 * i], s0[2 * i + 1], c, -st.m, st.l);
    pa[0] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
    pa[1] = __builtin_bit_cast(bf16x8, make_uint4(w[4], w[5], w[6], w[7]));
    sb = s1;
    if (last > 1) kc.finish(kb);
  }
  mfma_fence(st.acc);  // O's zeros are in their registers before the asm MFMAs that add to them
  land();
  const auto next_ids = [&](int n) __attribute__((always_inline)) {
    i0 = i1, i1 = i2, i2 = i3;
    i3 = ids_of(n + 3);
  };
  const auto copies = [&](int n) __attribute__((always_inline)) {
    if (n + 2 <= last) kc.start(kb + (n & 1) * kHalf, first + 32 * (n + 2), i2, ks, pg);
    vc.start(vb + (n & 1) * kHalf, first + 32 * n, i0, vs, pg);
  };
  const auto landed = [&](int n) __attribute__((always_inline)) {
    if (n + 2 <= last) kc.finish(kb + (n & 1) * kHalf);
    vc.finish(vb + (n & 1) * kHalf);
    land();
  };
  const auto odd = [&](int n) __attribute__((always_inline)) {
    next_ids(n);
    copies(n);
    window_step<E, D>(st, sb, sa, pa, pb, kl, vl, q, c);
    landed(n);
  };
  const auto even = [&](int n) __attribute__((always_inline)) {
    next_ids(n);
    copies(n);
    mask(sa, n, i0);
    window_step<E, D>(st, sa, sb, pb, pa, kl + kHalf, vl + kHalf, q, c);
    mask(sb, n + 1, i1);
    landed(n);
  };
  int n = 1;
#pragma unroll 1
  for (; n < last; n += 2) {
    odd(n);
    even(n + 1);
  }
  odd(n);
  mfma_fence(st.acc);
#pragma unroll
  for (int i = 0; i < NC; ++i)  // P.V of the last half
    st.acc[i % ND] = E::mfma32(v_op_x<D>(vl + kHalf, i / ND, i % ND), pb[i / ND], st.acc[i % ND]);
}

}  // namespace solattn
