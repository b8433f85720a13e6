// Attention of one new token of each sequence over a key-value cache, paged or
// contiguous: the visible keys are split over workgroups and waves, each with an
// online softmax of its own, and joined.
//
// Per sequence b the token sits at position len - 1 and sees the keys j < len,
// with a window those with j >= len - window or j < sinks. A query head shares its
// kv head with group - 1 others; these (up to 16) are the columns of the tiles.
//
// Bound: HBM, 2 Hkv D values a visible key; the matrix instructions do 16 query
// columns whether they exist or not, 256 of their cycles for 16 KiB of cache. Four
// sequences of 32768 to 131072 tokens, 24 heads over 8, bf16: 232-251 us, 5.3-5.8
// TB/s (a large copy reaches 5.0); 32 of 512 to 16384, 16 heads of 64 over 4, pages of
// 16: 65-68 us, 4.1 TB/s, of it the kernel 54 and the join and its launch the rest; one
// sequence with a window of 4096: 10.2 us, two launches of the host's (kernels 5.9 and 4.7).
// A wave takes 32 keys at a time straight from HBM into operand registers, no LDS:
//   S^T = K Q^T (v_mfma_f32_16x16x32): row r of tile t is key 8 (r/4) + 4 t + r%4
//     of the 32, so lane (q, g) = (lane % 16, lane / 16) gets the scores of the
//     keys 8 g + 0..7: the order in which P is the B operand of the next product;
//   O^T += V^T P^T: a lane reads the same keys 8 g + 0..7, D / 16 channels each,
//     and transposes them in registers (v_perm_b32), one A operand per channel of
//     the D / 16: row i of operand j is channel (D / 16) i + j.
// The row's statistics need an exchange between the lanes g only.
#include "elem.hpp"

namespace solattn {
namespace {

constexpr int kWaves = 4;
constexpr int kStep = 32;       // keys of a wave's step
constexpr int kMaxSplits = 64;
constexpr int kGroups = 16;     // query columns of a tile

struct PagedArgs {
  const uint16_t* q;
  int64_t sq_b, sq_h;
  const uint16_t* k;
  int64_t sk_p, sk_s, sk_h;
  const uint16_t* v;
  int64_t sv_p, sv_s, sv_h;
  const int32_t* table;      // null: sequence b is page b
  int64_t table_b;
  const int32_t* lengths;    // with a table: each sequence's. Without: one shorter than `length` holds no token
                             // here, the others `length` keys (null: all of them)
  int length, pages, page, max_pages;
  Divisor by_page;
  uint16_t* o;
  int64_t so_b, so_h;
  float* part;               // split > 1: [B][H][split][D] sums, then [B][H][split][2] max and sum
  int64_t part_ml;           // where the latter begin
  int B, H, Hkv, D, group, tiles, split;
  Divisor by_tiles, by_hkv, by_split;
  int window, sinks;         // window 0: none
  float c;                   // scale log2(e)
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

// exp2 of the distance to a maximum; a row without keys has the maximum -inf and weight 0.
__device__ __forceinline__ float weight_of(float m, float top) {
  return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
}

// The visible keys as steps of 32: first those of the sinks below the window, then the window's.
struct Visible {
  int len, low;        // keys [low, len) and [0, sinks_end)
  int sinks_end;       // <= low
  int sink_steps, first, steps;  // the window's steps begin at key `first`
};
__device__ __forceinline__ Visible visible(const PagedArgs& a, int b) {
  Visible s;
  const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
  int n = a.lengths ? a.lengths[b] : a.length;
  if (!a.table) n = n < a.length ? 0 : a.length;
  s.len = static_cast<int>(min(static_cast<int64_t>(max(n, 0)), cap));
  s.low = a.window ? max(s.len - a.window, 0) : 0;
  s.sinks_end = min(a.sinks, s.low);
  s.sink_steps = (s.sinks_end + kStep - 1) / kStep;
  s.first = s.low & ~(kStep - 1);
  s.steps = s.sink_steps + (s.len - s.first + kStep - 1) / kStep;
  return s;
}

// DP: the head dim that the registers hold; D < DP (kFull false) leaves the rest zero.
template <typename E, int DP, bool kFull>
__global__ void __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
paged_kernel(const PagedArgs a) {
  constexpr int NC = DP / 32;   // 32-channel pieces of a score
  constexpr int CH = DP / 16;   // channels of a lane's V piece = operands of the second product
  constexpr int VW = CH / 2;    // their registers
  __shared__ float lds_o[kWaves][kGroups][DP + 4];
  __shared__ float lds_m[kWaves][kGroups], lds_l[kWaves][kGroups];

  fetch_arguments(a);
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  uint32_t w = blockIdx.x;
  const int tile = a.by_tiles.split(w), hk = a.by_hkv.split(w), split = a.by_split.split(w), b = w;
  const int ncol = min(kGroups, a.group - tile * kGroups);
  const int head0 = hk * a.group + tile * kGroups;

  const Visible vis = visible(a, b);
  const int per = a.by_split.of(vis.steps + a.split - 1);
  const int step0 = split * per, step1 = min(step0 + per, vis.steps);
  if (step0 >= step1 && a.split > 1) {  // nothing here: the join passes over a sum of 0
    if (static_cast<int>(threadIdx.x) < ncol)
      reinterpret_cast<float2*>(a.part + a.part_ml)[(static_cast<int64_t>(b) * a.H + head0 + threadIdx.x) * a.split + split] =
          make_float2(-INFINITY, 0.f);
    return;
  }

  bf16x8 q[NC];
  {
    const uint16_t* qp = a.q + b * a.sq_b + (head0 + min(col, ncol - 1)) * a.sq_h;
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      const int ch = 32 * cc + 8 * g;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (kFull || ch < a.D) x = *reinterpret_cast<const uint4*>(qp + ch);
      q[cc] = __builtin_bit_cast(bf16x8, x);
    }
  }
  f32x4 acc[CH];
#pragma unroll
  for (int j = 0; j < CH; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;  // l: this lane's keys

  const int vch = kFull || CH * col < a.D ? CH * col : 0;
  const auto base_of = [&](int st) __attribute__((always_inline)) {
    return st < vis.sink_steps ? st * kStep : vis.first + (st - vis.sink_steps) * kStep;
  };
  // Where the eight consecutive keys from j8 on are: they share a page (its size is a
  // multiple of 8, or the page is a whole sequence). Page ids are read a step ahead, so
  // that a step waits for one round of memory, not two.
  const auto slot_of = [&](int j8, int& slot) __attribute__((always_inline)) {
    const uint32_t j = static_cast<uint32_t>(min(j8, max(vis.len - 1, 0) & ~7));
    const uint32_t pg = a.by_page.of(j);
    slot = static_cast<int>(j - pg * a.page);
    return a.table ? a.table[b * a.table_b + pg] : b;
  };
  int kslot = 0, vslot = 0, kid = 0, vid = 0;
  if (step0 + wave < step1) {
    const int base = base_of(step0 + wave);
    kid = slot_of(base + 8 * (col >> 2), kslot);
    vid = slot_of(base + 8 * g, vslot);
  }
  for (int st = step0 + wave; st < step1; st += kWaves) {
    const bool sink = st < vis.sink_steps;
    const int base = base_of(st);
    const int lo = sink ? 0 : vis.low, hi = sink ? vis.sinks_end : vis.len;  // visible: lo <= j < hi
    // Keys of page ids outside the cache are not visible (a key's score lane holds its V piece too).
    const bool vok = vid >= 0 && vid < a.pages;
    const int64_t kpage = kid >= 0 && kid < a.pages ? kid : 0, vpage = vok ? vid : 0;
    const int last = a.page - 1;  // a slot past the page's end (a whole-sequence page) repeats its last
    bf16x8 kr[2][NC];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t* kp = a.k + kpage * a.sk_p + static_cast<int64_t>(min(kslot + 4 * t + (col & 3), last)) * a.sk_s + hk * a.sk_h;
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) {
        const int ch = 32 * cc + 8 * g;
        kr[t][cc] = *reinterpret_cast<const bf16x8*>(kp + (kFull || ch < a.D ? ch : 0));
      }
    }
    uint32_t vr[8][VW];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t* vp = a.v + vpage * a.sv_p + static_cast<int64_t>(min(vslot + i, last)) * a.sv_s + hk * a.sv_h + vch;
      if constexpr (VW == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(vp);
        vr[i][0] = x.x, vr[i][1] = x.y, vr[i][2] = x.z, vr[i][3] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(vp);
        vr[i][0] = x.x, vr[i][1] = x.y;
      }
    }
    if (st + kWaves < step1) {
      const int next = base_of(st + kWaves);
      kid = slot_of(next + 8 * (col >> 2), kslot);
      vid = slot_of(next + 8 * g, vslot);
    }
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) s[t] = E::mfma16(kr[t][cc], q[cc], s[t]);
    }
    // keys of this lane: base + 8 g + 4 t + i, i.e. those of its V piece
    if (base < lo || base + kStep > hi || __any(!vok)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = base + 8 * g + i;
        const bool on = vok && j >= lo && j < hi;
        s[i >> 2][i & 3] = on ? s[i >> 2][i & 3] : -INFINITY;
#pragma unroll
        for (int r = 0; r < VW; ++r) vr[i][r] = on ? vr[i][r] : 0u;  // 0 P of a value that may be anything
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
    const float m_new = fmaxf(m, over_groups_max(mx) * a.c);
    if (__any(m_new != m)) {
      const float alpha = weight_of(m, m_new);
      l *= alpha;
#pragma unroll
      for (int j = 0; j < CH; ++j) acc[j] *= alpha;
      m = m_new;
    }
    const float neg = m == -INFINITY ? 0.f : -m;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], a.c, neg));
      l += p[i];
    }
    const bf16x8 pb = __builtin_bit_cast(
        bf16x8, make_uint4(E::pack(p[0], p[1]), E::pack(p[2], p[3]), E::pack(p[4], p[5]), E::pack(p[6], p[7])));
#pragma unroll
    for (int j = 0; j < CH; ++j) {  // channel j of the lane's piece, its eight keys
      const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
      uint32_t x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = __builtin_amdgcn_perm(vr[2 * r + 1][j >> 1], vr[2 * r][j >> 1], sel);
      acc[j] = E::mfma16(__builtin_bit_cast(bf16x8, make_uint4(x[0], x[1], x[2], x[3])), pb, acc[j]);
    }
  }
  l = over_groups_sum(l);

  // Join the waves: O[q][channel], channel CH (4 g + i) + j in acc[j][i].
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < CH; ++j) lds_o[wave][col][CH * (4 * g + i) + j] = acc[j][i];
  if (g == 0) {
    lds_m[wave][col] = m;
    lds_l[wave][col] = l;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < ncol * (DP / 2); e += kWaves * 64) {
    const int qc = e / (DP / 2), ch = 2 * (e % (DP / 2));
    if (!kFull && ch >= a.D) continue;
    float top = lds_m[0][qc];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) top = fmaxf(top, lds_m[i][qc]);
    float o0 = 0.f, o1 = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float f = weight_of(lds_m[i][qc], top);
      o0 = fmaf(lds_o[i][qc][ch], f, o0);
      o1 = fmaf(lds_o[i][qc][ch + 1], f, o1);
      sum = fmaf(lds_l[i][qc], f, sum);
    }
    const int64_t row = static_cast<int64_t>(b) * a.H + head0 + qc;
    if (a.split > 1) {
      const int64_t at = row * a.split + split;
      *reinterpret_cast<float2*>(a.part + at * a.D + ch) = make_float2(o0, o1);
      if (ch == 0) *reinterpret_cast<float2*>(a.part + a.part_ml + 2 * at) = make_float2(top, sum);
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no visible key: zeros
      *reinterpret_cast<uint32_t*>(a.o + b * a.so_b + (head0 + qc) * a.so_h + ch) = E::pack(o0 * inv, o1 * inv);
    }
  }
}

// Joins the splits of a row: a wave per (b, head), two channels a lane.
template <typename E>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedArgs a) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= static_cast<int64_t>(a.B) * a.H) return;
  const int lane = threadIdx.x & 63, ch = 2 * lane;
  const float2* ml = reinterpret_cast<const float2*>(a.part + a.part_ml) + row * a.split;
  const float2 mine = lane < a.split ? ml[lane] : make_float2(-INFINITY, 0.f);  // (split <= 64)
  float top = mine.x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float f = weight_of(mine.x, top);
  float sum = mine.y * f;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
  const bool on = ch < a.D;
  const float* p = a.part + row * a.split * a.D + (on ? ch : 0);
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
      const float fi = i0 + u < used ? __shfl(f, i0 + u) : 0.f;  // (split <= 64, so i0 + u < 64)
      o0 = fmaf(x[u].x, fi, o0);
      o1 = fmaf(x[u].y, fi, o1);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (on)
    *reinterpret_cast<uint32_t*>(a.o + (row / a.H) * a.so_b + (row % a.H) * a.so_h + ch) = E::pack(o0 * inv, o1 * inv);
}

// Splits of a sequence: as many as leave the launch within four workgroups a CU, eight
// in a batch of sixteen or more, whose sequences are rarely of one length; of at least a
// step a wave as long as the longest sequence allows. (Within four against one more
// split: three sequences of 32768 keys 84 -> 81 us, five 138 -> 127. Within eight against four: 32
// ragged sequences of up to 16384 keys 61 -> 56, 72 of up to 4096 156 -> 134; 96 of
// 4096 each 275 -> 284. Four of 32768 to 131072: within two 281, four 250, eight 258.)
// No split is longer than 4096 keys as far as there may be 64 of them: one long sequence
// in a large batch is not left to one workgroup a head.
int splits(int64_t B, int64_t Hkv, int64_t tiles, int64_t most, int64_t window, int64_t sinks) {
  const int64_t keys = window && window < most && sinks < most - window ? window + sinks : most;
  const int64_t steps = cdiv(keys, kStep) + 1;
  int64_t n = (B < 16 ? 1024 : 2048) / (B * Hkv * tiles);
  if (n < cdiv(keys, 4096)) n = cdiv(keys, 4096);
  if (n > steps / kWaves) n = steps / kWaves;
  if (n > kMaxSplits) n = kMaxSplits;
  return n < 1 ? 1 : static_cast<int>(n);
}

int64_t part_bytes(int64_t B, int64_t H, int64_t D, int64_t split) {
  return split > 1 ? B * H * split * (D + 2) * 4 : 0;
}

}  // namespace

// Checked arguments of both entries; keys: the longest sequence that the cache can hold.
int paged_attn(const uint16_t* q, int64_t sq_b, int64_t sq_h, const uint16_t* k, int64_t sk_p, int64_t sk_s,
               int64_t sk_h, const uint16_t* v, int64_t sv_p, int64_t sv_s, int64_t sv_h, int64_t pages,
               int64_t page_size, const int32_t* table, int64_t table_stride, int64_t max_pages,
               const int32_t* lengths, int64_t length, int64_t B, int64_t H, int64_t Hkv, int64_t D, int dtype,
               int64_t window, int64_t sinks, float scale, void* workspace, int64_t workspace_bytes, uint16_t* o,
               int64_t so_b, int64_t so_h, hipStream_t s, const char* what) {
  SOLATTN_REQUIRE(dtype == SOLATTN_BF16 || dtype == SOLATTN_FP16, SOLATTN_EINVAL, "%s: dtype %d", what, dtype);
  SOLATTN_REQUIRE(B > 0 && H > 0 && Hkv > 0 && H % Hkv == 0, SOLATTN_EINVAL,
                  "%s: %lld query heads over %lld kv heads", what, (long long)H, (long long)Hkv);
  SOLATTN_REQUIRE(B < (1ll << 31) && H < (1ll << 31) && B * H < (1ll << 31), SOLATTN_EUNSUPPORTED, "%s: grid too large",
                  what);
  SOLATTN_REQUIRE(D >= 8 && D <= 128 && D % 8 == 0, SOLATTN_EUNSUPPORTED,
                  "%s: head_dim %lld (multiples of 8 up to 128)", what, (long long)D);
  SOLATTN_REQUIRE(window >= 0 && sinks >= 0 && window < (1ll << 31) && sinks < (1ll << 31), SOLATTN_EINVAL,
                  "%s: window %lld, sinks %lld", what, (long long)window, (long long)sinks);
  SOLATTN_REQUIRE(pages > 0 && pages < (1ll << 31) && page_size > 0 && max_pages >= 0 &&
                      (!table || page_size % 8 == 0),
                  SOLATTN_EINVAL, "%s: %lld pages of %lld (a multiple of 8)", what, (long long)pages,
                  (long long)page_size);
  SOLATTN_REQUIRE(page_size < (1ll << 31) && max_pages < (1ll << 31) && max_pages * page_size < (1ll << 31) - kStep,
                  SOLATTN_EUNSUPPORTED, "%s: sequences beyond 2^31 keys", what);
  SOLATTN_REQUIRE(scale > 0.f, SOLATTN_EINVAL, "%s: scale %g", what, static_cast<double>(scale));
  SOLATTN_REQUIRE(q && k && v && o, SOLATTN_EINVAL, "%s: null pointer", what);
  const auto rows = [](const void* p, int64_t x, int64_t y, int64_t z) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && x % 8 == 0 && y % 8 == 0 && z % 8 == 0;
  };
  SOLATTN_REQUIRE(rows(q, sq_b, sq_h, 0) && rows(k, sk_p, sk_s, sk_h) && rows(v, sv_p, sv_s, sv_h) &&
                      rows(o, so_b, so_h, 0),
                  SOLATTN_EINVAL, "%s: rows must be 16-byte aligned with strides multiple of 8", what);
  PagedArgs a{};
  a.q = q, a.sq_b = sq_b, a.sq_h = sq_h;
  a.k = k, a.sk_p = sk_p, a.sk_s = sk_s, a.sk_h = sk_h;
  a.v = v, a.sv_p = sv_p, a.sv_s = sv_s, a.sv_h = sv_h;
  a.table = table, a.table_b = table_stride;
  a.lengths = lengths, a.length = static_cast<int>(length);
  a.pages = static_cast<int>(pages), a.page = static_cast<int>(page_size), a.max_pages = static_cast<int>(max_pages);
  a.by_page = divisor(page_size);
  a.o = o, a.so_b = so_b, a.so_h = so_h;
  a.B = static_cast<int>(B), a.H = static_cast<int>(H), a.Hkv = static_cast<int>(Hkv), a.D = static_cast<int>(D);
  a.group = static_cast<int>(H / Hkv);
  a.tiles = static_cast<int>(cdiv(a.group, kGroups));
  a.window = static_cast<int>(window), a.sinks = static_cast<int>(sinks);
  a.c = scale * kLog2e;
  a.split = splits(B, Hkv, a.tiles, max_pages * page_size, window, sinks);
  a.by_tiles = divisor(a.tiles), a.by_hkv = divisor(Hkv), a.by_split = divisor(a.split);
  const int64_t need = part_bytes(B, H, D, a.split);
  SOLATTN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), SOLATTN_ESIZE,
                  "%s: workspace %lld < %lld bytes", what, (long long)workspace_bytes, (long long)need);
  SOLATTN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, SOLATTN_EINVAL,
                  "%s: workspace must be 256-byte aligned", what);
  a.part = static_cast<float*>(workspace);
  a.part_ml = B * H * a.split * D;
  const int64_t grid = B * Hkv * a.tiles * a.split;
  SOLATTN_REQUIRE(grid < (1ll << 31), SOLATTN_EUNSUPPORTED, "%s: grid too large", what);
  const bool bf = dtype == SOLATTN_BF16;
  const auto kern = D == 128 ? (bf ? paged_kernel<Bf16, 128, true> : paged_kernel<Fp16, 128, true>)
                    : D == 64 ? (bf ? paged_kernel<Bf16, 64, true> : paged_kernel<Fp16, 64, true>)
                    : D > 64  ? (bf ? paged_kernel<Bf16, 128, false> : paged_kernel<Fp16, 128, false>)
                              : (bf ? paged_kernel<Bf16, 64, false> : paged_kernel<Fp16, 64, false>);
  hipLaunchKernelGGL(kern, dim3(static_cast<uint32_t>(grid)), dim3(kWaves * 64), 0, s, a);
  if (int rc = check_launch(what)) return rc;
  if (a.split == 1) return SOLATTN_OK;
  hipLaunchKernelGGL(bf ? paged_join_kernel<Bf16> : paged_join_kernel<Fp16>,
                     dim3(static_cast<uint32_t>(cdiv(B * H, 4))), dim3(256), 0, s, a);
  return check_launch(what);
}

int64_t paged_attn_workspace(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t keys, int64_t window,
                             int64_t sinks) {
  constexpr int64_t top = 1ll << 31;  // (what the call takes: nothing passes 64 bits)
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || keys < 0 || window < 0 || sinks < 0) return 0;
  if (B >= top || H >= top || B * H >= top || D > 128 || keys >= top) return 0;
  return part_bytes(B, H, D, splits(B, Hkv, cdiv(H / Hkv, kGroups), keys, window, sinks));
}

}  // namespace solattn

using namespace solattn;

extern "C" int64_t solattn_paged_attn_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t max_pages,
                                                      int64_t page_size, int64_t window, int64_t sinks) {
  const bool fit = max_pages >= 0 && page_size >= 0 && max_pages < (1ll << 31) && page_size < (1ll << 31);
  return fit ? paged_attn_workspace(B, H, Hkv, D, max_pages * page_size, window, sinks) : 0;
}

extern "C" int solattn_paged_attn(const uint16_t* q, int64_t sq_b, int64_t sq_h, const uint16_t* k_cache,
                                  int64_t sk_p, int64_t sk_s, int64_t sk_h, const uint16_t* v_cache, int64_t sv_p,
                                  int64_t sv_s, int64_t sv_h, int64_t pages, int64_t page_size,
                                  const int32_t* page_table, int64_t table_stride, int64_t max_pages,
                                  const int32_t* lengths, int64_t B, int64_t H, int64_t Hkv, int64_t D, int dtype,
                                  int64_t window, int64_t sinks, float scale, void* workspace,
                                  int64_t workspace_bytes, uint16_t* o, int64_t so_b, int64_t so_h,
                                  solattn_stream_t stream) {
  clear_error();
  SOLATTN_REQUIRE(page_table && lengths, SOLATTN_EINVAL, "paged_attn: null page table or lengths");
  return paged_attn(q, sq_b, sq_h, k_cache, sk_p, sk_s, sk_h, v_cache, sv_p, sv_s, sv_h, pages, page_size, page_table,
                    table_stride, max_pages, lengths, 0, B, H, Hkv, D, dtype, window, sinks, scale, workspace,
                    workspace_bytes, o, so_b, so_h, reinterpret_cast<hipStream_t>(stream), "paged_attn");
}
