// Norms of queries and keys per head with the position rotation in the same
// pass, forward and backward, and the form for new tokens that writes k and v
// into a paged cache.
//
// A row is one head of one token: x in R^D. With r = 1 / sqrt(mean(x^2) + eps)
// and n = x r w, the first R channels turn in pairs by the token's angles,
//   y1 = n1 cos - n2 sin,  y2 = n2 cos + n1 sin,
// pairs (i, i + R/2) or, interleaved, (2i, 2i + 1); the others are n.
// Backward, with g = dy turned back and u = g w:
//   dx = r (u - x r^2 mean(u x)),   dw = sum over rows of g x r.
// Everything is fp32 between the load and the one rounding at the store.
//
// Bound: HBM; for a few tokens the launch. 32760 tokens of 24 + 24 heads of 128
// channels, bf16: 156 us, 5.25 TB/s (a large copy reaches 5.0); one token of each of
// four sequences into its pages: 7 us a call (the host's), the kernel 4.9; gradients of 8200
// tokens of 16 + 4 heads of 64, fp16: 17 us and 4.9 for the weights' join, 3.7 TB/s.
// A lane holds 8 channels, so a row is LPR = 16 lanes (8 up to 64
// channels) and a wave works on G = 64 / LPR rows at a time, all of the same
// token: the token's cos and sin and the weights stay in registers while the
// wave walks the heads (a table entry is 8 bytes a pair, as much as two rows'
// values). Few tokens: their heads are dealt over S waves, so that one decode
// step is one or two rounds of loads.
#include "elem.hpp"

namespace solattn {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kUnroll = 4;          // rows in flight per lane
constexpr int kRopeMaxD = 128;
constexpr int kWaveTarget = 2048;   // waves below which a token's heads are dealt over more of them
constexpr int kBwdBlocks = 1024;    // workgroups of the backward: rows of its weight-gradient partials

struct Rows {  // a BTHD tensor, strides in elements
  void* p;
  int64_t b, t, h;
};

struct Cache {
  void* k;
  void* v;
  int64_t kp, ks, kh, vp, vs, vh;  // page, slot and head strides
  const int32_t* table;
  int64_t table_b;
  const int32_t* lengths;
  int npages, page, max_pages;
};

struct RopeArgs {
  Rows q, k, v;      // inputs
  Rows qo, ko;       // forward: outputs; backward: gradients of the inputs
  Rows dq, dk;       // backward: gradients of the outputs
  const float* qw;
  const float* kw;
  const float* cos;
  const float* sin;
  const int32_t* positions;
  int64_t pos_b;
  float* part;       // backward: [gridDim.x][2][D]
  float eps, inv_d;
  int T, H, Hkv, D, P, R, interleaved;
  int64_t tokens;    // B T
  int split, tpw;    // waves per token; tokens per wave (one of the two is 1)
  Cache cache;
};

// Sum over the LPR lanes of a row; every lane gets it.
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#define SOLATTN_DPP_ADD(ctrl) \
  x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), ctrl, 0xf, 0xf, true))
  SOLATTN_DPP_ADD(0xB1);   // quad_perm 1 0 3 2
  SOLATTN_DPP_ADD(0x4E);   // quad_perm 2 3 0 1
  SOLATTN_DPP_ADD(0x141);  // row_half_mirror
  if constexpr (LPR == 16) SOLATTN_DPP_ADD(0x140);  // row_mirror
#undef SOLATTN_DPP_ADD
  return x;
}

// What a lane keeps of its token's rotation: y = x c + partner(x) s, with the
// sign of the pair's half in s. Lanes past R: c = 1, s = 0.
struct Turn {
  float c[8], s[8];
  int partner;  // lane that holds the other halves (half-split pairs)
};

template <int LPR>
__device__ __forceinline__ void load_turn(Turn& t, const RopeArgs& a, int pos, int l, int lane) {
  const int half = a.R >> 1;
  t.partner = lane;
#pragma unroll
  for (int i = 0; i < 8; ++i) t.c[i] = 1.f, t.s[i] = 0.f;
  if (8 * l >= a.R) return;
  const int64_t at = static_cast<int64_t>(pos) * half;
  if (a.interleaved) {
    const float4 c = *reinterpret_cast<const float4*>(a.cos + at + 4 * l);
    const float4 s = *reinterpret_cast<const float4*>(a.sin + at + 4 * l);
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t.c[2 * i] = t.c[2 * i + 1] = cc[i];
      t.s[2 * i] = -ss[i];
      t.s[2 * i + 1] = ss[i];
    }
  } else {
    const bool first = 8 * l < half;
    const int i0 = first ? 8 * l : 8 * l - half;
    t.partner = first ? lane + (half >> 3) : lane - (half >> 3);
    const float sign = first ? -1.f : 1.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 c = *reinterpret_cast<const float4*>(a.cos + at + i0 + 4 * j);
      const float4 s = *reinterpret_cast<const float4*>(a.sin + at + i0 + 4 * j);
      t.c[4 * j] = c.x, t.c[4 * j + 1] = c.y, t.c[4 * j + 2] = c.z, t.c[4 * j + 3] = c.w;
      t.s[4 * j] = sign * s.x, t.s[4 * j + 1] = sign * s.y, t.s[4 * j + 2] = sign * s.z, t.s[4 * j + 3] = sign * s.w;
    }
  }
}

// dir = 1: turned by the angles, -1: turned back.
__device__ __forceinline__ void turn(float (&x)[8], const Turn& t, int interleaved, float dir) {
  float o[8];
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = x[i ^ 1];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl(x[i], t.partner);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(o[i], dir * t.s[i], x[i] * t.c[i]);
}

__device__ __forceinline__ void load_weight(float (&w)[8], const float* p, int l, bool active) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (p == nullptr || !active) return;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float4 v = reinterpret_cast<const float4*>(p + 8 * l)[j];
    w[4 * j] = v.x, w[4 * j + 1] = v.y, w[4 * j + 2] = v.z, w[4 * j + 3] = v.w;
  }
}

// Where a wave's lane works: token (b, t) and the heads first, first + step, ...
struct Place {
  int64_t b;
  int t, first, step;
  bool on;
};

template <int LPR>
__device__ __forceinline__ Place place(const RopeArgs& a, int64_t wave, int group) {
  constexpr int G = 64 / LPR;
  Place p;
  int64_t token;
  if (a.tpw > 1) {  // fewer rows in a token than a wave holds: several tokens, one pass
    const int per = G / a.tpw;
    token = wave * a.tpw + group / per;
    p.first = group % per;
    p.step = per;
    p.on = group / per < a.tpw;
  } else {
    token = wave / a.split;
    p.first = static_cast<int>(wave % a.split) * G + group;
    p.step = a.split * G;
    p.on = true;
  }
  p.on = p.on && token < a.tokens;
  if (token >= a.tokens) token = a.tokens - 1;
  p.b = token / a.T;
  p.t = static_cast<int>(token - p.b * a.T);
  return p;
}

template <typename E>
__device__ __forceinline__ typename E::Raw* row_of(const Rows& r, int64_t b, int64_t t, int64_t h) {
  return static_cast<typename E::Raw*>(r.p) + b * r.b + t * r.t + h * r.h;
}

// One tensor's heads of this lane's token: norm, rotation, store at dst(h).
// Every lane of a wave makes the same passes (its rows' sums and exchanges are
// wave operations); heads past `heads` read the last one and are not stored.
template <typename E, int LPR, typename Dst>
__device__ __forceinline__ void norm_turn_rows(const RopeArgs& a, const Rows& src, const Place& p, int heads,
                                               const float* weight, const Turn& tr, int l, bool active, bool store,
                                               Dst&& dst) {
  float w[8];
  load_weight(w, weight, l, active);
  const int n = (heads + p.step - 1) / p.step;
  const int chan = active ? 8 * l : 0;
  for (int i0 = 0; i0 < n; i0 += kUnroll) {
    Row8<E> in[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i0 + u < n) in[u].load(row_of<E>(src, p.b, p.t, min(p.first + (i0 + u) * p.step, heads - 1)) + chan);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (i0 + u >= n) break;
      float x[8], ss = 0.f;
      in[u].get(x);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
      const float r = rsqrtf(fmaf(row_sum<LPR>(active ? ss : 0.f), a.inv_d, a.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
      if (a.R) turn(x, tr, a.interleaved, 1.f);
      const int h = p.first + (i0 + u) * p.step;
      if (store && active && h < heads) Row8<E>::store(dst(h) + chan, x);
    }
  }
}

template <typename E, int LPR, bool APPEND>
__global__ void __launch_bounds__(kRopeThreads) qk_rope_kernel(const RopeArgs a) {
  const int lane = threadIdx.x & 63, l = lane & (LPR - 1), group = lane / LPR;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * (kRopeThreads / 64) + (threadIdx.x >> 6);
  const Place p = place<LPR>(a, wave, group);
  const bool active = 8 * l < a.D;
  int pos = p.t;
  bool keep = p.on;  // the token has a position (append: the sequence holds it)
  if constexpr (APPEND) {
    const int64_t cap = static_cast<int64_t>(a.cache.max_pages) * a.cache.page;
    const int64_t at = static_cast<int64_t>(a.cache.lengths[p.b]) - a.T + p.t;
    keep = keep && at >= 0 && at < cap;
    pos = static_cast<int>(at < 0 ? 0 : at < cap ? at : cap - 1);
  } else if (a.positions) {
    pos = a.positions[p.b * a.pos_b + p.t];
  }
  Turn tr;
  if (a.R) load_turn<LPR>(tr, a, min(max(pos, 0), a.P - 1), l, lane);
  if constexpr (!APPEND) {
    norm_turn_rows<E, LPR>(a, a.q, p, a.H, a.qw, tr, l, active, p.on,
                           [&](int h) { return row_of<E>(a.qo, p.b, p.t, h); });
    norm_turn_rows<E, LPR>(a, a.k, p, a.Hkv, a.kw, tr, l, active, p.on,
                           [&](int h) { return row_of<E>(a.ko, p.b, p.t, h); });
  } else {
    // q rows of tokens without a position are written too: they are finite and no
    // attention call reads them as anything but an empty row
    norm_turn_rows<E, LPR>(a, a.q, p, a.H, a.qw, tr, l, active, p.on,
                           [&](int h) { return row_of<E>(a.qo, p.b, p.t, h); });
    const Cache& c = a.cache;
    const int page = c.max_pages ? c.table[p.b * c.table_b + pos / c.page] : -1;
    const bool put = keep && page >= 0 && page < c.npages;
    const int64_t kat = put ? static_cast<int64_t>(page) * c.kp + static_cast<int64_t>(pos % c.page) * c.ks : 0;
    const int64_t vat = put ? static_cast<int64_t>(page) * c.vp + static_cast<int64_t>(pos % c.page) * c.vs : 0;
    typename E::Raw* kc = static_cast<typename E::Raw*>(c.k) + kat;
    typename E::Raw* vc = static_cast<typename E::Raw*>(c.v) + vat;
    norm_turn_rows<E, LPR>(a, a.k, p, a.Hkv, a.kw, tr, l, active, put, [&](int h) { return kc + h * c.kh; });
    if (put && active)
      for (int h = p.first; h < a.Hkv; h += p.step) {
        Row8<E> in;
        in.load(row_of<E>(a.v, p.b, p.t, h) + 8 * l);
        *reinterpret_cast<Row8<E>*>(vc + h * c.vh + 8 * l) = in;
      }
  }
}

// One tensor's gradients: dx, and g x r added to this lane's weight gradient.
template <typename E, int LPR>
__device__ __forceinline__ void norm_turn_rows_bwd(const RopeArgs& a, const Rows& src, const Rows& dy, const Rows& dx,
                                                   const Place& p, int heads, const float (&w)[8], const Turn& tr,
                                                   int l, bool active, float (&dw)[8]) {
  constexpr int U = 2;
  const int n = (heads + p.step - 1) / p.step;
  const int chan = active ? 8 * l : 0;
  for (int i0 = 0; i0 < n; i0 += U) {
    Row8<E> in[U], gin[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u < n) {
        const int h = min(p.first + (i0 + u) * p.step, heads - 1);
        in[u].load(row_of<E>(src, p.b, p.t, h) + chan);
        gin[u].load(row_of<E>(dy, p.b, p.t, h) + chan);
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u >= n) break;
      const int h = p.first + (i0 + u) * p.step;
      const bool on = p.on && active && h < heads;
      float x[8], g[8], ss = 0.f, ux = 0.f;
      in[u].get(x);
      gin[u].get(g);
      if (a.R) turn(g, tr, a.interleaved, -1.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss = fmaf(x[i], x[i], ss);
        ux = fmaf(g[i] * w[i], x[i], ux);
      }
      const float r = rsqrtf(fmaf(row_sum<LPR>(active ? ss : 0.f), a.inv_d, a.eps));
      const float m = r * r * row_sum<LPR>(active ? ux : 0.f) * a.inv_d;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float gx = g[i] * x[i] * r;
        dw[i] += on ? gx : 0.f;
        x[i] = r * (g[i] * w[i] - x[i] * m);
      }
      if (on) Row8<E>::store(row_of<E>(dx, p.b, p.t, h) + chan, x);
    }
  }
}

// The workgroups walk the tokens with a fixed stride and sum their weight
// gradients in registers, in an order that the launch alone fixes; one row of
// partials per workgroup, summed by qk_rope_dw_kernel. No atomics.
template <typename E, int LPR>
__global__ void __launch_bounds__(kRopeThreads) qk_rope_bwd_kernel(const RopeArgs a) {
  constexpr int W = kRopeThreads / 64;
  __shared__ float sum[W][2][kRopeMaxD];
  const int lane = threadIdx.x & 63, l = lane & (LPR - 1), group = lane / LPR, wv = threadIdx.x >> 6;
  const bool active = 8 * l < a.D;
  float dqw[8] = {}, dkw[8] = {}, qw[8], kw[8];
  load_weight(qw, a.qw, l, active);
  load_weight(kw, a.kw, l, active);
  const int64_t waves = (a.tokens * a.split + a.tpw - 1) / a.tpw;
  for (int64_t w0 = static_cast<int64_t>(blockIdx.x) * W; w0 < waves; w0 += static_cast<int64_t>(gridDim.x) * W) {
    const Place p = place<LPR>(a, w0 + wv, group);  // (a wave past the last: nothing stored or summed)
    const int pos = a.positions ? a.positions[p.b * a.pos_b + p.t] : p.t;
    Turn tr;
    if (a.R) load_turn<LPR>(tr, a, min(max(pos, 0), a.P - 1), l, lane);
    norm_turn_rows_bwd<E, LPR>(a, a.q, a.dq, a.qo, p, a.H, qw, tr, l, active, dqw);
    norm_turn_rows_bwd<E, LPR>(a, a.k, a.dk, a.ko, p, a.Hkv, kw, tr, l, active, dkw);
  }
  if (a.part == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // the wave's rows
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1) {
      dqw[i] += __shfl_xor(dqw[i], o);
      dkw[i] += __shfl_xor(dkw[i], o);
    }
  }
  if (group == 0 && active)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum[wv][0][8 * l + i] = dqw[i];
      sum[wv][1][8 * l + i] = dkw[i];
    }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * a.D; e += kRopeThreads) {
    const int which = e / a.D, d = e % a.D;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) t += sum[i][which][d];
    a.part[static_cast<int64_t>(blockIdx.x) * 2 * a.D + e] = t;
  }
}

// Columns of part [n][2][D] summed: a workgroup takes 16 of them, 16 threads a column.
__global__ void __launch_bounds__(256) qk_rope_dw_kernel(const float* __restrict__ part, int n, int D,
                                                         float* __restrict__ dqw, float* __restrict__ dkw) {
  __shared__ float sum[16][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  float t = 0.f;
  if (col < 2 * D) {
#pragma unroll 8
    for (int i = g; i < n; i += 16) t += part[static_cast<int64_t>(i) * 2 * D + col];
  }
  sum[g][c] = t;
  __syncthreads();
  if (threadIdx.x >= 16 || col >= 2 * D) return;
  t = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) t += sum[i][c];
  float* out = col < D ? dqw : dkw;
  if (out) out[col < D ? col : col - D] = t;
}

int esize(int dtype) { return dtype == SOLATTN_FP32 ? 4 : 2; }

int check_rows(const Rows& r, int e, const char* what, const char* name) {
  const int64_t m = 16 / e;  // rows are read and written in 16-byte pieces
  SOLATTN_REQUIRE(r.p, SOLATTN_EINVAL, "%s: null %s", what, name);
  SOLATTN_REQUIRE(reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.b % m == 0 && r.t % m == 0 && r.h % m == 0,
                  SOLATTN_EINVAL, "%s: %s must be 16-byte aligned with strides that keep its rows so", what, name);
  return 0;
}

// Sizes and launch shape; fills a.
int setup(RopeArgs& a, int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t D, int dtype, int64_t P, int64_t R,
          int interleaved, float eps, const char* what) {
  SOLATTN_REQUIRE(dtype >= SOLATTN_BF16 && dtype <= SOLATTN_FP32, SOLATTN_EINVAL, "%s: dtype %d", what, dtype);
  SOLATTN_REQUIRE(B > 0 && T > 0 && H > 0 && Hkv >= 0, SOLATTN_EINVAL, "%s: bad sizes", what);
  SOLATTN_REQUIRE(D >= 8 && D <= kRopeMaxD && D % 8 == 0, SOLATTN_EUNSUPPORTED,
                  "%s: head_dim %lld (multiples of 8 up to %d)", what, (long long)D, kRopeMaxD);
  SOLATTN_REQUIRE(R >= 0 && R <= D && R % (interleaved ? 8 : 16) == 0, SOLATTN_EUNSUPPORTED,
                  "%s: %lld rotated channels of %lld (multiples of %d)", what, (long long)R, (long long)D,
                  interleaved ? 8 : 16);
  SOLATTN_REQUIRE(eps >= 0.f, SOLATTN_EINVAL, "%s: eps %g", what, static_cast<double>(eps));
  SOLATTN_REQUIRE(R == 0 || (a.cos && a.sin && P > 0), SOLATTN_EINVAL, "%s: rotation without a table", what);
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  SOLATTN_REQUIRE(aligned(a.qw) && aligned(a.kw) && (R == 0 || (aligned(a.cos) && aligned(a.sin))), SOLATTN_EINVAL,
                  "%s: weights and tables must be 16-byte aligned", what);
  SOLATTN_REQUIRE(T < (1ll << 31) && H < (1ll << 24) && Hkv < (1ll << 24) && P < (1ll << 31) && B < (1ll << 31) &&
                      B * T < (1ll << 31),
                  SOLATTN_EUNSUPPORTED, "%s: too many tokens or heads", what);
  a.T = static_cast<int>(T);
  a.H = static_cast<int>(H);
  a.Hkv = static_cast<int>(Hkv);
  a.D = static_cast<int>(D);
  a.P = static_cast<int>(P);
  a.R = static_cast<int>(R);
  a.interleaved = interleaved;
  a.eps = eps;
  a.inv_d = 1.f / static_cast<float>(D);
  a.tokens = B * T;
  const int G = D > 64 ? 4 : 8;
  const int64_t most = H > Hkv ? H : Hkv;
  a.tpw = 1;
  while (a.tpw * 2 * most <= G && a.tpw * 2 <= G) a.tpw *= 2;
  a.split = 1;
  while (a.tpw == 1 && a.tokens * a.split * 2 <= kWaveTarget && a.split * G < most) a.split *= 2;
  return 0;
}

int64_t wave_count(const RopeArgs& a) { return (a.tokens * a.split + a.tpw - 1) / a.tpw; }

template <bool APPEND>
int launch(const RopeArgs& a, int dtype, hipStream_t s, const char* what) {
  const int64_t blocks = cdiv(wave_count(a), kRopeThreads / 64);
  SOLATTN_REQUIRE(blocks < (1ll << 31), SOLATTN_EUNSUPPORTED, "%s: grid too large", what);
  const dim3 grid(static_cast<uint32_t>(blocks)), block(kRopeThreads);
  const bool wide = a.D > 64;
  const auto kern = dtype == SOLATTN_BF16   ? (wide ? qk_rope_kernel<Bf16, 16, APPEND> : qk_rope_kernel<Bf16, 8, APPEND>)
                    : dtype == SOLATTN_FP16 ? (wide ? qk_rope_kernel<Fp16, 16, APPEND> : qk_rope_kernel<Fp16, 8, APPEND>)
                                            : (wide ? qk_rope_kernel<Fp32, 16, APPEND> : qk_rope_kernel<Fp32, 8, APPEND>);
  hipLaunchKernelGGL(kern, grid, block, 0, s, a);
  return check_launch(what);
}

uint32_t bwd_blocks(const RopeArgs& a) {
  const int64_t blocks = cdiv(wave_count(a), kRopeThreads / 64);
  return static_cast<uint32_t>(blocks < kBwdBlocks ? blocks : kBwdBlocks);
}

}  // namespace
}  // namespace solattn

using namespace solattn;

extern "C" int solattn_qk_norm_rope(const void* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const void* k,
                                    int64_t sk_b, int64_t sk_t, int64_t sk_h, int64_t B, int64_t T, int64_t H,
                                    int64_t Hkv, int64_t D, int dtype, const float* q_weight, const float* k_weight,
                                    const float* cos, const float* sin, int64_t P, int64_t R, int interleaved,
                                    const int32_t* positions, int64_t pos_stride_b, float eps, void* qo,
                                    int64_t sqo_b, int64_t sqo_t, int64_t sqo_h, void* ko, int64_t sko_b,
                                    int64_t sko_t, int64_t sko_h, solattn_stream_t stream) {
  clear_error();
  RopeArgs a{};
  a.q = {const_cast<void*>(q), sq_b, sq_t, sq_h};
  a.k = {const_cast<void*>(k), sk_b, sk_t, sk_h};
  a.qo = {qo, sqo_b, sqo_t, sqo_h};
  a.ko = {ko, sko_b, sko_t, sko_h};
  a.qw = q_weight;
  a.kw = k_weight;
  a.cos = cos;
  a.sin = sin;
  a.positions = positions;
  a.pos_b = pos_stride_b;
  if (int rc = setup(a, B, T, H, Hkv, D, dtype, P, R, interleaved, eps, "qk_norm_rope")) return rc;
  SOLATTN_REQUIRE(R == 0 || positions || T <= P, SOLATTN_EINVAL, "qk_norm_rope: %lld tokens, a table of %lld",
                  (long long)T, (long long)P);
  const int e = esize(dtype);
  int rc = check_rows(a.q, e, "qk_norm_rope", "q");
  if (!rc) rc = check_rows(a.qo, e, "qk_norm_rope", "q output");
  if (!rc && Hkv) rc = check_rows(a.k, e, "qk_norm_rope", "k");
  if (!rc && Hkv) rc = check_rows(a.ko, e, "qk_norm_rope", "k output");
  if (rc) return rc;
  return launch<false>(a, dtype, reinterpret_cast<hipStream_t>(stream), "qk_norm_rope");
}

extern "C" int solattn_qk_norm_rope_append(
    const void* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
    const void* v, int64_t sv_b, int64_t sv_t, int64_t sv_h, int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t D,
    int dtype, const float* q_weight, const float* k_weight, const float* cos, const float* sin, int64_t P, int64_t R,
    int interleaved, float eps, void* qo, int64_t sqo_b, int64_t sqo_t, int64_t sqo_h, void* k_cache, int64_t skc_p,
    int64_t skc_s, int64_t skc_h, void* v_cache, int64_t svc_p, int64_t svc_s, int64_t svc_h, int64_t pages,
    int64_t page_size, const int32_t* page_table, int64_t table_stride, int64_t max_pages, const int32_t* lengths,
    solattn_stream_t stream) {
  clear_error();
  const char* what = "qk_norm_rope_append";
  RopeArgs a{};
  a.q = {const_cast<void*>(q), sq_b, sq_t, sq_h};
  a.k = {const_cast<void*>(k), sk_b, sk_t, sk_h};
  a.v = {const_cast<void*>(v), sv_b, sv_t, sv_h};
  a.qo = {qo, sqo_b, sqo_t, sqo_h};
  a.qw = q_weight;
  a.kw = k_weight;
  a.cos = cos;
  a.sin = sin;
  if (int rc = setup(a, B, T, H, Hkv, D, dtype, P, R, interleaved, eps, what)) return rc;
  SOLATTN_REQUIRE(Hkv > 0 && page_table && lengths, SOLATTN_EINVAL, "%s: null page table or lengths", what);
  SOLATTN_REQUIRE(pages >= 0 && pages < (1ll << 31) && page_size > 0 && page_size < (1ll << 31) && max_pages >= 0 &&
                      max_pages < (1ll << 31) && max_pages * page_size < (1ll << 31),
                  SOLATTN_EUNSUPPORTED, "%s: pages beyond 2^31 tokens", what);
  const int e = esize(dtype);
  const Rows kc{k_cache, skc_p, skc_s, skc_h}, vc{v_cache, svc_p, svc_s, svc_h};
  int rc = check_rows(a.q, e, what, "q");
  if (!rc) rc = check_rows(a.k, e, what, "k");
  if (!rc) rc = check_rows(a.v, e, what, "v");
  if (!rc) rc = check_rows(a.qo, e, what, "q output");
  if (!rc) rc = check_rows(kc, e, what, "k_cache");
  if (!rc) rc = check_rows(vc, e, what, "v_cache");
  if (rc) return rc;
  a.cache = {k_cache, v_cache, skc_p, skc_s, skc_h, svc_p, svc_s, svc_h, page_table, table_stride, lengths,
             static_cast<int>(pages), static_cast<int>(page_size), static_cast<int>(max_pages)};
  return launch<true>(a, dtype, reinterpret_cast<hipStream_t>(stream), what);
}

extern "C" int64_t solattn_qk_norm_rope_bwd_workspace_bytes(int64_t D) {
  return D <= 0 ? 0 : static_cast<int64_t>(kBwdBlocks) * 2 * D * 4;
}

extern "C" int solattn_qk_norm_rope_bwd(
    const void* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
    const void* dqo, int64_t sdq_b, int64_t sdq_t, int64_t sdq_h, const void* dko, int64_t sdk_b, int64_t sdk_t,
    int64_t sdk_h, int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t D, int dtype, const float* q_weight,
    const float* k_weight, const float* cos, const float* sin, int64_t P, int64_t R, int interleaved,
    const int32_t* positions, int64_t pos_stride_b, float eps, void* dq, int64_t sgq_b, int64_t sgq_t, int64_t sgq_h,
    void* dk, int64_t sgk_b, int64_t sgk_t, int64_t sgk_h, float* dq_weight, float* dk_weight, void* workspace,
    int64_t workspace_bytes, solattn_stream_t stream) {
  clear_error();
  const char* what = "qk_norm_rope_bwd";
  RopeArgs a{};
  a.q = {const_cast<void*>(q), sq_b, sq_t, sq_h};
  a.k = {const_cast<void*>(k), sk_b, sk_t, sk_h};
  a.dq = {const_cast<void*>(dqo), sdq_b, sdq_t, sdq_h};
  a.dk = {const_cast<void*>(dko), sdk_b, sdk_t, sdk_h};
  a.qo = {dq, sgq_b, sgq_t, sgq_h};
  a.ko = {dk, sgk_b, sgk_t, sgk_h};
  a.qw = q_weight;
  a.kw = k_weight;
  a.cos = cos;
  a.sin = sin;
  a.positions = positions;
  a.pos_b = pos_stride_b;
  if (int rc = setup(a, B, T, H, Hkv, D, dtype, P, R, interleaved, eps, what)) return rc;
  SOLATTN_REQUIRE(R == 0 || positions || T <= P, SOLATTN_EINVAL, "%s: %lld tokens, a table of %lld", what,
                  (long long)T, (long long)P);
  const int e = esize(dtype);
  int rc = check_rows(a.q, e, what, "q");
  if (!rc) rc = check_rows(a.dq, e, what, "q output's gradient");
  if (!rc) rc = check_rows(a.qo, e, what, "q gradient");
  if (!rc && Hkv) rc = check_rows(a.k, e, what, "k");
  if (!rc && Hkv) rc = check_rows(a.dk, e, what, "k output's gradient");
  if (!rc && Hkv) rc = check_rows(a.ko, e, what, "k gradient");
  if (rc) return rc;
  const bool dw = dq_weight || dk_weight;
  if (dw) {
    SOLATTN_REQUIRE(workspace && workspace_bytes >= solattn_qk_norm_rope_bwd_workspace_bytes(D), SOLATTN_ESIZE,
                    "%s: workspace %lld < %lld bytes", what, (long long)workspace_bytes,
                    (long long)solattn_qk_norm_rope_bwd_workspace_bytes(D));
    SOLATTN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, SOLATTN_EINVAL,
                    "%s: workspace must be 256-byte aligned", what);
    a.part = static_cast<float*>(workspace);
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const uint32_t n = bwd_blocks(a);
  const dim3 grid(n), block(kRopeThreads);
  const bool wide = D > 64;
  const auto kern = dtype == SOLATTN_BF16   ? (wide ? qk_rope_bwd_kernel<Bf16, 16> : qk_rope_bwd_kernel<Bf16, 8>)
                    : dtype == SOLATTN_FP16 ? (wide ? qk_rope_bwd_kernel<Fp16, 16> : qk_rope_bwd_kernel<Fp16, 8>)
                                            : (wide ? qk_rope_bwd_kernel<Fp32, 16> : qk_rope_bwd_kernel<Fp32, 8>);
  hipLaunchKernelGGL(kern, grid, block, 0, s, a);
  if ((rc = check_launch(what)) || !dw) return rc;
  hipLaunchKernelGGL(qk_rope_dw_kernel, dim3(static_cast<uint32_t>(cdiv(2 * D, 16))), dim3(256), 0, s, a.part,
                     static_cast<int>(n), static_cast<int>(D), dq_weight, dk_weight);
  return check_launch(what);
}
