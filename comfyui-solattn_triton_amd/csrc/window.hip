// Sliding-window attention with sinks: forward and gradients, causal or symmetric,
// kv heads shared by a group of query heads, padded batches (window_common.hpp has
// the rule of what a row sees).
//
//   o_i = sum_j P_ij v_j,  P_ij = exp(scale q_i.k_j - lse_i)
//   D_i = do_i . o_i,  dS = P (do_i . v_j - D_i)
//   dv_j = sum_i P do_i,  dq_i = scale sum_j dS k_j,  dk_j = scale sum_i dS q_i
//
// Bound: the LDS reads of the products' operands beside the products themselves (a
// wave's 32 rows use an operand once, so a CU's reads take nearly as long as its matrix
// instructions: 3770 against 4100 cycles for 64 rows of the dk, dv kernel, 1080 against
// 1020 for the forward's 32 keys), then the exps and the power limit: matrix cores are
// busy 61% of a long forward's cycles, the VALU 45%, either 82%, at 1.6 GHz; 38-42% and
// 36-42% of the gradients'. Short sequences are bound by the latency of a step. 16001 tokens, window 4096, 24 heads of 128 over
// 8: 663-704 us, 1000-1060 TFLOP/s; 12133 tokens, symmetric window 2401, 1333 sinks:
// 724-765 us, 1040-1100 TFLOP/s; 8192 tokens, window 1024, with gradients: 534-574 us
// (forward 133-143, dq 179-196, dk and dv 221-240, join 8); 2000 tokens of 16 heads of
// 64, batch 2, window 512, with gradients: 82-84 us (23, 29, 33, 6).
// Everything between the products stays in registers: S^T = K Q^T puts a row on a lane column, so its
// statistics need one exchange (lanes 32 apart) and P converts in place into the B
// operand of the next product, whose A operand is read transposed from LDS
// (ds_read_b64_tr_b16). P and dS are rounded to the inputs' type (in the
// gradients of short windows twice: the value and what that left) for the matrix
// instruction; row sums add P as rounded, every other sum is fp32.
#include <type_traits>

#include "window_common.hpp"

namespace solattn {
namespace {

constexpr int kRows = 128;            // query rows (or keys) of a workgroup
constexpr int kThreads = 2 * kRows;   // a wave for 32 of them

// Running maximum before any visible key: finite, so that exp2 of a masked score
// stays 0, and below every score that counts.
constexpr float kNoMax = -1e30f;

// Workgroup -> (batch, kv head, block of rows, query head, part): the query heads of
// one kv head and block run side by side. Causal blocks go last first: where the
// window is wide, the last rows have the most keys.
__device__ __forceinline__ void row_item(const WindowArgs& a, int& b, int& h, int& qb, int& part) {
  uint32_t w = xcd_item(a, blockIdx.x, gridDim.x);
  part = a.by_split.split(w);
  const int g = a.by_group.split(w);
  qb = a.by_nqb.split(w);
  if (a.causal) qb = a.nqb - 1 - qb;
  h = a.by_hkv.split(w) * a.group + g;
  b = w;
}

// What the rows of this wave see (rows past Tq repeat the last).
__device__ __forceinline__ RowsKeys wave_keys(const WindowArgs& a, int r0, int len) {
  const int first = r0 + 32 * wave_id();
  return rows_keys(a, a.q_start + min(first, a.Tq - 1), a.q_start + min(first + 31, a.Tq - 1), len);
}

// P and dS of fp16 are rounded as multiples of themselves by powers of two. As they are,
// those of many keys and of small gradients lie among or below fp16's subnormals (8192
// keys: dq and dk 4.5 to 15 times as far from exact values as these are when rounded,
// for do of 1e-2 and 1e-3), and those of large gradients above its largest number.
//   dk, dv: P by 2^kPScale, and dS by what takes a bound of it, max |v_j| max |do_i| +
//     max |D_i| over a wave's keys and the rows that see its block, to 2^14;
//   dq: dS of row i by 2^13 / |do_i|, less where that passes 2^15 in a tile (its sums are
//     then made smaller too, as those of a softmax whose maximum grows).
// The sums are multiplied back in fp32. bf16 has the range and needs none of it. 8192
// tokens, window 1024, with gradients: 565 -> 579 us.
constexpr int kPScale = 12;
template <typename E>
constexpr bool kScaled = std::is_same_v<E, Fp16>;
__device__ __forceinline__ float pow2(int x) { return __uint_as_float(static_cast<uint32_t>(127 + x) << 23); }
__device__ __forceinline__ float finite_or_0(float x) { return fabsf(x) < INFINITY ? x : 0.f; }
// The largest over the 32 lanes of a wave's half.
__device__ __forceinline__ float max32(float x) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}

template <int ND>
struct RowState {
  float m, l;      // running max (log2 domain) and this lane's row sum
  f32x16 acc[ND];  // O^T
};

// One step of the forward's pipeline over half tiles of 32 keys, in one hand-ordered
// stream: S(n+1) = K(n+1) Q^T, O += P(n-1) V(n-1) and the softmax of S(n). Slot i
// issues a score MFMA, two exps and a P.V MFMA; the operands of slot i + 2 are read
// at its top (the empty asm keeps them there). The running max stays as it is unless
// a lane's sum of P passes 255 (no sum above 255: no score more than 8 above it), in
// which case P is made again and O rescaled, behind the products with P(n-1).
template <typename E, int D>
__device__ __forceinline__ void window_step(RowState<D / 32>& st, const f32x16& sc, f32x16& sn, const bf16x8 (&pp)[2],
                                            bf16x8 (&pn)[2], uint32_t kl, uint32_t vl, const bf16x8 (&q)[D / 16],
                                            float c) {
  constexpr int ND = D / 32, NM = D / 16, SLOTS = 8 / NM;
  bf16x8 ka[3], va[3];
  uint32_t pw[2][4];
  float psum = 0.f;
  const float neg = -st.m;
  ka[0] = k_op_x<D>(kl, 0, 0);
  ka[1] = k_op_x<D>(kl, 0, 1);
  va[0] = v_op_x<D>(vl, 0, 0);
  va[1] = v_op_x<D>(vl, 0, 1);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int j = i / SLOTS;
    if (i % SLOTS == 0) {
      if (j + 2 < NM) {
        ka[(j + 2) % 3] = k_op_x<D>(kl, 0, j + 2);
        va[(j + 2) % 3] = v_op_x<D>(vl, (j + 2) / ND, (j + 2) % ND);
        asm volatile("" ::: "memory");
      }
      if (j == 0)
        E::amfma0(sn, ka[0], q[0]);
      else
        E::amfma(sn, ka[j % 3], q[j]);
    }
    pw[i >> 2][i & 3] = E::exp_pair(sc[2 * i], sc[2 * i + 1], c, neg, psum);
    if (i % SLOTS == SLOTS - 1) {
      if (j == 0)
        E::amfma_first(st.acc[0], va[0], pp[0]);
      else if (j == NM - 1)
        E::amfma_tie(st.acc[ND - 1], va[j % 3], pp[1], sn);
      else
        E::amfma(st.acc[j % ND], va[j % 3], pp[j / ND]);
    }
    if (i == 0) __builtin_amdgcn_s_setprio(1);
  }
  __builtin_amdgcn_s_setprio(0);
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)
    pn[ks] = __builtin_bit_cast(bf16x8, make_uint4(pw[ks][0], pw[ks][1], pw[ks][2], pw[ks][3]));
  if (__any(!(psum <= 255.f))) {  // (also infinities and NaN)
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[r]);
    float alpha;
    const float m_new = new_max(st.m, xhalf_max(mx) * c, alpha);
    if (__any(m_new != st.m)) {  // lanes whose max stays make the same P
      st.m = m_new;
      st.l *= alpha;
      psum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) pw[i >> 2][i & 3] = E::exp_pair(sc[2 * i], sc[2 * i + 1], c, -m_new, psum);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        pn[ks] = __builtin_bit_cast(bf16x8, make_uint4(pw[ks][0], pw[ks][1], pw[ks][2], pw[ks][3]));
      mfma_fence(st.acc);  // the rescale reads O
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) st.acc[dt] *= alpha;
    }
  }
  st.l += psum;
}

// The forward. Two half buffers of 32 rows each for K and V: step n copies K(n+2)
// over K(n) and V(n) over V(n-2), so a copy has a whole step to land. (Four half
// buffers, copies two steps further ahead: 757 -> 773 us at 16001 tokens, 130 -> 135 for
// 517 rows of 64 channels. Steps of 64 keys at 64 channels: 77 -> 86 us there.)
template <typename E, int BLK, int D>
__global__ void __launch_bounds__(2 * BLK) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2)))
window_fwd_kernel(const WindowArgs a) {
  constexpr int ND = D / 32, NC = D / 16, NT = 2 * BLK;
  constexpr uint32_t kHalf = kKeys * D;  // bytes of half a tile
  __shared__ __align__(256) uint16_t kbuf[kKeys * D];
  __shared__ __align__(256) uint16_t vbuf[kKeys * D];
  fetch_arguments(a);
  const int lane = threadIdx.x & 63, half = lane >> 5;
  int b, h, qb, part;
  row_item(a, b, h, qb, part);
  const int len = sequence_length(a, b), hk = h / a.group;
  const int r0 = qb * BLK, row = r0 + wave_id() * 32 + (lane & 31), rr = min(row, a.Tq - 1);
  const int p0 = a.q_start + r0, p1 = a.q_start + min(r0 + BLK, a.Tq) - 1;
  const KeyTiles kt = key_tiles(a, p0, p1, len);
  const RowKeys rk = row_keys(a, a.q_start + rr, len);
  const int per = a.by_split.of(kt.n + a.split - 1), tile0 = min(part * per, kt.n);
  const int ntiles = __builtin_amdgcn_readfirstlane(min(per, kt.n - tile0));
  const uint16_t* kp = a.k.p + b * a.k.b + hk * a.k.h;
  const uint16_t* vp = a.v.p + b * a.v.b + hk * a.v.h;
  const uint32_t kb = lds_addr(kbuf), vb = lds_addr(vbuf);
  const uint32_t kl = k_lane<D>(kb, lane & 31, half), vl = v_lane<D>(vb, lane);

  RowState<ND> st;
  st.m = kNoMax;
  st.l = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) st.acc[dt] = f32x16{};

  if (ntiles > 0) {
    CopyOffsets<NT, D> off;
    off.init(a.k.t, a.v.t);
    // Half n of the part's tiles into buffer n & 1.
    const auto issue = [&](int kv, int n) __attribute__((always_inline)) {
      const int t = tile0 + (n >> 1), hh = n & 1, j0 = kt.first(t);
      const uint32_t dst = (kv ? vb : kb) + hh * kHalf;
      const uint16_t* base = kv ? vp : kp;
      const int64_t stride = kv ? a.v.t : a.k.t;
      if (kt.whole(t)) {
        issue_half<NT, D>(dst, base + (j0 + 32 * hh) * stride, stride, kv ? off.v : off.k);
      } else {
        const auto safe = [&](int r) { return kt.safe(j0 + r); };
        if (kv)
          copy_half<NT, D, kTransposed>(dst, hh, base, stride, safe);
        else
          copy_half<NT, D, kByRow>(dst, hh, base, stride, safe);
      }
    };
    const auto land = [&]() __attribute__((always_inline)) {
      wait_tile_copies();
      __syncthreads();
    };
    const RowsKeys wave = wave_keys(a, r0, len);
    const auto mask = [&](f32x16& s, int n) __attribute__((always_inline)) {
      const int j0 = kt.first(tile0 + (n >> 1)) + 32 * (n & 1);
      if (!wave.all(j0, 32)) mask_keys(s, rk, j0, half);
    };
    const int last = 2 * ntiles - 1;

    issue(0, 0);
    issue(0, 1);
    issue(1, 0);
    bf16x8 q[NC];
    load_row<D>(q, a.q.p + b * a.q.b + static_cast<int64_t>(rr) * a.q.t + h * a.q.h, half);
    f32x16 sa, sb;  // scores of even and odd halves
    bf16x8 pa[2], pb[2];
    land();
    // Step 0, without a stream: both halves are scored, the running max is the whole tile's.
    {
      f32x16 s0 = {}, s1 = {};
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) s0 = E::mfma32(k_op_x<D>(kl, 0, cc), q[cc], s0);
      __syncthreads();  // every wave is done with K(0)
      if (last > 1) issue(0, 2);
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) s1 = E::mfma32(k_op_x<D>(kl + kHalf, 0, cc), q[cc], s1);
      mask(s0, 0);
      f32x16 t = s1;
      mask(t, 1);
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fmaxf(s0[r], t[r]));
      st.m = fmaxf(kNoMax, xhalf_max(mx) * a.c);
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = E::exp_pair(s0[2 * i], s0[2 * i + 1], a.c, -st.m, st.l);
      pa[0] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
      pa[1] = __builtin_bit_cast(bf16x8, make_uint4(w[4], w[5], w[6], w[7]));
      sb = t;
    }
    mfma_fence(st.acc);  // O's zeros are in their registers before the asm MFMAs that add to them
    land();
    // (plain: copies and scores of tiles inside the run, at the pointers kn and vn)
    const uint16_t *kn = kp, *vn = vp;
    const int64_t k32 = 32 * a.k.t, v32 = 32 * a.v.t;
    const auto copies = [&](int n, auto plain) __attribute__((always_inline)) {
      if constexpr (decltype(plain)::value) {
        issue_half<NT, D>(kb + (n & 1) * kHalf, kn, a.k.t, off.k);
        issue_half<NT, D>(vb + (n & 1) * kHalf, vn, a.v.t, off.v);
        kn += k32, vn += v32;
      } else {
        if (n + 2 <= last) issue(0, n + 2);
        issue(1, n);
      }
    };
    const auto odd = [&](int n, auto plain) __attribute__((always_inline)) {
      copies(n, plain);
      window_step<E, D>(st, sb, sa, pa, pb, kl, vl, q, a.c);
      land();
    };
    const auto even = [&](int n, auto plain) __attribute__((always_inline)) {
      copies(n, plain);
      if constexpr (!decltype(plain)::value) mask(sa, n);
      window_step<E, D>(st, sa, sb, pb, pa, kl + kHalf, vl + kHalf, q, a.c);
      if constexpr (!decltype(plain)::value) mask(sb, n + 1);
      land();
    };
    // Steps 2 t + 1 and 2 t + 2 work on tiles t to t + 2 of the part. Where these lie in
    // a run of tiles that every row of the block sees whole, among the sinks' or the
    // window's, they need no masks, and their copies are 32 rows apart.
    const int lo = max(p1 - a.window + 1, 0), hi = min(a.causal ? p0 : p0 + a.window - 1, len - 1);
    int run0 = 0, run1 = p1 < len ? min(kt.s_end / kKeys, kt.ns) : 0;
    int t = 0;
#pragma unroll 1
    for (int run = 0; run < 3; ++run) {  // (the last one has no run: what is left)
      run0 = max(min(run0 - tile0, ntiles - 1), 0);
      run1 = min(run1 - tile0, ntiles) - 2;
      for (; t < run0; ++t) {
        odd(2 * t + 1, std::false_type());
        even(2 * t + 2, std::false_type());
      }
      if (t < run1) {
        const int j0 = kt.first(tile0 + t);
        kn = kp + (j0 + 96) * a.k.t;
        vn = vp + (j0 + 32) * a.v.t;
      }
      for (; t < run1; ++t) {
        odd(1, std::true_type());
        even(2, std::true_type());
      }
      run0 = run == 0 ? max(kt.ns, kt.ns + (lo - kt.w0 + kKeys - 1) / kKeys) : kt.n;
      run1 = run == 0 && p1 < len ? kt.ns + (hi + 1 - kt.w0) / kKeys : 0;
    }
    odd(2 * t + 1, std::false_type());
    // P.V of the last half
    mfma_fence(st.acc);
#pragma unroll
    for (int i = 0; i < NC; ++i)
      st.acc[i % ND] = E::mfma32(v_op_x<D>(vl + kHalf, i / ND, i % ND), pb[i / ND], st.acc[i % ND]);
  }

  const float l = xhalf_sum(st.l);
  const bool on = row < a.Tq;
  const int64_t at = (static_cast<int64_t>(b) * a.H + h) * a.Tq + row;
  if (a.split > 1) {
    if (!on) return;
    float* p = a.part + (at * a.split + part) * D + 4 * half;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x16& x = st.acc[dt];
        *reinterpret_cast<float4*>(p + 32 * dt + 8 * i) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
      }
    if (half == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * (at * a.split + part)) = make_float2(st.m, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  store_row<E>(st.acc, inv, a.out + b * a.out_b + static_cast<int64_t>(row) * a.out_t + h * a.out_h, on, half);
  if (a.o_lo) {
    rounded_off<E>(st.acc, inv);
    store_row<E>(st.acc, 1.f, a.o_lo + ((static_cast<int64_t>(b) * a.Tq + row) * a.H + h) * D, on, half);
  }
  if (a.lse && on && half == 0) a.lse[at] = l == 0.f ? INFINITY : st.m + __builtin_amdgcn_logf(l);
}

// The parts of the rows joined, four channels a lane.
template <typename E, int D>
__global__ void __launch_bounds__(256) window_join_kernel(const WindowArgs a) {
  constexpr int L = D / 4;  // lanes of a row
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
  if (at >= static_cast<int64_t>(a.B) * a.H * a.Tq) return;
  const int ch = 4 * (threadIdx.x % L);
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + at * a.split;
  float top = kNoMax, l = 0.f, o[4] = {};
  for (int i = 0; i < a.split; ++i) top = fmaxf(top, ml[i].x);
  const float* p = a.part + at * a.split * D + ch;
#pragma unroll 4
  for (int i = 0; i < a.split; ++i) {
    const float2 u = ml[i];
    const float f = __builtin_amdgcn_exp2f(u.x - top);
    const float4 x = *reinterpret_cast<const float4*>(p + static_cast<int64_t>(i) * D);
    l = fmaf(u.y, f, l);
    o[0] = fmaf(x.x, f, o[0]), o[1] = fmaf(x.y, f, o[1]), o[2] = fmaf(x.z, f, o[2]), o[3] = fmaf(x.w, f, o[3]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int row = static_cast<int>(at % a.Tq);
  const int64_t bh = at / a.Tq;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] *= inv;
  const uint2 w = make_uint2(E::pack(o[0], o[1]), E::pack(o[2], o[3]));
  *reinterpret_cast<uint2*>(a.out + (bh / a.H) * a.out_b + static_cast<int64_t>(row) * a.out_t + (bh % a.H) * a.out_h +
                            ch) = w;
  if (a.o_lo)
    *reinterpret_cast<uint2*>(a.o_lo + ((bh / a.H * a.Tq + row) * a.H + bh % a.H) * D + ch) =
        make_uint2(E::pack(o[0] - E::lo(w.x), o[1] - E::hi(w.x)), E::pack(o[2] - E::lo(w.y), o[3] - E::hi(w.y)));
  if (a.lse && ch == 0) a.lse[at] = l == 0.f ? INFINITY : top + __builtin_amdgcn_logf(l);
}

// The products of a half step of the backward (32 rows by 32 keys), hand-ordered: an
// operand is read AHEAD products before its own (left to itself the compiler reads it
// right in front and waits: the matrix instructions were busy a third of the time). A
// product takes 32 cycles, an LDS read beside those of seven other waves several times
// that. Raised wave priority: the issue arbiter prefers a wave inside its products.
// Two scores from the tiles at x and y, rows by rows: s = X B^T, t = Y C^T.
template <typename E, int D, int AHEAD, typename AX, typename AY>
__device__ __forceinline__ void two_scores(f32x16& s, f32x16& t, const AX& x, uint32_t x_at, const bf16x8 (&b)[D / 16],
                                           const AY& y, uint32_t y_at, const bf16x8 (&c)[D / 16]) {
  constexpr int NC = D / 16, R = AHEAD + 1;
  bf16x8 r[R];
  __builtin_amdgcn_s_setprio(1);
  const auto operand = [&](int i) { return i < NC ? x.by_row(0, i, x_at) : y.by_row(0, i - NC, y_at); };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) r[i] = operand(i);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < 2 * NC; ++i) {
    if (i + AHEAD < 2 * NC) {
      r[(i + AHEAD) % R] = operand(i + AHEAD);
      asm volatile("" ::: "memory");
    }
    if (i == 0)
      E::amfma0(s, r[0], b[0]);
    else if (i < NC)
      E::amfma(s, r[i % R], b[i]);
    else if (i == NC)
      E::amfma0(t, r[i % R], c[0]);
    else
      E::amfma(t, r[i % R], c[i - NC]);
  }
  __builtin_amdgcn_s_setprio(0);
  asm volatile("s_nop 7\n\ts_nop 7" : "+v"(s), "+v"(t));  // readers of s and t come after their wait states
}

// acc += X^T W for the 32 rows at x, read transposed; w: W's packed operands, in one
// rounding or the two of pack_all, which share the reads.
template <typename E, int D, int AHEAD, int NW, typename AX>
__device__ __forceinline__ void add_product(f32x16 (&acc)[D / 32], const AX& x, uint32_t at,
                                            const bf16x8 (&w)[NW][2]) {
  constexpr int ND = D / 32, N = 2 * ND, R = AHEAD + 1;
  bf16x8 r[R];
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) r[i] = x.transposed(i / ND, i % ND, at);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i + AHEAD < N) {
      r[(i + AHEAD) % R] = x.transposed((i + AHEAD) / ND, (i + AHEAD) % ND, at);
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int n = 0; n < NW; ++n) E::amfma_after_valu(acc[i % ND], r[i % R], w[n][i / ND]);
  }
  __builtin_amdgcn_s_setprio(0);
}

// dq, a block of rows at a time as the forward; D_i on the way, for the other kernel.
// (The softmax work between the products of the next half, as the forward has it, with
// four half buffers and a barrier for each: 191 -> 208 us at 8192 tokens.)
template <typename E, int D, int NW>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
window_dq_kernel(const WindowArgs a) {
  constexpr int ND = D / 32, NC = D / 16;
  constexpr uint32_t kBuf = kKeys * D * 2;  // bytes of a tile
  __shared__ __align__(256) uint16_t kbuf[2 * kKeys * D];
  __shared__ __align__(256) uint16_t vbuf[2 * kKeys * D];
  fetch_arguments(a);
  const int lane = threadIdx.x & 63, half = lane >> 5;
  int b, h, qb, part;
  row_item(a, b, h, qb, part);
  const int len = sequence_length(a, b), hk = h / a.group;
  const int r0 = qb * kRows, row = r0 + wave_id() * 32 + (lane & 31), rr = min(row, a.Tq - 1);
  const int p = a.q_start + rr;
  const KeyTiles kt = key_tiles(a, a.q_start + r0, a.q_start + min(r0 + kRows, a.Tq) - 1, len);
  const RowKeys rk = row_keys(a, p, len);
  const uint16_t* kp = a.k.p + b * a.k.b + hk * a.k.h;
  const uint16_t* vp = a.v.p + b * a.v.b + hk * a.v.h;
  const uint32_t kb = lds_addr(kbuf), vb = lds_addr(vbuf);
  TileAddr<D, kBoth> ka(kb, lane);
  TileAddr<D, kByRow> va(vb, lane);
  const uint32_t off_k = copy_offset<kThreads, D, kBoth>(a.k.t), off_v = copy_offset<kThreads, D, kByRow>(a.v.t);
  const auto issue = [&](int t) __attribute__((always_inline)) {
    const int j0 = kt.first(t);
    const uint32_t at = (t & 1) * kBuf;
    if (kt.whole(t)) {
      copy_whole<kThreads, D>(kb + at, kp + j0 * a.k.t, a.k.t, off_k);
      copy_whole<kThreads, D>(vb + at, vp + j0 * a.v.t, a.v.t, off_v);
    } else {
      const auto safe = [&](int r) { return kt.safe(j0 + r); };
      copy_tile<kThreads, D, kBoth>(kb + at, kp, a.k.t, safe);
      copy_tile<kThreads, D, kByRow>(vb + at, vp, a.v.t, safe);
    }
  };
  const RowsKeys wave = wave_keys(a, r0, len);
  if (kt.n) issue(0);
  bf16x8 q[NC], g[NC];
  load_row<D>(q, a.q.p + b * a.q.b + static_cast<int64_t>(rr) * a.q.t + h * a.q.h, half);
  load_row<D>(g, a.d_o.p + b * a.d_o.b + static_cast<int64_t>(rr) * a.d_o.t + h * a.d_o.h, half);
  const int64_t at = (static_cast<int64_t>(b) * a.H + h) * a.Tq + rr;
  // D_i from o and what its rounding took away: the rounding alone is one error for all
  // keys of a row, and took dq and dk from 1.45 to 1.55 times the error of exact ones
  // rounded to the type.
  float delta = 0.f, size = 0.f;  // size: |do_i|^2
  {
    bf16x8 o[NC];
    const auto add = [&](const uint16_t* row_o) __attribute__((always_inline)) {
      load_row<D>(o, row_o, half);
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) {
        const uint4 x = __builtin_bit_cast(uint4, o[cc]), y = __builtin_bit_cast(uint4, g[cc]);
        const uint32_t u[4] = {x.x, x.y, x.z, x.w}, w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) delta = fmaf(E::lo(u[i]), E::lo(w[i]), fmaf(E::hi(u[i]), E::hi(w[i]), delta));
      }
    };
    add(a.o.p + b * a.o.b + static_cast<int64_t>(rr) * a.o.t + h * a.o.h);
    if (a.o_lo) add(a.o_lo + ((static_cast<int64_t>(b) * a.Tq + rr) * a.H + h) * D);
    delta = xhalf_sum(delta);
    if constexpr (kScaled<E>) {
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) {
        const uint4 y = __builtin_bit_cast(uint4, g[cc]);
        const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) size = fmaf(E::lo(w[i]), E::lo(w[i]), fmaf(E::hi(w[i]), E::hi(w[i]), size));
      }
      size = xhalf_sum(size);
    }
  }
  const float lse = a.lse[at];
  float neg = -lse;  // -inf for a row that sees nothing
  if (row < a.Tq && half == 0) a.delta[at] = delta;
  int up = 0;  // dS is held as 2^up of itself
  if constexpr (kScaled<E>) {
    if (row < a.Tq && half == 0) a.lse_p[at] = lse - kPScale;
    const bool on = row < a.Tq && lse < INFINITY;
    const float big = max32(on ? sqrtf(finite_or_0(size)) : 0.f), big_d = max32(on ? fabsf(finite_or_0(delta)) : 0.f);
    if (lane == 0) a.mag[(static_cast<int64_t>(b) * a.H + h) * (4 * a.nqb) + 4 * qb + wave_id()] = make_float2(big, big_d);
    up = 13 - ((__builtin_amdgcn_frexp_expf(size) + 1) >> 1);
    neg += static_cast<float>(up);
  }

  f32x16 acc[ND] = {};
  for (int t = 0; t < kt.n; ++t) {
    const int j0 = kt.first(t);
    wait_tile_copies();
    __syncthreads();  // this tile is in, and every wave is done with the buffers of the last
    if (t + 1 < kt.n) issue(t + 1);
    if (wave.none(j0, kKeys)) continue;
    const bool masked = !wave.all(j0, kKeys);
#pragma unroll
    for (int m2 = 0; m2 < 2; ++m2) {
      ka.remade();
      va.remade();
      const uint32_t at = (t & 1) * kBuf + m2 * (64 * D);
      f32x16 s, dp;
      two_scores<E, D, D == 64 ? 6 : 4>(s, dp, ka, at, q, va, at, g);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float pr = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, neg));
        dp[r] = pr * (dp[r] - delta);
      }
      if (masked) {  // (what the row does not see may be anything up to here)
        const uint32_t bits = key_bits(rk, j0 + 32 * m2, half);
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = keep(dp[r], bit_word(bits, r));
      }
      if constexpr (kScaled<E>) {
        float top = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(dp[r]));
        if (__any(top > 32768.f)) {
          top = xhalf_max(top);
          const int down = top > 32768.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 13 : 0;
          const float f = __builtin_amdgcn_ldexpf(1.f, -down);
          up -= down;
          neg -= static_cast<float>(down);
          mfma_fence(acc);
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) acc[dt] *= f;
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] *= f;
        }
      }
      bf16x8 ds[NW][2];
      pack_all<E>(ds, dp);
      add_product<E, D, 3>(acc, ka, at, ds);
    }
  }
  mfma_fence(acc);
  store_row<E>(acc, kScaled<E> ? __builtin_amdgcn_ldexpf(a.scale, -up) : a.scale,
               a.out + b * a.out_b + static_cast<int64_t>(row) * a.out_t + h * a.out_h, row < a.Tq, half);
}

// dk and dv: a workgroup owns 128 keys of a kv head and walks, head by head of the
// group, the tiles of 64 rows that see any of them; a wave's 32 keys (k, v and the
// sums) stay in registers: S = Q K^T and dP = dO V^T put a key on a lane column, and
// P and dS convert in place into B operands of dv^T += dO^T P and dk^T += Q^T dS.
// Q and dO tiles are double buffered: the next one lands while this one is used.
//
// Parts: the steps (heads x tiles) of a block of keys are cut into parts of their
// own workgroups, sinks' blocks into `ks` and the others into `kn`: every row sees
// the sinks, and few or short heads leave CUs without a block. A part's sums go to
// the workspace in fp32 and window_dkv_join_kernel adds them up in order; a block
// of one part is stored straight.
template <typename E, int D, int NW>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
window_dkv_kernel(const WindowArgs a) {
  constexpr int ND = D / 32, NC = D / 16;
  constexpr int kAhead = D == 64 ? 3 : NW == 1 ? 2 : 1;  // (what the registers leave: one more at 128 channels spills)
  constexpr uint32_t kBuf = kKeys * D * 2;  // bytes of a tile
  __shared__ __align__(256) uint16_t qbuf[2 * kKeys * D];
  __shared__ __align__(256) uint16_t gbuf[2 * kKeys * D];
  __shared__ __align__(16) float stat[2][2][kKeys];  // [buffer][lse, delta]
  fetch_arguments(a);
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = wave_id();
  uint32_t w = xcd_item(a, blockIdx.x, gridDim.x);
  const KeyPart kp = key_part(a, w);
  uint32_t bh = kp.bh;
  const int hk = a.by_hkv.split(bh), b = bh;
  const int len = sequence_length(a, b);
  const int j0 = kp.block * kRows, j = j0 + wave * 32 + (lane & 31), jj = min(j, a.Tk - 1);
  // (the lane asked for again where it is needed: at 128 channels no register is left to
  // hold it or what follows from it through the loop)
  const auto lane_again = []() __attribute__((always_inline)) {
    int ln = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(ln));
    return ln;
  };
  // rows that see a key of the block: a key's interval moves up with it, but that a sink's has no end
  const int jlast = min(min(j0 + kRows, a.Tk), len) - 1;
  const KeyRows k0 = key_rows(a, j0, len), k1 = key_rows(a, max(jlast, j0), len);
  const int i0 = k0.pl - a.q_start, i1 = (j0 < a.sinks ? k0.ph : k1.ph) - a.q_start;  // rows [i0, i1]
  const int tile0 = i0 & ~(kKeys - 1);
  const int tiles = j0 < len && i0 <= i1 ? (i1 - tile0) / kKeys + 1 : 0;
  const int per = (kp.block < a.nsb ? a.by_ks : a.by_kn).of(tiles * a.group + kp.parts - 1);
  const int s0 = min(kp.part * per, tiles * a.group), s1 = min(s0 + per, tiles * a.group);
  // rows that see every key of the wave, and those that see any (a step without is skipped)
  const KeysRows kw = keys_rows(a, j0 + wave * 32, j0 + wave * 32 + 31, len);
  const int all_lo = kw.all_lo - a.q_start, all_hi = kw.all_hi - a.q_start;
  const int any_lo = kw.any_lo - a.q_start, any_hi = kw.any_hi - a.q_start;

  const uint32_t qb = lds_addr(qbuf), gb = lds_addr(gbuf), sb = lds_addr(stat);
  TileAddr<D, kBoth> qa(qb, lane);  // (dO's tiles: the same, at to_g)
  const uint32_t to_g = gb - qb;
  bf16x8 k[NC], v[NC];
  load_row<D>(k, a.k.p + b * a.k.b + static_cast<int64_t>(jj) * a.k.t + hk * a.k.h, half);
  load_row<D>(v, a.v.p + b * a.v.b + static_cast<int64_t>(jj) * a.v.t + hk * a.v.h, half);
  int down = 0;  // |dS| < 2^down
  if constexpr (kScaled<E>) {
    if (tiles) {
      float size = 0.f;
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) {
        const uint4 y = __builtin_bit_cast(uint4, v[cc]);
        const uint32_t x[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) size = fmaf(E::lo(x[i]), E::lo(x[i]), fmaf(E::hi(x[i]), E::hi(x[i]), size));
      }
      const KeyRows kr = key_rows(a, j, len);
      size = max32(kr.pl <= kr.ph ? finite_or_0(xhalf_sum(size)) : 0.f);
      float big = 0.f, big_d = 0.f;
      const uint32_t c0 = static_cast<uint32_t>(i0) >> 5, cells = (static_cast<uint32_t>(i1) >> 5) - c0 + 1;
      const float2* mag = a.mag + (static_cast<int64_t>(b) * a.H + hk * a.group) * (4 * a.nqb) + c0;
      for (int g = 0; g < a.group; ++g, mag += 4 * a.nqb)
        for (uint32_t c = lane; c < cells; c += 64) {
          big = fmaxf(big, mag[c].x);
          big_d = fmaxf(big_d, mag[c].y);
        }
      big = xhalf_max(max32(big)), big_d = xhalf_max(max32(big_d));
      down = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(fmaf(sqrtf(size), big, big_d)));
    }
  }
  const float to_ds = pow2(2 - down);

  const uint32_t off_q = copy_offset<kThreads, D, kBoth>(a.q.t), off_g = copy_offset<kThreads, D, kBoth>(a.d_o.t);
  // The next step to copy: head g of the group, rows from t0 on.
  int g = tiles ? static_cast<uint32_t>(s0) / static_cast<uint32_t>(tiles) : 0, t0 = tiles ? tile0 + (s0 - g * tiles) * kKeys : 0;
  const auto issue = [&](int buf) __attribute__((always_inline)) {
    const int h = hk * a.group + g;
    const uint16_t* qp = a.q.p + b * a.q.b + h * a.q.h;
    const uint16_t* gp = a.d_o.p + b * a.d_o.b + h * a.d_o.h;
    const auto safe = [&](int r) { return min(max(t0 + r, i0), i1); };
    if (t0 >= i0 && t0 + kKeys - 1 <= i1) {
      copy_whole<kThreads, D>(qb + buf * kBuf, qp + t0 * a.q.t, a.q.t, off_q);
      copy_whole<kThreads, D>(gb + buf * kBuf, gp + t0 * a.d_o.t, a.d_o.t, off_g);
    } else {
      copy_tile<kThreads, D, kBoth>(qb + buf * kBuf, qp, a.q.t, safe);
      copy_tile<kThreads, D, kBoth>(gb + buf * kBuf, gp, a.d_o.t, safe);
    }
    const float* st = wave ? a.delta : kScaled<E> ? a.lse_p : a.lse;
    if (wave < 2)
      g2l4(st + (static_cast<int64_t>(b) * a.H + h) * a.Tq + safe(lane), sb + (2 * buf + wave) * kKeys * 4);
    t0 += kKeys;
    if (t0 >= tile0 + tiles * kKeys) t0 = tile0, ++g;
  };

  f32x16 dk[ND] = {}, dv[ND] = {};
  if (s0 < s1) issue(0);
  for (int st = s0; st < s1; ++st) {
    const int buf = (st - s0) & 1;
    // the rows of this step (the copy that was issued last)
    const int r0 = t0 == tile0 ? tile0 + (tiles - 1) * kKeys : t0 - kKeys;
    wait_tile_copies();
    __syncthreads();  // this step's tiles are in, and every wave is done with the buffers of the last
    if (st + 1 < s1) issue(buf ^ 1);
    if (r0 > any_hi || r0 + kKeys - 1 < any_lo) continue;
    const bool masked = r0 < all_lo || r0 + kKeys - 1 > all_hi;
#pragma unroll
    for (int m2 = 0; m2 < 2; ++m2) {
      const uint32_t at = buf * kBuf + m2 * (64 * D);
      qa.remade();
      f32x16 s, dp;
      two_scores<E, D, kAhead>(s, dp, qa, at, k, qa, at + to_g, v);
      const float* lse = stat[buf][0] + 32 * m2 + 4 * half;
      const float* delta = stat[buf][1] + 32 * m2 + 4 * half;
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const float4 l4 = *reinterpret_cast<const float4*>(lse + 8 * r4);
        const float4 d4 = *reinterpret_cast<const float4*>(delta + 8 * r4);
        const float lx[4] = {l4.x, l4.y, l4.z, l4.w}, dx[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * r4 + i;
          s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lx[i]));
          dp[r] = s[r] * (kScaled<E> ? (dp[r] - dx[i]) * to_ds : dp[r] - dx[i]);
        }
        asm volatile("" ::: "memory");  // (the next four's statistics are read behind these, not held with them)
      }
      if (masked) {  // (what a key does not see may be anything up to here)
        const int ln = lane_again();  // (a key past the last is past the sequence)
        const uint32_t bits = row_bits(key_rows(a, j0 + wave * 32 + (ln & 31), len), a.q_start + r0 + 32 * m2, ln >> 5);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const uint32_t w = bit_word(bits, r);
          s[r] = keep(s[r], w);
          dp[r] = keep(dp[r], w);
        }
      }
      bf16x8 pb[NW][2], ds[NW][2];
      pack_all<E>(pb, s);
      if constexpr (NW == 1) pack_all<E>(ds, dp);
      add_product<E, D, kAhead>(dv, qa, at + to_g, pb);
      if constexpr (NW == 2) pack_all<E>(ds, dp);  // (not held through the other product)
      add_product<E, D, kAhead>(dk, qa, at, ds);
    }
  }
  mfma_fence(dk);
  mfma_fence(dv);
  const int ln = lane_again(), hf = ln >> 5;
  const int key = wave * 32 + (ln & 31);
  const float from_p = kScaled<E> ? pow2(-kPScale) : 1.f, from_ds = kScaled<E> ? pow2(down - 2 - kPScale) : 1.f;
  if (kp.parts == 1) {
    const int64_t at = j0 + key;
    const bool on = at < a.Tk;
    store_row<E>(dk, a.scale * from_ds, a.dk + b * a.dk_b + at * a.dk_t + hk * a.dk_h, on, hf);
    store_row<E>(dv, from_p, a.dv + b * a.dv_b + at * a.dv_t + hk * a.dv_h, on, hf);
    return;
  }
  // [dk, dv][key][channel]: a lane has 4 consecutive channels of its key at a time
  float* part = a.part + static_cast<int64_t>(kp.slot) * (2 * kRows * D) + key * D + 4 * hf;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x16 x = dk[dt] * from_ds, y = dv[dt] * from_p;
      *reinterpret_cast<float4*>(part + 32 * dt + 8 * i) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
      *reinterpret_cast<float4*>(part + kRows * D + 32 * dt + 8 * i) =
          make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
    }
}

// The parts of the cut blocks added up: a thread has 8 channels of a key, dk or dv.
template <typename E, int D>
__global__ void __launch_bounds__(256) window_dkv_join_kernel(const WindowArgs a, int blocks) {
  constexpr int C = D / 8;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int ch = static_cast<int>(e % C) * 8, key = static_cast<int>(e / C % kRows);
  const int which = static_cast<int>(e / (C * kRows) & 1);
  const int64_t bk = e / (C * kRows * 2);
  const int bh = static_cast<int>(bk / blocks), block = static_cast<int>(bk % blocks);
  const int j = block * kRows + key;
  if (bh >= a.B * a.Hkv || j >= a.Tk) return;
  const bool sink = block < a.nsb;
  const int parts = sink ? a.ks : a.kn;
  const int64_t slot = static_cast<int64_t>(bh) * a.slots + (sink ? block * a.ks : a.nsb * a.ks + (block - a.nsb) * a.kn);
  const float* p = a.part + (slot * 2 + which) * (kRows * D) + key * D + ch;
  float x[8] = {};
#pragma unroll 8
  for (int i = 0; i < parts; ++i) {
    const float4 u = reinterpret_cast<const float4*>(p)[0], v = reinterpret_cast<const float4*>(p)[1];
    x[0] += u.x, x[1] += u.y, x[2] += u.z, x[3] += u.w, x[4] += v.x, x[5] += v.y, x[6] += v.z, x[7] += v.w;
    p += 2 * kRows * D;
  }
  const int b = bh / a.Hkv, hk = bh % a.Hkv;
  uint16_t* out = which ? a.dv + b * a.dv_b + static_cast<int64_t>(j) * a.dv_t + hk * a.dv_h
                        : a.dk + b * a.dk_b + static_cast<int64_t>(j) * a.dk_t + hk * a.dk_h;
  if (!which)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= a.scale;
  Row8<E>::store(out + ch, x);
}

// How the key blocks of the backward are cut (WindowArgs::nsb, ks, kn, slots): every
// block into as many parts as leave the launch within the CUs' two workgroups each (one
// more, and the last wait for a second round: 6000 tokens of 8 heads, backward: 183 us as
// it is, 209 with one more), as long as a part keeps eight steps; the sinks' blocks, which
// every row behind them sees, into parts no longer than another block, but no more than
// 1024 of them, four a CU (a part writes its keys' dk and dv in fp32: 12133 tokens of 24
// heads, window 64, 1333 sinks in 792 parts 1190 us, in 10296 parts of 1.35 GB 1610), and
// where there are several such blocks also of eight steps at least.
void cut_keys(WindowArgs& a) {
  const int64_t tiles_all = cdiv(a.Tq, kKeys) + 1;
  int64_t tiles = cdiv(static_cast<int64_t>(a.causal ? a.window : 2 * static_cast<int64_t>(a.window)) + kRows, kKeys) + 1;
  if (tiles > tiles_all) tiles = tiles_all;
  const int64_t steps = tiles * a.group, heads = static_cast<int64_t>(a.B) * a.Hkv;
  a.nsb = static_cast<int>(cdiv(a.sinks, kRows));
  int64_t kn = 512 / (heads * a.nkb);
  if (kn > steps / 8) kn = steps / 8;
  if (kn < 1) kn = 1;
  // (a block with few sinks keeps one wave busy: its parts are last and a quarter as long,
  // unless there are many of them)
  const int64_t whole = cdiv(tiles_all * a.group, cdiv(steps, kn));
  const int64_t items = heads * a.nsb * whole;
  const int64_t finer = items > 256 ? 1 : items > 128 ? 2 : 4;
  int64_t ks = whole > 1 ? cdiv(tiles_all * a.group, cdiv(steps, finer * kn)) : whole;
  if (a.nsb > 0 && ks > 1024 / (heads * a.nsb)) ks = 1024 / (heads * a.nsb);
  if (a.nsb > 1 && ks > tiles_all * a.group / 8) ks = tiles_all * a.group / 8;
  if (ks < 1) ks = 1;
  a.kn = static_cast<int>(kn);
  a.ks = static_cast<int>(ks);
  if (a.nsb == a.nkb) a.kn = a.ks;  // (only sinks' blocks)
  // (kn above 1 leaves ks above 1: then heads nkb <= 256 and steps >= 16. So the slots are
  // those of both kinds of blocks or of the sinks' alone)
  a.by_ks = divisor(a.ks), a.by_kn = divisor(a.kn);
  a.by_items = divisor(static_cast<int64_t>(a.nsb) * a.ks + static_cast<int64_t>(a.nkb - a.nsb) * a.kn);
  a.slots = (a.ks > 1 ? a.nsb * a.ks : 0) + (a.kn > 1 ? (a.nkb - a.nsb) * a.kn : 0);
}

int check_mat(const Mat& m, const char* what, const char* name) {
  // (a copy's lane offsets are 32-bit bytes)
  SOLATTN_REQUIRE(m.t >= 0 && m.t < (1ll << 24), SOLATTN_EUNSUPPORTED, "%s: %s token stride %lld beyond 2^24 elements",
                  what, name, (long long)m.t);
  SOLATTN_REQUIRE(m.p, SOLATTN_EINVAL, "%s: null %s", what, name);
  SOLATTN_REQUIRE(reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.b % 8 == 0 && m.t % 8 == 0 && m.h % 8 == 0,
                  SOLATTN_EINVAL, "%s: %s must be 16-byte aligned with strides multiple of 8", what, name);
  return 0;
}

int setup(WindowArgs& a, int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hkv, int64_t D, int dtype,
          int64_t q_start, int64_t window, int64_t sinks, int causal, float scale, const char* what) {
  SOLATTN_REQUIRE(dtype == SOLATTN_BF16 || dtype == SOLATTN_FP16, SOLATTN_EINVAL, "%s: dtype %d", what, dtype);
  SOLATTN_REQUIRE(B > 0 && Tq > 0 && Tk > 0 && H > 0 && Hkv > 0 && H % Hkv == 0, SOLATTN_EINVAL,
                  "%s: bad sizes (%lld query heads over %lld kv heads)", what, (long long)H, (long long)Hkv);
  SOLATTN_REQUIRE(B < (1ll << 31) && H < (1ll << 31) && B * H < (1ll << 31), SOLATTN_EUNSUPPORTED, "%s: grid too large",
                  what);  // (nothing below passes 64 bits)
  SOLATTN_REQUIRE(D == 64 || D == 128, SOLATTN_EUNSUPPORTED, "%s: head_dim %lld not in {64, 128}", what, (long long)D);
  SOLATTN_REQUIRE(Tk < (1ll << 29), SOLATTN_EUNSUPPORTED, "%s: %lld keys", what, (long long)Tk);
  SOLATTN_REQUIRE(Tq <= Tk && q_start >= 0 && q_start <= Tk - Tq, SOLATTN_EINVAL, "%s: rows %lld + %lld past %lld keys", what,
                  (long long)q_start, (long long)Tq, (long long)Tk);
  SOLATTN_REQUIRE(window > 0 && sinks >= 0, SOLATTN_EINVAL, "%s: window %lld, sinks %lld", what, (long long)window,
                  (long long)sinks);
  SOLATTN_REQUIRE(scale > 0.f, SOLATTN_EINVAL, "%s: scale %g", what, static_cast<double>(scale));
  a.B = static_cast<int>(B), a.H = static_cast<int>(H), a.Hkv = static_cast<int>(Hkv);
  a.group = static_cast<int>(H / Hkv);
  a.Tq = static_cast<int>(Tq), a.Tk = static_cast<int>(Tk), a.q_start = static_cast<int>(q_start);
  // wider than the sequence is the same as wide as it
  a.window = static_cast<int>(window < Tk ? window : Tk), a.sinks = static_cast<int>(sinks < Tk ? sinks : Tk);
  // and sinks that reach every key, alone or (causal) with the window, are no window
  if (a.window == Tk || a.sinks == Tk || (causal && static_cast<int64_t>(a.window) + a.sinks >= Tk))
    a.window = static_cast<int>(Tk), a.sinks = 0;
  a.causal = causal;
  a.nqb = static_cast<int>(cdiv(Tq, kRows)), a.nkb = static_cast<int>(cdiv(Tk, kRows));
  a.split = 1;
  a.c = scale * kLog2e, a.scale = scale;
  a.by_split = divisor(1), a.by_group = divisor(a.group), a.by_nqb = divisor(a.nqb), a.by_hkv = divisor(Hkv);
  SOLATTN_REQUIRE(B * H * a.nqb < (1ll << 31) && B * Hkv * a.nkb < (1ll << 31), SOLATTN_EUNSUPPORTED,
                  "%s: grid too large", what);
  return 0;
}

}  // namespace
}  // namespace solattn

using namespace solattn;

// One causal row per sequence: the kernel of single tokens, which splits the keys.
static bool single_token(int64_t Tq, int causal, const float* lse) { return Tq == 1 && causal && !lse; }

// Rows of a workgroup and parts of their keys. 128 rows share the copies of a tile
// among four waves (16000 tokens: 668 us against 710 with 64 rows). Launches that would
// not give every CU four such workgroups take 64 rows, which leave fewer CUs idle at
// the end (3900 tokens of 32 heads, 992 workgroups: 173 -> 132 us; 1128 of them: 199
// against 211). Their key tiles are cut into as many parts, of at least eight tiles and
// joined by a second launch, as leave the launch within four workgroups a CU (256 rows
// of 24 heads against 32000 keys: ten parts 113 us, eleven, which take a second round,
// 143). Padded batches too: within eight, short and empty sequences leave more of the CUs
// to the others, but whole ones share less of their keys in the L2 (517 rows against 16000
// keys, two sequences, one of them past its end: 46.6 us against 53.6, neither: 70.5
// against 62; 128 rows of eight sequences of 32000 keys 206 against 139, half of these
// past their end 101 against 95; prompts of 2000 that no launch needs to cut 86 against 55).
static int cut_rows(WindowArgs& a) {
  const int64_t bh = static_cast<int64_t>(a.B) * a.H;
  const int blk = bh * cdiv(a.Tq, 128) >= 1024 ? 128 : 64;
  a.nqb = static_cast<int>(cdiv(a.Tq, blk));
  const int64_t reach = static_cast<int64_t>(a.causal ? a.window : 2 * static_cast<int64_t>(a.window)) + blk + a.sinks;
  const int64_t keys = a.causal ? a.q_start + a.Tq : a.Tk;  // (none behind the last row)
  const int64_t tiles = cdiv(reach < keys ? reach : keys, kKeys);
  int64_t n = 1024 / (bh * a.nqb);
  if (n > tiles / 8) n = tiles / 8;
  a.split = static_cast<int>(n < 1 ? 1 : n > 64 ? 64 : n);
  a.by_split = divisor(a.split), a.by_nqb = divisor(a.nqb);
  return blk;
}

static int64_t fwd_workspace(const WindowArgs& a, int64_t D) {
  return a.split > 1 ? static_cast<int64_t>(a.B) * a.H * a.Tq * a.split * (D + 2) * 4 : 0;
}

extern "C" int64_t solattn_window_attn_workspace_bytes(int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hkv,
                                                       int64_t D, int64_t q_start, int64_t window, int64_t sinks,
                                                       int causal, int with_lse) {
  clear_error();
  if (Tq == 1 && causal && !with_lse)
    return q_start < 0 || q_start >= Tk ? 0 : paged_attn_workspace(B, H, Hkv, D, q_start + 1, window, sinks);
  WindowArgs a{};
  if (setup(a, B, Tq, Tk, H, Hkv, D, SOLATTN_BF16, q_start, window, sinks, causal, 1.f, "window_attn")) return 0;
  cut_rows(a);
  return fwd_workspace(a, D);
}

extern "C" int solattn_window_attn(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const uint16_t* k,
                                   int64_t sk_b, int64_t sk_t, int64_t sk_h, const uint16_t* v, int64_t sv_b,
                                   int64_t sv_t, int64_t sv_h, int64_t B, int64_t Tq, int64_t Tk, int64_t H,
                                   int64_t Hkv, int64_t D, int dtype, int64_t q_start, const int32_t* lengths,
                                   int64_t window, int64_t sinks, int causal, float scale, uint16_t* o, int64_t so_b,
                                   int64_t so_t, int64_t so_h, float* lse, uint16_t* o_lo, void* workspace,
                                   int64_t workspace_bytes, solattn_stream_t stream) {
  clear_error();
  const char* what = "window_attn";
  if (single_token(Tq, causal, lse)) {
    SOLATTN_REQUIRE(window > 0 && q_start >= 0 && q_start < Tk, SOLATTN_EINVAL, "%s: row %lld of %lld keys, window %lld",
                    what, (long long)q_start, (long long)Tk, (long long)window);
    if (window > Tk) window = Tk;
    if (sinks > Tk) sinks = Tk;
    return paged_attn(q, sq_b, sq_h, k, sk_b, sk_t, sk_h, v, sv_b, sv_t, sv_h, B, q_start + 1, nullptr, 0, 1, lengths,
                      q_start + 1, B, H, Hkv, D, dtype, window, sinks, scale, workspace, workspace_bytes, o, so_b, so_h,
                      reinterpret_cast<hipStream_t>(stream), what);
  }
  WindowArgs a{};
  a.q = {q, sq_b, sq_t, sq_h}, a.k = {k, sk_b, sk_t, sk_h}, a.v = {v, sv_b, sv_t, sv_h};
  a.out = o, a.out_b = so_b, a.out_t = so_t, a.out_h = so_h;
  a.lse = lse, a.o_lo = o_lo, a.lengths = lengths;
  int rc = setup(a, B, Tq, Tk, H, Hkv, D, dtype, q_start, window, sinks, causal, scale, what);
  if (!rc) rc = check_mat(a.q, what, "q");
  if (!rc) rc = check_mat(a.k, what, "k");
  if (!rc) rc = check_mat(a.v, what, "v");
  if (!rc) rc = check_mat({o, so_b, so_t, so_h}, what, "o");
  if (rc) return rc;
  SOLATTN_REQUIRE(reinterpret_cast<uintptr_t>(o_lo) % 16 == 0, SOLATTN_EINVAL, "%s: o_lo must be 16-byte aligned", what);
  const bool bf = dtype == SOLATTN_BF16;
  const int blk = cut_rows(a);
  const int64_t need = fwd_workspace(a, D);
  SOLATTN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), SOLATTN_ESIZE, "%s: workspace %lld < %lld bytes",
                  what, (long long)workspace_bytes, (long long)need);
  SOLATTN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, SOLATTN_EINVAL,
                  "%s: workspace must be 256-byte aligned", what);
  const int64_t rows = B * H * Tq;
  SOLATTN_REQUIRE(rows < (1ll << 31) && B * H * a.nqb * a.split < (1ll << 31), SOLATTN_EUNSUPPORTED,
                  "%s: grid too large", what);
  a.part = static_cast<float*>(workspace);
  a.part_ml = a.part + rows * a.split * D;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const auto k128 = D == 128 ? (bf ? window_fwd_kernel<Bf16, 128, 128> : window_fwd_kernel<Fp16, 128, 128>)
                             : (bf ? window_fwd_kernel<Bf16, 128, 64> : window_fwd_kernel<Fp16, 128, 64>);
  const auto k64 = D == 128 ? (bf ? window_fwd_kernel<Bf16, 64, 128> : window_fwd_kernel<Fp16, 64, 128>)
                            : (bf ? window_fwd_kernel<Bf16, 64, 64> : window_fwd_kernel<Fp16, 64, 64>);
  hipLaunchKernelGGL(blk == 128 ? k128 : k64, dim3(static_cast<uint32_t>(B * H * a.nqb * a.split)),
                     dim3(static_cast<uint32_t>(2 * blk)), 0, s, a);
  if ((rc = check_launch(what)) || a.split == 1) return rc;
  const auto kj = D == 128 ? (bf ? window_join_kernel<Bf16, 128> : window_join_kernel<Fp16, 128>)
                           : (bf ? window_join_kernel<Bf16, 64> : window_join_kernel<Fp16, 64>);
  hipLaunchKernelGGL(kj, dim3(static_cast<uint32_t>(cdiv(rows, 1024 / D))), dim3(256), 0, s, a);
  return check_launch(what);
}

// D_i and lse_p, the 32-row blocks' magnitudes, the parts of dk and dv.
static int64_t stat_bytes(const WindowArgs& a) { return cdiv(static_cast<int64_t>(a.B) * a.H * a.Tq * 4, 256) * 256; }
static int64_t mag_bytes(const WindowArgs& a) { return cdiv(static_cast<int64_t>(a.B) * a.H * a.nqb * 32, 256) * 256; }
static int64_t bwd_workspace(const WindowArgs& a, int64_t D) {
  return 2 * stat_bytes(a) + mag_bytes(a) + static_cast<int64_t>(a.B) * a.Hkv * a.slots * 2 * kRows * D * 4;
}

extern "C" int64_t solattn_window_attn_bwd_workspace_bytes(int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hkv,
                                                           int64_t D, int64_t window, int64_t sinks, int causal) {
  clear_error();
  WindowArgs a{};
  if (setup(a, B, Tq, Tk, H, Hkv, D, SOLATTN_BF16, Tk - Tq, window, sinks, causal, 1.f, "window_attn_bwd")) return 0;
  cut_keys(a);
  return bwd_workspace(a, D);
}

extern "C" int solattn_window_attn_bwd(
    const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const uint16_t* k, int64_t sk_b, int64_t sk_t,
    int64_t sk_h, const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h, const uint16_t* o, int64_t so_b,
    int64_t so_t, int64_t so_h, const uint16_t* d_o, int64_t sg_b, int64_t sg_t, int64_t sg_h, const float* lse,
    const uint16_t* o_lo, int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hkv, int64_t D, int dtype, int64_t q_start,
    const int32_t* lengths, int64_t window, int64_t sinks, int causal, float scale, uint16_t* dq, int64_t sdq_b,
    int64_t sdq_t, int64_t sdq_h, uint16_t* dk, int64_t sdk_b, int64_t sdk_t, int64_t sdk_h, uint16_t* dv,
    int64_t sdv_b, int64_t sdv_t, int64_t sdv_h, void* workspace, int64_t workspace_bytes, solattn_stream_t stream) {
  clear_error();
  const char* what = "window_attn_bwd";
  WindowArgs a{};
  a.q = {q, sq_b, sq_t, sq_h}, a.k = {k, sk_b, sk_t, sk_h}, a.v = {v, sv_b, sv_t, sv_h};
  a.o = {o, so_b, so_t, so_h}, a.d_o = {d_o, sg_b, sg_t, sg_h};
  a.out = dq, a.out_b = sdq_b, a.out_t = sdq_t, a.out_h = sdq_h;
  a.dk = dk, a.dk_b = sdk_b, a.dk_t = sdk_t, a.dk_h = sdk_h;
  a.dv = dv, a.dv_b = sdv_b, a.dv_t = sdv_t, a.dv_h = sdv_h;
  a.lse = const_cast<float*>(lse), a.o_lo = const_cast<uint16_t*>(o_lo), a.lengths = lengths;
  int rc = setup(a, B, Tq, Tk, H, Hkv, D, dtype, q_start, window, sinks, causal, scale, what);
  const Mat outs[3] = {{dq, sdq_b, sdq_t, sdq_h}, {dk, sdk_b, sdk_t, sdk_h}, {dv, sdv_b, sdv_t, sdv_h}};
  const Mat* mats[8] = {&a.q, &a.k, &a.v, &a.o, &a.d_o, &outs[0], &outs[1], &outs[2]};
  const char* names[8] = {"q", "k", "v", "o", "do", "dq", "dk", "dv"};
  for (int i = 0; i < 8 && !rc; ++i) rc = check_mat(*mats[i], what, names[i]);
  if (rc) return rc;
  SOLATTN_REQUIRE(lse && reinterpret_cast<uintptr_t>(o_lo) % 16 == 0, SOLATTN_EINVAL, "%s: null lse or unaligned o_lo",
                  what);
  cut_keys(a);
  const int64_t need = bwd_workspace(a, D);
  SOLATTN_REQUIRE(workspace && workspace_bytes >= need, SOLATTN_ESIZE, "%s: workspace %lld < %lld bytes", what,
                  (long long)workspace_bytes, (long long)need);
  SOLATTN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, SOLATTN_EINVAL,
                  "%s: workspace must be 256-byte aligned", what);
  a.delta = static_cast<float*>(workspace);
  a.lse_p = a.delta + stat_bytes(a) / 4;
  a.mag = reinterpret_cast<float2*>(a.lse_p + stat_bytes(a) / 4);
  a.part = reinterpret_cast<float*>(a.mag) + mag_bytes(a) / 4;
  const int64_t items = B * Hkv * (static_cast<int64_t>(a.nsb) * a.ks + static_cast<int64_t>(a.nkb - a.nsb) * a.kn);
  const int64_t cut = a.kn > 1 ? a.nkb : a.ks > 1 ? a.nsb : 0;  // blocks of keys to join
  const int64_t join = cdiv(B * Hkv * cut * 2 * kRows * (D / 8), 256);
  SOLATTN_REQUIRE(items < (1ll << 31) && join < (1ll << 31), SOLATTN_EUNSUPPORTED, "%s: grid too large", what);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool bf = dtype == SOLATTN_BF16;
  // P and dS in two roundings where rows see few keys or few rows see a key: the fewer, the
  // more of dq and dk cancels, but not of the errors of one rounding (these took dq to
  // 1.45 to 1.65 times the error of exact values rounded once, two to 1.02 to 1.2). From
  // windows of 512 keys, 1024 keys and 128 rows on it is 1.42 to 1.49 in one, and two
  // would take 8192 tokens 540 -> 607 us, 2000 of 64 channels 83 -> 93: where the line
  // is drawn is a choice between the two, the errors do not jump there. The rule is on
  // what the call as a whole can see, up to its last position; what `lengths` hold and the
  // first rows of a long causal call are not looked at.
  const int64_t reach = causal ? q_start + Tq : Tk;
  const int64_t wide = (causal ? a.window : 2 * static_cast<int64_t>(a.window) - 1) + a.sinks;
  const bool two = wide < 512 || reach < 1024 || Tq < 128;
  const auto kq = D == 128 ? (bf ? (two ? window_dq_kernel<Bf16, 128, 2> : window_dq_kernel<Bf16, 128, 1>)
                                 : (two ? window_dq_kernel<Fp16, 128, 2> : window_dq_kernel<Fp16, 128, 1>))
                           : (bf ? (two ? window_dq_kernel<Bf16, 64, 2> : window_dq_kernel<Bf16, 64, 1>)
                                 : (two ? window_dq_kernel<Fp16, 64, 2> : window_dq_kernel<Fp16, 64, 1>));
  hipLaunchKernelGGL(kq, dim3(static_cast<uint32_t>(B * H * a.nqb)), dim3(kThreads), 0, s, a);
  if ((rc = check_launch(what))) return rc;
  const auto kk = D == 128 ? (bf ? (two ? window_dkv_kernel<Bf16, 128, 2> : window_dkv_kernel<Bf16, 128, 1>)
                                 : (two ? window_dkv_kernel<Fp16, 128, 2> : window_dkv_kernel<Fp16, 128, 1>))
                           : (bf ? (two ? window_dkv_kernel<Bf16, 64, 2> : window_dkv_kernel<Bf16, 64, 1>)
                                 : (two ? window_dkv_kernel<Fp16, 64, 2> : window_dkv_kernel<Fp16, 64, 1>));
  hipLaunchKernelGGL(kk, dim3(static_cast<uint32_t>(items)), dim3(kThreads), 0, s, a);
  if ((rc = check_launch(what)) || cut == 0) return rc;
  const auto kj = D == 128 ? (bf ? window_dkv_join_kernel<Bf16, 128> : window_dkv_join_kernel<Fp16, 128>)
                           : (bf ? window_dkv_join_kernel<Bf16, 64> : window_dkv_join_kernel<Fp16, 64>);
  hipLaunchKernelGGL(kj, dim3(static_cast<uint32_t>(join)), dim3(256), 0, s, a, static_cast<int>(cut));
  return check_launch(what);
}
