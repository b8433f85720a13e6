// Keys and values into the 8-bit rows of a paged cache, and rows of sequences back out
// of it (cache8.hpp has the format).
//
// Bound: HBM; for a few tokens the launch and three dependent rounds of memory (length,
// page id, row). A lane holds 8 channels, a row is LPR = 16 lanes (8 up to 64 channels), so
// that the largest magnitude is four lane moves away and a row needs no second pass; k's and
// v's rows of the same place are worked on together and share the page's id. One or two rows a
// lane group and no loop: the launch has thousands of workgroups where bandwidth counts, and
// one round where latency does.
//   Append, 12133 tokens of 24 heads of 128, bf16 to e4m3: 46-48 us, 4.7-4.9 TB/s (a large
//   copy reaches 5.15); two chunks of 1000, 4 heads of 64: 2.8-3.5 us.
//   Read, four sequences of up to 32760 tokens, 8 heads of 128, e4m3 to bf16: 134 us, 5.3 TB/s; the
//   last 1333 of eight, 4 heads of 64: 5.3-5.7 us.
#include "cache8.hpp"

namespace solattn {
namespace {

constexpr int kThreads = 256;

struct Rows {  // [B, T, Hkv, D], strides in elements
  void* p;
  int64_t b, t, h;
};
struct CacheArgs {
  Rows k, v;
  CodePages kc, vc;
  const int32_t* table;
  int64_t table_b;
  const int32_t* lengths;
  const int32_t* start;  // read: null: 0
  int64_t cap;           // tokens that a row of the table holds
  int T, Hkv, D, npages, page;
  int64_t rows;          // B T Hkv
  Divisor by_hkv, by_t, by_page;
};

// Row r of the call: its sequence, token, head and place in the cache (page -1: none).
struct Place {
  int b, t, h, page, slot;
};
__device__ __forceinline__ Place place(const CacheArgs& a, int64_t row, bool append) {
  Place p;
  uint32_t n = static_cast<uint32_t>(row);
  p.h = a.by_hkv.split(n);
  p.t = a.by_t.split(n);
  p.b = n;
  const int64_t len = a.lengths[p.b];
  const int64_t at = append ? len - a.T + p.t : (a.start ? static_cast<int64_t>(a.start[p.b]) : 0) + p.t;
  const bool on = at >= 0 && at < a.cap && (append || at < len);
  const uint32_t j = on ? static_cast<uint32_t>(at) : 0u, pg = a.by_page.of(j);
  p.slot = static_cast<int>(j - pg * a.page);
  p.page = on ? a.table[p.b * a.table_b + pg] : -1;
  if (p.page >= a.npages) p.page = -1;
  return p;
}

template <typename E, typename C, int LPR>
__device__ __forceinline__ void put_row(const CacheArgs& a, const Rows& src, const CodePages& to, const Place& p, int l,
                                        bool active) {
  Row8<E> in;
  in.load(static_cast<const typename E::Raw*>(src.p) + p.b * src.b + p.t * src.t + p.h * src.h + (active ? 8 * l : 0));
  float x[8];
  in.get(x);
  put_codes<C, LPR>(x, to, p.page, p.slot, p.h, l, active, p.page >= 0);
}

template <typename E, typename C, int LPR>
__global__ void __launch_bounds__(kThreads) cache_append_kernel(const CacheArgs a) {
  const int lane = threadIdx.x & 63, l = lane & (LPR - 1);
  const bool active = 8 * l < a.D;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / LPR;
  Place p = place(a, min(row, a.rows - 1), true);
  if (row >= a.rows) p.page = -1;
  put_row<E, C, LPR>(a, a.k, a.kc, p, l, active);
  put_row<E, C, LPR>(a, a.v, a.vc, p, l, active);
}

// Two rows of k and of v a lane group, whose loads are all on their way before the first
// store (four sequences of up to 32760 e4m3 tokens: a row of k, then one of v 144 us, one of
// both 136, two of both 134, four 141).
constexpr int kReadRows = 2;
template <typename E, typename C, int LPR>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const CacheArgs a) {
  constexpr int G = 64 / LPR;  // rows of a wave's access
  const int l = threadIdx.x & (LPR - 1);
  if (8 * l >= a.D) return;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
  const int64_t row = wave * (G * kReadRows) + (threadIdx.x & 63) / LPR;
  Place p[kReadRows];
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) p[u] = place(a, min(row + u * G, a.rows - 1), false);
  uint2 kc[kReadRows], vc[kReadRows];
  float kp[kReadRows], vp[kReadRows];
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    kc[u] = vc[u] = make_uint2(0, 0), kp[u] = vp[u] = 0.f;
    if (p[u].page < 0) continue;
    const auto codes = [&](const CodePages& from) {
      return *reinterpret_cast<const uint2*>(from.codes + p[u].page * from.p + p[u].slot * from.s + p[u].h * from.h + 8 * l);
    };
    const auto power = [&](const CodePages& from) {
      return power_of(from.exps[p[u].page * from.ep + p[u].h * from.eh + p[u].slot]);
    };
    kc[u] = codes(a.kc), vc[u] = codes(a.vc);
    kp[u] = power(a.kc), vp[u] = power(a.vc);
  }
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    if (row + u * G >= a.rows) return;
    const auto put = [&](const Rows& dst, const uint2& c, float power) {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(dst.p) + p[u].b * dst.b + p[u].t * dst.t + p[u].h * dst.h + 8 * l) =
          make_uint4(C::template scaled<E>(c.x, 0, power), C::template scaled<E>(c.x, 2, power),
                     C::template scaled<E>(c.y, 0, power), C::template scaled<E>(c.y, 2, power));
    };
    put(a.k, kc[u], kp[u]);
    put(a.v, vc[u], vp[u]);
  }
}

int setup(CacheArgs& a, int64_t B, int64_t T, int64_t Hkv, int64_t D, int dtype, bool fp32, int64_t pages,
          int64_t page_size, int cache_type, int64_t max_pages, const char* what) {
  SOLATTN_REQUIRE(dtype == SOLATTN_BF16 || dtype == SOLATTN_FP16 || (fp32 && dtype == SOLATTN_FP32), SOLATTN_EINVAL,
                  "%s: dtype %d", what, dtype);
  SOLATTN_REQUIRE(cache_type == SOLATTN_INT8 || cache_type == SOLATTN_E4M3, SOLATTN_EINVAL, "%s: cache type %d", what,
                  cache_type);
  SOLATTN_REQUIRE(B > 0 && T > 0 && Hkv > 0, SOLATTN_EINVAL, "%s: bad sizes", what);
  SOLATTN_REQUIRE(D >= 16 && D <= 128 && D % 16 == 0, SOLATTN_EUNSUPPORTED, "%s: head_dim %lld (multiples of 16 up to 128)",
                  what, (long long)D);
  constexpr int64_t top = 1ll << 31;
  SOLATTN_REQUIRE(B < top && T < top && Hkv < top && B * T < top && B * T * Hkv < top, SOLATTN_EUNSUPPORTED,
                  "%s: too many tokens or heads", what);
  static_assert(kThreads == kLaunchThreads, "one bound");
  SOLATTN_REQUIRE(cdiv(B * T * Hkv, kThreads / (D > 64 ? 16 : 8)) < kMostBlocks, SOLATTN_EUNSUPPORTED,
                  "%s: too many rows for one launch", what);
  SOLATTN_REQUIRE(a.table && a.lengths, SOLATTN_EINVAL, "%s: null page table or lengths", what);
  SOLATTN_REQUIRE(pages >= 0 && pages < top && page_size > 0 && page_size < top && max_pages >= 0 && max_pages < top &&
                      max_pages * page_size < top,
                  SOLATTN_EUNSUPPORTED, "%s: pages beyond 2^31 tokens", what);
  const int64_t whole = dtype == SOLATTN_FP32 ? 4 : 8;
  const auto rows = [&](const Rows& m, const char* name) -> int {
    SOLATTN_REQUIRE(m.p, SOLATTN_EINVAL, "%s: null %s", what, name);
    SOLATTN_REQUIRE(reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.b % whole == 0 && m.t % whole == 0 && m.h % whole == 0,
                    SOLATTN_EINVAL, "%s: %s must be 16-byte aligned with strides that keep its rows so", what, name);
    return 0;
  };
  const auto cache = [&](const CodePages& c, const char* name) -> int {
    SOLATTN_REQUIRE(c.codes && c.exps, SOLATTN_EINVAL, "%s: null %s or its scales", what, name);
    SOLATTN_REQUIRE(reinterpret_cast<uintptr_t>(c.codes) % 16 == 0 && c.p % 16 == 0 && c.s % 16 == 0 && c.h % 16 == 0,
                    SOLATTN_EINVAL, "%s: %s must be 16-byte aligned with strides that keep its rows so", what, name);
    return 0;
  };
  int rc = rows(a.k, "k");
  if (!rc) rc = rows(a.v, "v");
  if (!rc) rc = cache(a.kc, "k_cache");
  if (!rc) rc = cache(a.vc, "v_cache");
  if (rc) return rc;
  a.T = static_cast<int>(T), a.Hkv = static_cast<int>(Hkv), a.D = static_cast<int>(D);
  a.npages = static_cast<int>(pages), a.page = static_cast<int>(page_size);
  a.cap = max_pages * page_size;
  a.rows = B * T * Hkv;
  a.by_hkv = divisor(Hkv), a.by_t = divisor(T), a.by_page = divisor(page_size);
  return 0;
}

}  // namespace
}  // namespace solattn

using namespace solattn;

#define SOLATTN_BY_CODES(KERN, E, codes, wide)                              \
  ((codes) == SOLATTN_INT8 ? ((wide) ? KERN<E, Int8Codes, 16> : KERN<E, Int8Codes, 8>) \
                           : ((wide) ? KERN<E, Fp8Codes, 16> : KERN<E, Fp8Codes, 8>))

extern "C" int solattn_cache_append(const void* k, int64_t sk_b, int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_b,
                                    int64_t sv_t, int64_t sv_h, int64_t B, int64_t T, int64_t Hkv, int64_t D, int dtype,
                                    void* k_cache, int64_t skc_p, int64_t skc_s, int64_t skc_h, void* v_cache,
                                    int64_t svc_p, int64_t svc_s, int64_t svc_h, int64_t pages, int64_t page_size,
                                    int cache_type, uint8_t* k_scale, int64_t sks_p, int64_t sks_h, uint8_t* v_scale,
                                    int64_t svs_p, int64_t svs_h, const int32_t* page_table, int64_t table_stride,
                                    int64_t max_pages, const int32_t* lengths, solattn_stream_t stream) {
  clear_error();
  CacheArgs a{};
  a.k = {const_cast<void*>(k), sk_b, sk_t, sk_h};
  a.v = {const_cast<void*>(v), sv_b, sv_t, sv_h};
  a.kc = {static_cast<uint8_t*>(k_cache), skc_p, skc_s, skc_h, k_scale, sks_p, sks_h};
  a.vc = {static_cast<uint8_t*>(v_cache), svc_p, svc_s, svc_h, v_scale, svs_p, svs_h};
  a.table = page_table, a.table_b = table_stride, a.lengths = lengths;
  if (int rc = setup(a, B, T, Hkv, D, dtype, true, pages, page_size, cache_type, max_pages, "cache_append")) return rc;
  const bool wide = D > 64;
  const auto kern = dtype == SOLATTN_BF16   ? SOLATTN_BY_CODES(cache_append_kernel, Bf16, cache_type, wide)
                    : dtype == SOLATTN_FP16 ? SOLATTN_BY_CODES(cache_append_kernel, Fp16, cache_type, wide)
                                            : SOLATTN_BY_CODES(cache_append_kernel, Fp32, cache_type, wide);
  const int64_t blocks = cdiv(a.rows, kThreads / (wide ? 16 : 8));
  hipLaunchKernelGGL(kern, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, reinterpret_cast<hipStream_t>(stream), a);
  return check_launch("cache_append");
}

extern "C" int solattn_cache_read(const void* k_cache, int64_t skc_p, int64_t skc_s, int64_t skc_h, const void* v_cache,
                                  int64_t svc_p, int64_t svc_s, int64_t svc_h, int64_t pages, int64_t page_size,
                                  int cache_type, const uint8_t* k_scale, int64_t sks_p, int64_t sks_h,
                                  const uint8_t* v_scale, int64_t svs_p, int64_t svs_h, const int32_t* page_table,
                                  int64_t table_stride, int64_t max_pages, const int32_t* lengths, const int32_t* start,
                                  int64_t B, int64_t T, int64_t Hkv, int64_t D, int dtype, uint16_t* k, int64_t sk_b,
                                  int64_t sk_t, int64_t sk_h, uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h,
                                  solattn_stream_t stream) {
  clear_error();
  CacheArgs a{};
  a.k = {k, sk_b, sk_t, sk_h};
  a.v = {v, sv_b, sv_t, sv_h};
  a.kc = {static_cast<uint8_t*>(const_cast<void*>(k_cache)), skc_p, skc_s, skc_h, const_cast<uint8_t*>(k_scale), sks_p, sks_h};
  a.vc = {static_cast<uint8_t*>(const_cast<void*>(v_cache)), svc_p, svc_s, svc_h, const_cast<uint8_t*>(v_scale), svs_p, svs_h};
  a.table = page_table, a.table_b = table_stride, a.lengths = lengths, a.start = start;
  if (int rc = setup(a, B, T, Hkv, D, dtype, false, pages, page_size, cache_type, max_pages, "cache_read")) return rc;
  const bool wide = D > 64;
  const auto kern = dtype == SOLATTN_BF16 ? SOLATTN_BY_CODES(cache_read_kernel, Bf16, cache_type, wide)
                                          : SOLATTN_BY_CODES(cache_read_kernel, Fp16, cache_type, wide);
  const int64_t blocks = cdiv(a.rows, kReadRows * (kThreads / (wide ? 16 : 8)));
  hipLaunchKernelGGL(kern, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, reinterpret_cast<hipStream_t>(stream), a);
  return check_launch("cache_read");
}
