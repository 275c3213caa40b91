// Operators for drafted tokens that are bound by memory: rotary positions with the cache rows they go to, cache rows read back,
// and adjusted logits.  Shapes and errors: include/vdcores.h.
#include "mk_stage.cuh"

namespace vdc {
namespace {

constexpr int D = VDC_HEAD_DIM, PAGE = VDC_KV_PAGE;

// Byte of row `row` of a page at which lane (0..15) of the row's half-warp keeps its eight values.
template <bool kF8>
__device__ __forceinline__ int lane_place(int row, int lane) {
  return kF8 ? ((((lane >> 1) ^ (row & 7)) << 4) | ((lane & 1) << 3)) : ((lane ^ (row & 7)) << 4);
}

// The page of row `at` of a sequence, or -1 (reported) where the row or the page does not exist.
__device__ __forceinline__ int page_of(const vdc_cache& c, const int* pages, int64_t at, int max_pages, vdc_status* status, int kind,
                                       int b) {
  if (at < 0 || at >= (int64_t)max_pages * PAGE) {
    report(status, VDC_ERR_RANGE, kind, 0, b, (int)at);
    return -1;
  }
  const int p = __ldg(pages + at / PAGE);
  if (p < 0 || p >= c.n_pages) {
    report(status, VDC_ERR_RANGE, kind, 1, b, p);
    return -1;
  }
  return p;
}

// ------------------------------------------------------------------------- //
// rope_append: a block per token; a half-warp takes one head's row of 128 values at a time.  A lane keeps the two values of four pairs
// (x, y): two pieces of four values, which lie next to each other where pairs do, else half the rotated part apart.  So a pair never
// crosses lanes, and the token's cosines and sines stay in registers over its heads.  Query rows are loaded four at a time and ahead
// of the page table, whose chain of loads is what a token would otherwise wait for.  Products and sums are rounded one by one (no
// contraction), so that the codes of a row do not depend on how the compiler pairs them.
// 8192 tokens, 32 query and 2 x 4 cache heads, norms, e4m3: 44.5 us (bytes alone: 25); two thirds of the issue slots, the rest waits for
// loads.  One token: 4.3 us.
// ------------------------------------------------------------------------- //
constexpr int kAppendMaxThreads = 256, kAppendRows = 4;

// From a half-warp's query row to its next one: heads of the cache and places in their groups, and what that adds to the addresses.
struct AppendStep {
  int kv, g;
  int64_t q, o, q_wrap, o_wrap;
};

// x / s for finite s and x, correctly rounded: one correction of the product with the correctly rounded reciprocal (Markstein's theorem;
// the residue is exact for the x that have a code, those above s 2^-10).
__device__ __forceinline__ uint64_t quotient2(uint64_t x, uint64_t minus_s, uint64_t inv) {
  const uint64_t q = mul2(x, inv);
  return fma2(fma2(q, minus_s, x), inv, q);
}

// Four pairs: the first values x, the second ones y.
template <bool kPairs>
struct FourPairs {
  uint64_t x[2], y[2];
  __device__ __forceinline__ FourPairs(uint2 l, uint2 h) {
    if constexpr (kPairs) {
      x[0] = two(bf_lo(l.x), bf_lo(l.y)); y[0] = two(bf_hi(l.x), bf_hi(l.y));
      x[1] = two(bf_lo(h.x), bf_lo(h.y)); y[1] = two(bf_hi(h.x), bf_hi(h.y));
    } else {
      x[0] = two(bf_lo(l.x), bf_hi(l.x)); x[1] = two(bf_lo(l.y), bf_hi(l.y));
      y[0] = two(bf_lo(h.x), bf_hi(h.x)); y[1] = two(bf_lo(h.y), bf_hi(h.y));
    }
  }
  __device__ __forceinline__ void norm(const FourPairs& w, float eps, unsigned mask) {
    const float2 sums = apart(fma2(y[1], y[1], fma2(y[0], y[0], fma2(x[1], x[1], mul2(x[0], x[0])))));
    float ss = sums.x + sums.y;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
    const float rs = rsqrtf(ss * (1.f / D) + eps);
    const uint64_t rs2 = two(rs, rs);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[i] = mul2(mul2(x[i], rs2), w.x[i]);
      y[i] = mul2(mul2(y[i], rs2), w.y[i]);
    }
  }
  __device__ __forceinline__ void turn(const uint64_t (&cs)[2], const uint64_t (&sn)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint64_t was = x[i];
      x[i] = fma2(mul2(y[i], sn[i]), two(-1.f, -1.f), mul2(was, cs[i]));
      y[i] = add2(mul2(y[i], cs[i]), mul2(was, sn[i]));
    }
  }
  __device__ __forceinline__ void pack(uint2& l, uint2& h) const {
    const float2 x0 = apart(x[0]), x1 = apart(x[1]), y0 = apart(y[0]), y1 = apart(y[1]);
    l = kPairs ? make_uint2(pack_bf16x2(x0.x, y0.x), pack_bf16x2(x0.y, y0.y)) : make_uint2(pack_bf16x2(x0.x, x0.y), pack_bf16x2(x1.x, x1.y));
    h = kPairs ? make_uint2(pack_bf16x2(x1.x, y1.x), pack_bf16x2(x1.y, y1.y)) : make_uint2(pack_bf16x2(y0.x, y0.y), pack_bf16x2(y1.x, y1.y));
  }
  // e4m3 codes of the row, and its scale
  __device__ __forceinline__ float encode(uint32_t& l, uint32_t& h, unsigned mask) const {
    // magnitudes compare as whole numbers, infinity above all finite ones and NaN above infinity: a row with either gets a scale that
    // says so, codes of zero, and none where there is no finite number
    auto size = [](uint64_t v) {
      const float2 f = apart(v);
      return max(__float_as_uint(f.x) & 0x7FFFFFFFu, __float_as_uint(f.y) & 0x7FFFFFFFu);
    };
    uint32_t top = max(max(size(x[0]), size(x[1])), max(size(y[0]), size(y[1])));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
    const float most = __uint_as_float(top), scale = __fdiv_rn(most < 1e-12f ? 1e-12f : most, 448.f);
    const bool finite = top < 0x7F800000u;
    const float inv = finite ? __frcp_rn(scale) : 0.f, minus = finite ? -scale : 0.f;
    const uint64_t inv2 = two(inv, inv), minus2 = two(minus, minus);
    auto codes = [](float a, float b, float c, float d) {
      return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
             (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
    };
    const float2 x0 = apart(quotient2(x[0], minus2, inv2)), x1 = apart(quotient2(x[1], minus2, inv2));
    const float2 y0 = apart(quotient2(y[0], minus2, inv2)), y1 = apart(quotient2(y[1], minus2, inv2));
    l = kPairs ? codes(x0.x, y0.x, x0.y, y0.y) : codes(x0.x, x0.y, x1.x, x1.y);
    h = kPairs ? codes(x1.x, y1.x, x1.y, y1.y) : codes(y0.x, y0.y, y1.x, y1.y);
    return scale;
  }
};

template <bool kF8, bool kPairs>
__global__ void __launch_bounds__(kAppendMaxThreads, 4)
rope_append(const __grid_constant__ vdc_rope_append_args a, const __grid_constant__ AppendStep step, vdc_status* status) {
  const int t = blockIdx.x, lane = threadIdx.x & 15, half_warp = threadIdx.x >> 4, half_warps = blockDim.x >> 4;
  const unsigned mask = 0xFFFFu << (threadIdx.x & 16);
  const vdc_cache& c = a.cache;
  const int n_q = c.n_kv * a.group;
  const bool rotates = lane < a.rot / 8;
  const int c0 = kPairs || !rotates ? 2 * lane : lane, c1 = kPairs || !rotates ? 2 * lane + 1 : lane + a.rot / 8;      // the pieces
  const int first_kv = (unsigned)half_warp / (unsigned)a.group, first_g = half_warp - first_kv * a.group;

  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const uint2* q = reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + b * a.q_b + t * a.q_t + first_kv * a.q_kv + first_g * a.q_g) + c0;
    uint2* out = reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + b * a.o_b + t * a.o_t + first_kv * a.o_kv + first_g * a.o_g) + c0;
    int g_in = first_g, g_out = first_g;
    uint2 lo[kAppendRows], hi[kAppendRows];
    auto load = [&](int r) {
#pragma unroll
      for (int j = 0; j < kAppendRows; ++j, r += half_warps) {
        if (r < n_q) lo[j] = q[0], hi[j] = q[c1 - c0];
        q += step.q;
        g_in += step.g;
        if (g_in >= a.group) g_in -= a.group, q += step.q_wrap;
      }
    };
    load(half_warp);

    const int64_t at = (int64_t)__ldg(reinterpret_cast<const int*>(a.lengths) + b) + t;
    bool live = !a.counts || t < __ldg(reinterpret_cast<const int*>(a.counts) + b);
    int64_t turn = at;
    if (a.positions) turn = __ldg(reinterpret_cast<const int*>(a.positions) + b * a.pos_b + t * a.pos_t);
    int page = 0;
    if (live) {
      page = page_of(c, reinterpret_cast<const int*>(a.pages) + b * a.pages_b, at, a.max_pages, status, VDC_ROPE_APPEND_KIND, b);
      if (a.rot && (turn < 0 || turn >= a.table_rows)) {
        report(status, VDC_ERR_RANGE, VDC_ROPE_APPEND_KIND, 2, b, (int)turn);
        page = -1;
      }
      live = page >= 0;
    }
    uint64_t cs[2], sn[2];
    if (live && rotates) {
      const float* tab = reinterpret_cast<const float*>(a.table) + turn * a.rot + lane * 4;
      const float4 x = __ldg(reinterpret_cast<const float4*>(tab)), y = __ldg(reinterpret_cast<const float4*>(tab + a.rot / 2));
      cs[0] = two(x.x, x.y); cs[1] = two(x.z, x.w);
      sn[0] = two(y.x, y.y); sn[1] = two(y.z, y.w);
    }
    auto weights = [&](uint64_t norm) {
      const uint2* w = reinterpret_cast<const uint2*>(norm);
      return FourPairs<kPairs>(__ldg(w + c0), __ldg(w + c1));
    };

    // ---- queries
    FourPairs<kPairs> w(make_uint2(0, 0), make_uint2(0, 0));
    if (a.q_norm) w = weights(a.q_norm);
    for (int r = half_warp; r < n_q;) {
#pragma unroll
      for (int j = 0; j < kAppendRows; ++j, r += half_warps) {
        if (r >= n_q) break;
        FourPairs<kPairs> x(lo[j], hi[j]);
        if (a.q_norm) x.norm(w, a.eps, mask);
        if (rotates) x.turn(cs, sn);
        uint2 l, h;
        x.pack(l, h);
        out[0] = live ? l : make_uint2(0, 0);
        out[c1 - c0] = live ? h : make_uint2(0, 0);
        out += step.o;
        g_out += step.g;
        if (g_out >= a.group) g_out -= a.group, out += step.o_wrap;
      }
      if (r < n_q) load(r);
    }
    if (!live) continue;

    // ---- keys and values
    if (a.k_norm) w = weights(a.k_norm);
    const int row = (int)(at & (PAGE - 1));
    for (int r = half_warp; r < 2 * c.n_kv; r += half_warps) {
      const bool value = r >= c.n_kv;
      const int head = value ? r - c.n_kv : r;
      const uint2* src = reinterpret_cast<const uint2*>(value ? reinterpret_cast<const __nv_bfloat16*>(a.v) + b * a.v_b + t * a.v_t + head * a.v_kv
                                                              : reinterpret_cast<const __nv_bfloat16*>(a.k) + b * a.k_b + t * a.k_t + head * a.k_kv);
      FourPairs<kPairs> x(__ldg(src + c0), __ldg(src + c1));
      if (!value) {
        if (a.k_norm) x.norm(w, a.eps, mask);
        if (rotates) x.turn(cs, sn);
      }
      uint8_t* dst = reinterpret_cast<uint8_t*>(value ? c.v : c.k) + page * (value ? c.v_page : c.k_page) + head * (value ? c.v_head : c.k_head) +
                     row * (kF8 ? D : 2 * D);
      if constexpr (!kF8) {
        uint2 l, h;
        x.pack(l, h);
        *reinterpret_cast<uint2*>(dst + (((c0 >> 1) ^ (row & 7)) << 4) + (c0 & 1) * 8) = l;
        *reinterpret_cast<uint2*>(dst + (((c1 >> 1) ^ (row & 7)) << 4) + (c1 & 1) * 8) = h;
      } else {
        uint32_t l, h;
        const float scale = x.encode(l, h, mask);
        *reinterpret_cast<uint32_t*>(dst + (((c0 >> 2) ^ (row & 7)) << 4) + (c0 & 3) * 4) = l;
        *reinterpret_cast<uint32_t*>(dst + (((c1 >> 2) ^ (row & 7)) << 4) + (c1 & 3) * 4) = h;
        if (lane == 0)
          *reinterpret_cast<float*>((value ? c.v_scale + page * c.vs_page + head * c.vs_head : c.k_scale + page * c.ks_page + head * c.ks_head) + row * 4) = scale;
      }
    }
  }
}

// ------------------------------------------------------------------------- //
// read_cache: a half-warp per row of one head, keys and values, two rows at a time so that more loads are on their way; rows are bytes
// in and bytes out, so memory is the bound.  16 sequences of up to 4131 e4m3 rows of 8 heads: 65.6 us, 88 % of a plain copy's rate.
// ------------------------------------------------------------------------- //
constexpr int kReadThreads = 256, kReadRows = 2, kReadUnits = kReadThreads / 16 * kReadRows;

template <bool kF8>
__device__ __forceinline__ uint4 stored8(const uint8_t* src, float scale) {
  if constexpr (!kF8) {
    return __ldg(reinterpret_cast<const uint4*>(src));
  } else {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(src));
    float x[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = e4m3x2_to_float2(((j < 2 ? w.x : w.y) >> (16 * (j & 1))) & 0xFFFFu);
      x[2 * j] = f.x * scale;
      x[2 * j + 1] = f.y * scale;
    }
    return pack8(x);
  }
}

template <bool kF8>
__global__ void __launch_bounds__(kReadThreads) read_cache(const vdc_read_cache_args a, vdc_status* status) {
  const vdc_cache& c = a.cache;
  const int b = blockIdx.y, lane = threadIdx.x & 15;
  const unsigned units = (unsigned)a.n * c.n_kv, unit0 = blockIdx.x * kReadUnits + (threadIdx.x >> 4);
  const int start = a.start ? __ldg(reinterpret_cast<const int*>(a.start) + b) : 0, length = __ldg(reinterpret_cast<const int*>(a.lengths) + b);
  uint4 ks[kReadRows], vs[kReadRows];
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    const unsigned unit = unit0 + u * (kReadThreads / 16);
    const int i = (int)(unit / (unsigned)c.n_kv), head = (int)(unit - i * (unsigned)c.n_kv);
    const int64_t at = (int64_t)start + i;
    uint4 &k = ks[u], &v = vs[u];
    k = v = make_uint4(0, 0, 0, 0);
    if (unit >= units || at >= length) continue;
    const int page = page_of(c, reinterpret_cast<const int*>(a.pages) + b * a.pages_b, at, a.max_pages, status, VDC_READ_CACHE_KIND, b);
    if (page >= 0) {
      const int row = (int)(at & (PAGE - 1)), place = row * (kF8 ? D : 2 * D) + lane_place<kF8>(row, lane);
      float k_scale = 1.f, v_scale = 1.f;
      if constexpr (kF8) {
        k_scale = __ldg(reinterpret_cast<const float*>(c.k_scale + page * c.ks_page + head * c.ks_head) + row);
        v_scale = __ldg(reinterpret_cast<const float*>(c.v_scale + page * c.vs_page + head * c.vs_head) + row);
      }
      k = stored8<kF8>(reinterpret_cast<const uint8_t*>(c.k) + page * c.k_page + head * c.k_head + place, k_scale);
      v = stored8<kF8>(reinterpret_cast<const uint8_t*>(c.v) + page * c.v_page + head * c.v_head + place, v_scale);
    }
  }
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    const unsigned unit = unit0 + u * (kReadThreads / 16);
    if (unit >= units) break;
    const int64_t to = ((int64_t)b * units + unit) * D + lane * 8;
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.k_out) + to) = ks[u];
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.v_out) + to) = vs[u];
  }
}

// ------------------------------------------------------------------------- //
// adjust_logits: a row is shared by the CTAs of a cluster, a contiguous part of the vocabulary each, walked in tiles.  For a tile a
// CTA counts the row's ids that fall into it in shared memory: a word a token with the times generated and, above them, a bit for
// "biased" and one for "in the prompt".  Then one pass over the tile's logits, eight at a time: most have a word of zero and need
// nothing.  The words have 16 bits where the ids cannot overflow 14 of them, otherwise 32 and half the tile.
// The largest logits meet over the cluster.
// ------------------------------------------------------------------------- //
constexpr int kLogitThreads = 512, kLogitCountBytes = 65536, kLogitMaxBias = 4096, kLogitShort = 0x3FFF;

__device__ __forceinline__ float2 pair_of(uint32_t u, __nv_bfloat16) { return make_float2(bf_lo(u), bf_hi(u)); }
__device__ __forceinline__ float2 pair_of(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ uint32_t pair_to(float x, float y, __nv_bfloat16) { return pack_bf16x2(x, y); }
__device__ __forceinline__ uint32_t pair_to(float x, float y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

// Eight logits as they lie in memory, at a multiple of 16 bytes.
template <class T>
struct Eight {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    if constexpr (sizeof(T) == 4) {
      const uint32_t u[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(u[i]);
    } else {
      const uint32_t u[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = pair_of(u[i], T());
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
};
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pair_to(x[0], x[1], T()), pair_to(x[2], x[3], T()), pair_to(x[4], x[5], T()), pair_to(x[6], x[7], T()));
  }
}

// Largest first, and the lower id of two equal ones; NaN never.
__device__ __forceinline__ void better(float& v, int& i, float v2, int i2) {
  if (v2 > v || (v2 == v && i2 < i)) v = v2, i = i2;
}

struct LogitShared {
  float best[32];
  int at[32];
  float cta_best;
  int cta_at;
};

template <class Tin, class Tout, class Count>
__global__ void __launch_bounds__(kLogitThreads, 3) adjust_logits(const vdc_adjust_logits_args a, int parts, vdc_status* status) {
  constexpr int kTile = kLogitCountBytes / (int)sizeof(Count);       // tokens
  constexpr uint32_t kPrompt = 1u << (8 * sizeof(Count) - 1), kBiased = kPrompt >> 1;
  extern __shared__ uint4 dyn[];                                     // the tile's words, then the row's biases: ids, values
  __shared__ LogitShared sh;
  uint32_t* count = reinterpret_cast<uint32_t*>(dyn);
  int* ids = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(dyn) + kLogitCountBytes);
  float* add = reinterpret_cast<float*>(ids + a.n_bias);
  const int row = blockIdx.x / parts, part = blockIdx.x % parts, tid = threadIdx.x;
  const Tin* in = reinterpret_cast<const Tin*>(a.logits) + row * a.logits_s;
  Tout* out = reinterpret_cast<Tout*>(a.out) + row * a.out_s;
  int req = row;
  if (a.requests) req = __ldg(reinterpret_cast<const int*>(a.requests) + row);
  const bool known = req >= 0 && req < a.n;
  if (!known && part == 0 && tid == 0) report(status, VDC_ERR_RANGE, VDC_ADJUST_LOGITS_KIND, 3, row, req);
  auto factor = [&](uint64_t p, float none) { return p && known ? __ldg(reinterpret_cast<const float*>(p) + req) : none; };
  const float rep = factor(a.repetition, 1.f), freq = factor(a.frequency, 0.f), pres = factor(a.presence, 0.f);
  const bool seen_matters = known && (a.repetition || a.frequency || a.presence);
  const int* hist = reinterpret_cast<const int*>(a.history) + (known ? req * a.history_s : 0);
  int n_hist = 0, n_prompt = 0;
  if (seen_matters && a.history) {
    n_hist = a.history_lens ? max(0, min(a.L, __ldg(reinterpret_cast<const int*>(a.history_lens) + req))) : a.L;
    n_prompt = a.prompt_lens ? max(0, min(n_hist, __ldg(reinterpret_cast<const int*>(a.prompt_lens) + req))) : 0;
  }
  const int n_path = seen_matters && a.path ? a.path_n : 0;
  const int* path = reinterpret_cast<const int*>(a.path) + row * a.path_s;
  const int n_bias = known && a.bias_ids ? a.n_bias : 0;
  const bool counted = n_hist + n_path + n_bias > 0;
  for (int i = tid; i < n_bias; i += kLogitThreads) {
    ids[i] = __ldg(reinterpret_cast<const int*>(a.bias_ids) + req * a.bias_s + i);
    add[i] = __ldg(reinterpret_cast<const float*>(a.bias) + req * a.bias_s + i);
  }
  const uint32_t* allowed = a.allowed ? reinterpret_cast<const uint32_t*>(a.allowed) + row * a.allowed_s : nullptr;

  // Groups of eight tokens start where a load of eight logits may: group g holds tokens 8 g - lead .. 8 g - lead + 7, of which the
  // first and the last group have some only.
  const int lead = (int)(((uintptr_t)in & 15) / sizeof(Tin)), n_groups = (a.vocab + lead + 7) / 8;
  const int per = (n_groups + parts - 1) / parts, g_begin = min(n_groups, part * per), g_end = min(n_groups, g_begin + per);
  const bool wide_out = (((uintptr_t)(out - lead)) & 15) == 0;
  auto whole = [&](int g) { return 8 * g >= lead && 8 * g + 8 - lead <= a.vocab; };

  float best = -INFINITY;
  int best_at = 0x7FFFFFFF;
  for (int g0 = g_begin; g0 < g_end; g0 += kTile / 8) {
    const int g1 = min(g_end, g0 + kTile / 8), first = 8 * g0 - lead;       // the tile's first token
    if (counted) {
      __syncthreads();
      for (int i = tid; i < (g1 - g0) * (int)sizeof(Count) / 2; i += kLogitThreads) dyn[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      const unsigned n = (unsigned)(g1 - g0) * 8;
      auto mark = [&](unsigned k, uint32_t bit, bool once) {
        if (k >= n) return;
        uint32_t* word = sizeof(Count) == 4 ? count + k : count + (k >> 1);
        bit <<= sizeof(Count) == 4 ? 0 : 16 * (k & 1);
        if (once) atomicOr(word, bit);
        else atomicAdd(word, bit);
      };
#pragma unroll 4
      for (int i = tid; i < n_hist; i += kLogitThreads) {
        const unsigned k = (unsigned)(__ldg(hist + i) - first);
        mark(k, i < n_prompt ? kPrompt : 1u, i < n_prompt);
      }
      for (int i = tid; i < n_path; i += kLogitThreads) mark((unsigned)(__ldg(path + i) - first), 1u, false);
      for (int i = tid; i < n_bias; i += kLogitThreads) mark((unsigned)(ids[i] - first), kBiased, true);
      __syncthreads();
    }
    Eight<Tin> next;
    int g = g0 + tid;
    if (g < g1 && whole(g)) next.load(in + (8 * g - lead));
    for (; g < g1; g += kLogitThreads) {
      const int v = 8 * g - lead;
      const bool full = whole(g);
      float x[8];
      uint32_t exist = 0xFF;
      if (full) {
        next.get(x);
      } else {
        exist = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool is = v + j >= 0 && v + j < a.vocab;
          x[j] = is ? to_f32(in[v + j]) : -INFINITY;
          exist |= (uint32_t)is << j;
        }
      }
      const int g2 = g + kLogitThreads;
      if (g2 < g1 && whole(g2)) next.load(in + (8 * g2 - lead));
      if (counted) {
        uint32_t w[8];
        uint32_t any;
        if constexpr (sizeof(Count) == 2) {
          const uint4 c = dyn[g - g0];
          any = c.x | c.y | c.z | c.w;
          w[0] = c.x & 0xFFFF; w[1] = c.x >> 16; w[2] = c.y & 0xFFFF; w[3] = c.y >> 16;
          w[4] = c.z & 0xFFFF; w[5] = c.z >> 16; w[6] = c.w & 0xFFFF; w[7] = c.w >> 16;
        } else {
          const uint4 c = dyn[2 * (g - g0)], d = dyn[2 * (g - g0) + 1];
          any = c.x | c.y | c.z | c.w | d.x | d.y | d.z | d.w;
          w[0] = c.x; w[1] = c.y; w[2] = c.z; w[3] = c.w; w[4] = d.x; w[5] = d.y; w[6] = d.z; w[7] = d.w;
        }
        if (any) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (w[j] & ~kBiased) {
              const uint32_t times = w[j] & (kBiased - 1);
              if (a.repetition) x[j] = x[j] > 0.f ? __fdiv_rn(x[j], rep) : __fmul_rn(x[j], rep);
              x[j] = __fsub_rn(x[j], __fmul_rn(freq, (float)times));
              if (times) x[j] = __fsub_rn(x[j], pres);
            }
            if (w[j] & kBiased) {
              float sum = 0.f;
              for (int i = 0; i < n_bias; ++i)
                if (ids[i] == v + j) sum += add[i];
              x[j] = __fadd_rn(x[j], sum);
            }
          }
        }
      }
      if (allowed) {
        const int v1 = max(v, 0), word = v1 >> 5;
        const uint32_t lo = __ldg(allowed + word), hi = (v1 & 31) > 24 && 32 * (word + 1) < a.vocab ? __ldg(allowed + word + 1) : 0u;
        const uint32_t bits = __funnelshift_r(lo, hi, v1 & 31) << (v1 - v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!((bits >> j) & 1)) x[j] = -INFINITY;
      }
      const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      if (top > best) {
        best = top;
#pragma unroll
        for (int j = 7; j >= 0; --j)
          if (x[j] == top) best_at = v + j;
      }
      if (full && wide_out) {
        store8(out + v, x);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if ((exist >> j) & 1) out[v + j] = from_f32<Tout>(x[j]);
      }
    }
  }
  if (!a.tokens) return;      // the same for every CTA of a cluster
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(best, best_at, __shfl_xor_sync(~0u, best, o), __shfl_xor_sync(~0u, best_at, o));
  if ((tid & 31) == 0) sh.best[tid >> 5] = best, sh.at[tid >> 5] = best_at;
  __syncthreads();
  if (tid < 32) {
    best = tid < kLogitThreads / 32 ? sh.best[tid] : -INFINITY;
    best_at = tid < kLogitThreads / 32 ? sh.at[tid] : 0x7FFFFFFF;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) better(best, best_at, __shfl_xor_sync(~0u, best, o), __shfl_xor_sync(~0u, best_at, o));
    if (tid == 0) sh.cta_best = best, sh.cta_at = best_at;
  }
  if (parts > 1) {
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    if (part == 0 && tid == 0) {
      for (int p = 1; p < parts; ++p)
        better(best, best_at, ld_cluster1(peer_smem(smem_u32(&sh.cta_best), p)),
               __float_as_int(ld_cluster1(peer_smem(smem_u32(&sh.cta_at), p))));
    }
    cluster_arrive();
    cluster_wait();
  }
  if (part == 0 && tid == 0) reinterpret_cast<int*>(a.tokens)[row] = known && best > -INFINITY ? best_at : -1;
}

bool al(uint64_t p, int n) { return p % n == 0; }

const char* check_cache(const vdc_cache& c, int max_pages) {
  if (c.kind != 0 && c.kind != 1) return "cache: unknown kind";
  if (c.n_kv < 1 || c.n_kv > 4096 || c.n_pages < 1 || max_pages < 1) return "cache: heads or pages out of range";
  if (!c.k || !c.v || !al(c.k | c.v, 16) || !al(c.k_page | c.k_head | c.v_page | c.v_head, 16)) return "cache: null or misaligned pages";
  if (c.kind == 1 && (!c.k_scale || !c.v_scale || !al(c.k_scale | c.v_scale, 16) ||
                      !al(c.ks_page | c.ks_head | c.vs_page | c.vs_head, 16)))
    return "cache: null or misaligned scales";
  return nullptr;
}

}  // namespace
}  // namespace vdc

using namespace vdc;

extern "C" const char* vdc_cache_refuses(const vdc_cache* c, int max_pages) { return check_cache(*c, max_pages); }

extern "C" const char* vdc_rope_append_refuses(const vdc_rope_append_args* a) {
  if (const char* why = check_cache(a->cache, a->max_pages)) return why;
  if (a->B < 1 || a->T < 1 || a->group < 1 || a->group > 4096 || (int64_t)a->B * a->T > 0x7FFFFFFF) return "rope_append: tokens or heads out of range";
  if (a->rot < 0 || a->rot > VDC_HEAD_DIM || a->rot % 16) return "rope_append: the rotated part must be a multiple of 16 up to 128";
  if (a->rot && (!a->table || a->table_rows < 1 || !al(a->table, 16))) return "rope_append: null or misaligned table";
  if (!a->q || !a->k || !a->v || !a->out || !al(a->q | a->k | a->v | a->out | a->q_norm | a->k_norm, 16))
    return "rope_append: null or misaligned rows";
  if (!al(a->q_b | a->q_t | a->q_kv | a->q_g | a->k_b | a->k_t | a->k_kv | a->v_b | a->v_t | a->v_kv | a->o_b | a->o_t | a->o_kv | a->o_g, 8))
    return "rope_append: row strides must be multiples of 8";
  if (!a->pages || !a->lengths || !al(a->pages | a->lengths | a->counts | a->positions, 4)) return "rope_append: null or misaligned tables";
  return nullptr;
}

extern "C" cudaError_t vdc_rope_append_launch(const vdc_rope_append_args* a, vdc_status* status, cudaStream_t stream) {
  const dim3 grid((unsigned)a->T, (unsigned)(a->B < 65535 ? a->B : 65535));
  // As many half-warps for a token as the warps that can be resident allow: few tokens wait for one chain of loads, many for what each
  // warp does per token.  32 query and 2 x 8 cache heads, us with 256 / 128 / 64 threads: 1 token 4.4 / 6.2 / 8.2, 512 tokens
  // 7.4 / 7.2 / 8.3, 1024 tokens 10+ / 8.4 / 10.3, 2048 tokens - / 14.4 / 13.7, 8192 tokens 68 / 49.3 / 47.3.
  int threads = kAppendMaxThreads;
  while (threads > 64 && (int64_t)a->B * a->T * (threads / 32) > VDC_MAX_SMS * 32) threads /= 2;
  AppendStep step;
  step.kv = threads / 16 / a->group;
  step.g = threads / 16 - step.kv * a->group;
  step.q = (step.kv * a->q_kv + step.g * a->q_g) / 4;
  step.o = (step.kv * a->o_kv + step.g * a->o_g) / 4;
  step.q_wrap = (a->q_kv - a->group * a->q_g) / 4;
  step.o_wrap = (a->o_kv - a->group * a->o_g) / 4;
  const auto run = a->cache.kind ? a->interleaved ? rope_append<true, true> : rope_append<true, false>
                                 : a->interleaved ? rope_append<false, true> : rope_append<false, false>;
  run<<<grid, threads, 0, stream>>>(*a, step, status);
  return cudaGetLastError();
}

extern "C" const char* vdc_read_cache_refuses(const vdc_read_cache_args* a) {
  if (const char* why = check_cache(a->cache, a->max_pages)) return why;
  if (a->B < 1 || a->B > 65535 || a->n < 1 || (int64_t)a->n * a->cache.n_kv > 0x40000000) return "read_cache: sequences or rows out of range";
  if (!a->pages || !a->lengths || !al(a->pages | a->lengths | a->start, 4)) return "read_cache: null or misaligned tables";
  return a->k_out && a->v_out && al(a->k_out | a->v_out, 16) ? nullptr : "read_cache: null or misaligned rows";
}

extern "C" cudaError_t vdc_read_cache_launch(const vdc_read_cache_args* a, vdc_status* status, cudaStream_t stream) {
  const unsigned units = (unsigned)a->n * a->cache.n_kv;
  const dim3 grid((units + kReadUnits - 1) / kReadUnits, (unsigned)a->B);
  if (a->cache.kind) read_cache<true><<<grid, kReadThreads, 0, stream>>>(*a, status);
  else read_cache<false><<<grid, kReadThreads, 0, stream>>>(*a, status);
  return cudaGetLastError();
}

extern "C" const char* vdc_adjust_logits_refuses(const vdc_adjust_logits_args* a) {
  if (a->rows < 1 || a->vocab < 1 || a->vocab > 0x3FFFFFFF || a->n < 1 || a->L < 0 || a->path_n < 0 || a->n_bias < 0 ||
      a->n_bias > kLogitMaxBias || (int64_t)a->rows * 8 > 0x7FFFFFFF)
    return "adjust_logits: rows, vocabulary, requests or biases out of range";
  if (a->type < 0 || a->type > 2 || (a->out_type != a->type && a->out_type != 0)) return "adjust_logits: unknown types";
  const int size = a->type ? 2 : 4, out_size = a->out_type ? 2 : 4;
  if (!a->logits || !a->out || !al(a->logits, size) || !al(a->out, out_size)) return "adjust_logits: null or misaligned logits";
  if ((a->bias_ids != 0) != (a->bias != 0)) return "adjust_logits: biases without ids, or ids without biases";
  if (!a->requests && a->n < a->rows) return "adjust_logits: fewer requests than rows, and nothing says which row is whose";
  if (!al(a->tokens | a->requests | a->history | a->prompt_lens | a->history_lens | a->path | a->repetition | a->frequency |
          a->presence | a->bias_ids | a->bias | a->allowed, 4))
    return "adjust_logits: misaligned tables";
  return nullptr;
}

constexpr int kLogitSmem = kLogitCountBytes + kLogitMaxBias * 8;

template <class Tin, class Tout>
static cudaError_t launch_logits(const vdc_adjust_logits_args* a, vdc_status* status, cudaStream_t stream) {
  const bool is_short = (int64_t)a->L + a->path_n <= kLogitShort;
  // a tile to a CTA; where that leaves SMs idle, more CTAs, of 2048 tokens at least
  int parts = (a->vocab + 8 + kLogitCountBytes / 2 - 1) / (kLogitCountBytes / 2);
  if (parts > 8) parts = 8;
  while (parts < 8 && (int64_t)a->rows * parts < 2 * VDC_MAX_SMS && a->vocab > parts * 2048) ++parts;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a->rows * parts));
  cfg.blockDim = dim3(kLogitThreads);
  cfg.dynamicSmemBytes = kLogitCountBytes + a->n_bias * 8;
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)parts;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return is_short ? cudaLaunchKernelEx(&cfg, adjust_logits<Tin, Tout, uint16_t>, *a, parts, status)
                  : cudaLaunchKernelEx(&cfg, adjust_logits<Tin, Tout, uint32_t>, *a, parts, status);
}

extern "C" cudaError_t vdc_adjust_logits_launch(const vdc_adjust_logits_args* a, vdc_status* status, cudaStream_t stream) {
  if (a->type == 0) return launch_logits<float, float>(a, status, stream);
  if (a->type == 1)
    return a->out_type ? launch_logits<__nv_bfloat16, __nv_bfloat16>(a, status, stream) : launch_logits<__nv_bfloat16, float>(a, status, stream);
  return a->out_type ? launch_logits<__half, __half>(a, status, stream) : launch_logits<__half, float>(a, status, stream);
}

template <class Tin, class Tout>
static cudaError_t prepare_logits() {
  const void* both[] = {(const void*)adjust_logits<Tin, Tout, uint16_t>, (const void*)adjust_logits<Tin, Tout, uint32_t>};
  for (const void* f : both)
    if (cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kLogitSmem)) return e;
  return cudaSuccess;
}
extern "C" cudaError_t vdc_adjust_logits_prepare() {
  cudaError_t e = prepare_logits<float, float>();
  if (e == cudaSuccess) e = prepare_logits<__nv_bfloat16, __nv_bfloat16>();
  if (e == cudaSuccess) e = prepare_logits<__nv_bfloat16, float>();
  if (e == cudaSuccess) e = prepare_logits<__half, __half>();
  if (e == cudaSuccess) e = prepare_logits<__half, float>();
  return e;
}
