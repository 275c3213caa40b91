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

__device__ __forceinline__ void unpack8(float (&x)[8], const uint4& v) {
  x[0] = bf_lo(v.x); x[1] = bf_hi(v.x); x[2] = bf_lo(v.y); x[3] = bf_hi(v.y);
  x[4] = bf_lo(v.z); x[5] = bf_hi(v.z); x[6] = bf_lo(v.w); x[7] = bf_hi(v.w);
}

// ------------------------------------------------------------------------- //
// rope_append: a block per token; a half-warp takes one head's row of 128 values at a time, eight values to a lane.  The token's
// cosines and sines stay in registers over its heads.  Products and sums are rounded one by one (no contraction), so that the
// codes of a row do not depend on how the compiler pairs them.
// ------------------------------------------------------------------------- //
constexpr int kAppendThreads = 256;

template <bool kF8>
__global__ void __launch_bounds__(kAppendThreads) rope_append(const vdc_rope_append_args a, vdc_status* status) {
  const int token = blockIdx.x, b = token / a.T, t = token % a.T;
  const int lane = threadIdx.x & 15, half_warp = threadIdx.x >> 4;
  const unsigned mask = 0xFFFFu << (threadIdx.x & 16);
  const vdc_cache& c = a.cache;
  const int n_q = c.n_kv * a.group, n_rows = n_q + 2 * c.n_kv;
  const int* pages = reinterpret_cast<const int*>(a.pages) + b * a.pages_b;

  const int64_t at = (int64_t)__ldg(reinterpret_cast<const int*>(a.lengths) + b) + t;
  bool live = !a.counts || t < __ldg(reinterpret_cast<const int*>(a.counts) + b);
  int64_t turn = at;
  if (a.positions) turn = __ldg(reinterpret_cast<const int*>(a.positions) + b * a.pos_b + t * a.pos_t);
  int page = 0;
  if (live) {
    page = page_of(c, pages, at, a.max_pages, status, VDC_ROPE_APPEND_KIND, b);
    if (a.rot && (turn < 0 || turn >= a.table_rows)) {
      report(status, VDC_ERR_RANGE, VDC_ROPE_APPEND_KIND, 2, b, (int)turn);
      page = -1;
    }
    live = page >= 0;
  }
  const int row = (int)(at & (PAGE - 1));

  const int h = a.rot / 2, d0 = lane * 8;
  const bool turned = live && d0 < a.rot;
  float cs[8], sn[8];
  if (turned) {
    const float* tab = reinterpret_cast<const float*>(a.table) + turn * a.rot;
    const int i0 = a.interleaved ? d0 / 2 : d0 < h ? d0 : d0 - h;
    const float4 c0 = __ldg(reinterpret_cast<const float4*>(tab + i0)), s0 = __ldg(reinterpret_cast<const float4*>(tab + h + i0));
    if (a.interleaved) {
      cs[0] = cs[1] = c0.x; cs[2] = cs[3] = c0.y; cs[4] = cs[5] = c0.z; cs[6] = cs[7] = c0.w;
      sn[0] = sn[1] = s0.x; sn[2] = sn[3] = s0.y; sn[4] = sn[5] = s0.z; sn[6] = sn[7] = s0.w;
    } else {
      const float4 c1 = __ldg(reinterpret_cast<const float4*>(tab + i0 + 4)), s1 = __ldg(reinterpret_cast<const float4*>(tab + h + i0 + 4));
      cs[0] = c0.x; cs[1] = c0.y; cs[2] = c0.z; cs[3] = c0.w; cs[4] = c1.x; cs[5] = c1.y; cs[6] = c1.z; cs[7] = c1.w;
      sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w; sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
    }
    // the first of a pair: own * cos - other * sin; the second: own * cos + other * sin
    if (a.interleaved) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) sn[j] = -sn[j];
    } else if (d0 < h) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sn[j] = -sn[j];
    }
  }
  const int partner = a.interleaved || d0 >= a.rot ? lane : d0 < h ? lane + h / 8 : lane - h / 8;

  for (int r = half_warp; r < n_rows; r += kAppendThreads / 16) {
    const int part = r < n_q ? 0 : r < n_q + c.n_kv ? 1 : 2, head = part == 0 ? r : (r - n_q) % c.n_kv;
    const __nv_bfloat16* src =
        part == 0 ? reinterpret_cast<const __nv_bfloat16*>(a.q) + b * a.q_b + t * a.q_t + (head / a.group) * a.q_kv + (head % a.group) * a.q_g
        : part == 1 ? reinterpret_cast<const __nv_bfloat16*>(a.k) + b * a.k_b + t * a.k_t + head * a.k_kv
                    : reinterpret_cast<const __nv_bfloat16*>(a.v) + b * a.v_b + t * a.v_t + head * a.v_kv;
    __nv_bfloat16* q_out = reinterpret_cast<__nv_bfloat16*>(a.out) + b * a.o_b + t * a.o_t + (head / a.group) * a.o_kv + (head % a.group) * a.o_g;
    if (!live) {
      if (part == 0) *reinterpret_cast<uint4*>(q_out + d0) = make_uint4(0, 0, 0, 0);
      continue;
    }
    float x[8];
    unpack8(x, *reinterpret_cast<const uint4*>(src + d0));
    const uint64_t norm = part == 0 ? a.q_norm : part == 1 ? a.k_norm : 0;
    if (norm) {
      float ss = 0.f, w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      const float rs = rsqrtf(ss * (1.f / D) + a.eps);
      unpack8(w, __ldg(reinterpret_cast<const uint4*>(norm) + lane));
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(__fmul_rn(x[j], rs), w[j]);
    }
    if (part < 2 && a.rot) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = a.interleaved ? x[j ^ 1] : __shfl_sync(mask, x[j], partner, 16);
      if (turned) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __fadd_rn(__fmul_rn(x[j], cs[j]), __fmul_rn(y[j], sn[j]));
      }
    }
    if (part == 0) {
      *reinterpret_cast<uint4*>(q_out + d0) = pack8(x);
      continue;
    }
    uint8_t* dst = reinterpret_cast<uint8_t*>(part == 1 ? c.k : c.v) + page * (part == 1 ? c.k_page : c.v_page) +
                   head * (part == 1 ? c.k_head : c.v_head) + row * (kF8 ? D : 2 * D) + lane_place<kF8>(row, lane);
    if constexpr (!kF8) {
      *reinterpret_cast<uint4*>(dst) = pack8(x);
    } else {
      // magnitudes compare as whole numbers, infinity above all finite ones and NaN above infinity: a row with either gets a
      // scale that says so
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
      const float most = __uint_as_float(top), scale = __fdiv_rn(most < 1e-12f ? 1e-12f : most, 448.f);
      uint32_t code[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        code[j] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[2 * j], scale), __fdiv_rn(x[2 * j + 1], scale)), __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<uint2*>(dst) = make_uint2(code[0] | code[1] << 16, code[2] | code[3] << 16);
      if (lane == 0)
        *reinterpret_cast<float*>((part == 1 ? c.k_scale + page * c.ks_page + head * c.ks_head
                                             : c.v_scale + page * c.vs_page + head * c.vs_head) + row * 4) = scale;
    }
  }
}

// ------------------------------------------------------------------------- //
// read_cache: a half-warp per row of one head, keys and values; rows are bytes in and bytes out, so memory is the bound.
// ------------------------------------------------------------------------- //
constexpr int kReadThreads = 256;

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
  const int64_t unit = (int64_t)blockIdx.x * (kReadThreads / 16) + (threadIdx.x >> 4);
  if (unit >= (int64_t)a.n * c.n_kv) return;
  const int i = (int)(unit / c.n_kv), head = (int)(unit % c.n_kv);
  const int64_t at = (int64_t)(a.start ? __ldg(reinterpret_cast<const int*>(a.start) + b) : 0) + i;
  const int64_t to = (((int64_t)b * a.n + i) * c.n_kv + head) * D + lane * 8;
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (at < __ldg(reinterpret_cast<const int*>(a.lengths) + b)) {
    const int page = page_of(c, reinterpret_cast<const int*>(a.pages) + b * a.pages_b, at, a.max_pages, status, VDC_READ_CACHE_KIND, b);
    if (page >= 0) {
      const int row = (int)(at & (PAGE - 1)), place = row * (kF8 ? D : 2 * D) + lane_place<kF8>(row, lane);
      float ks = 1.f, vs = 1.f;
      if constexpr (kF8) {
        ks = __ldg(reinterpret_cast<const float*>(c.k_scale + page * c.ks_page + head * c.ks_head) + row);
        vs = __ldg(reinterpret_cast<const float*>(c.v_scale + page * c.vs_page + head * c.vs_head) + row);
      }
      k = stored8<kF8>(reinterpret_cast<const uint8_t*>(c.k) + page * c.k_page + head * c.k_head + place, ks);
      v = stored8<kF8>(reinterpret_cast<const uint8_t*>(c.v) + page * c.v_page + head * c.v_head + place, vs);
    }
  }
  *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.k_out) + to) = k;
  *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.v_out) + to) = v;
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
  const int grid = a->B * a->T;
  if (a->cache.kind) rope_append<true><<<grid, kAppendThreads, 0, stream>>>(*a, status);
  else rope_append<false><<<grid, kAppendThreads, 0, stream>>>(*a, status);
  return cudaGetLastError();
}

extern "C" const char* vdc_read_cache_refuses(const vdc_read_cache_args* a) {
  if (const char* why = check_cache(a->cache, a->max_pages)) return why;
  if (a->B < 1 || a->B > 65535 || a->n < 1) return "read_cache: sequences or rows out of range";
  if (!a->pages || !a->lengths || !al(a->pages | a->lengths | a->start, 4)) return "read_cache: null or misaligned tables";
  return a->k_out && a->v_out && al(a->k_out | a->v_out, 16) ? nullptr : "read_cache: null or misaligned rows";
}

extern "C" cudaError_t vdc_read_cache_launch(const vdc_read_cache_args* a, vdc_status* status, cudaStream_t stream) {
  const int64_t units = (int64_t)a->n * a->cache.n_kv, per = kReadThreads / 16;
  const dim3 grid((unsigned)((units + per - 1) / per), (unsigned)a->B);
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
