// Attention of drafted tokens over a paged cache.  Shapes, masks and errors: include/vdcores.h.
//
// A warp per query row: running maximum and sum of the softmax over the sequence's rows, in fp32, four values of a head to a lane.
#include "mk_stage.cuh"

namespace vdc {
namespace {

constexpr int D = VDC_HEAD_DIM, PAGE = VDC_KV_PAGE, kWarps = 8;

template <bool kF8>
__device__ __forceinline__ float4 stored4(uint64_t page, uint64_t scale, int row, int lane) {
  if constexpr (kF8) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(page + row * D + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4);
    const float s = reinterpret_cast<const float*>(scale)[row];
    const float2 lo = e4m3x2_to_float2(w & 0xFFFFu), hi = e4m3x2_to_float2(w >> 16);
    return make_float4(lo.x * s, lo.y * s, hi.x * s, hi.y * s);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(page + row * 2 * D + (((lane >> 1) ^ (row & 7)) << 4) + (lane & 1) * 8);
    return make_float4(bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y));
  }
}

template <bool kF8>
__global__ void __launch_bounds__(kWarps * 32) tree_attention(const vdc_tree_attention_args a, vdc_status* status) {
  const vdc_cache& c = a.cache;
  const int lane = threadIdx.x & 31, rows = a.T * a.group;
  const int r = blockIdx.x * kWarps + (threadIdx.x >> 5), head = blockIdx.y, b = blockIdx.z;
  if (r >= rows) return;
  const int t = r / a.group, g = r % a.group;
  const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + b * a.q_b + t * a.q_t + head * a.q_kv + g * a.q_g;
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.out) + b * a.o_b + t * a.o_t + head * a.o_kv + g * a.o_g;
  const int* pages = reinterpret_cast<const int*>(a.pages) + b * a.pages_b;
  const long long* mask = reinterpret_cast<const long long*>(a.mask) + b * a.mask_b + t * a.mask_t;
  const int ctx = reinterpret_cast<const int*>(a.lengths)[b];
  const int live = a.counts ? max(0, min(a.T, reinterpret_cast<const int*>(a.counts)[b])) : a.T;
  int64_t keys = (int64_t)ctx + live;
  if (ctx < 0 || keys > (int64_t)a.max_pages * PAGE) {
    if (lane == 0) report(status, VDC_ERR_RANGE, VDC_TREE_ATTENTION_KIND, 0, b, ctx);
    keys = 0;
  }
  if (t >= live) keys = 0;
  float4 qv, acc = make_float4(0, 0, 0, 0);
  {
    const uint2 w = *reinterpret_cast<const uint2*>(q + lane * 4);
    qv = make_float4(bf_lo(w.x) * a.scale, bf_hi(w.x) * a.scale, bf_lo(w.y) * a.scale, bf_hi(w.y) * a.scale);
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t at = 0; at < keys; ++at) {
    const int p = pages[at / PAGE], row = (int)(at % PAGE);
    if (p < 0 || p >= c.n_pages) {
      if (lane == 0) report(status, VDC_ERR_RANGE, VDC_TREE_ATTENTION_KIND, 1, b, p);
      m = -INFINITY, l = 0.f, acc = make_float4(0, 0, 0, 0);
      break;
    }
    if (at >= ctx) {
      const int j = (int)(at - ctx);
      if (!(a.mask ? (mask[j >> 6] >> (j & 63)) & 1 : j <= t)) continue;
    }
    const float4 k = stored4<kF8>(c.k + p * c.k_page + head * c.k_head, c.k_scale + p * c.ks_page + head * c.ks_head, row, lane);
    const float4 v = stored4<kF8>(c.v + p * c.v_page + head * c.v_head, c.v_scale + p * c.vs_page + head * c.vs_head, row, lane);
    const float s = warp_sum(qv.x * k.x + qv.y * k.y + qv.z * k.z + qv.w * k.w);
    const float m2 = fmaxf(m, s), f = expf(m - m2), e = expf(s - m2);
    m = m2;
    l = l * f + e;
    acc = make_float4(acc.x * f + e * v.x, acc.y * f + e * v.y, acc.z * f + e * v.z, acc.w * f + e * v.w);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(o + lane * 4) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

}  // namespace
}  // namespace vdc

using namespace vdc;

extern "C" const char* vdc_cache_refuses(const vdc_cache* c, int max_pages);

extern "C" const char* vdc_tree_attention_refuses(const vdc_tree_attention_args* a, bool pointers) {
  auto al = [](uint64_t p, int n) { return p % n == 0; };
  if (a->B < 1 || a->T < 1 || a->T > 4096 || a->group < 1 || a->group > 128 || a->B > 65535) return "tree_attention: tokens or heads out of range";
  if (a->words * 64 < a->T) return "tree_attention: the mask has fewer bits than there are tokens";
  if (!pointers) return nullptr;
  if (const char* why = vdc_cache_refuses(&a->cache, a->max_pages)) return why;
  if (!a->q || !a->out || !al(a->q | a->out, 16)) return "tree_attention: null or misaligned rows";
  if (!al(a->q_b | a->q_t | a->q_kv | a->q_g | a->o_b | a->o_t | a->o_kv | a->o_g, 8)) return "tree_attention: row strides must be multiples of 8";
  if (!a->pages || !a->lengths || !al(a->pages | a->lengths | a->counts, 4) || !al(a->mask, 8)) return "tree_attention: null or misaligned tables";
  return nullptr;
}

extern "C" long long vdc_tree_attention_bytes(const vdc_tree_attention_args*) { return 0; }

extern "C" cudaError_t vdc_tree_attention_prepare() { return cudaSuccess; }

extern "C" cudaError_t vdc_tree_attention_launch(const vdc_tree_attention_args* a, int, vdc_status* status, uint64_t, cudaStream_t stream) {
  const dim3 grid((a->T * a->group + kWarps - 1) / kWarps, a->cache.n_kv, a->B);
  if (a->cache.kind) tree_attention<true><<<grid, kWarps * 32, 0, stream>>>(*a, status);
  else tree_attention<false><<<grid, kWarps * 32, 0, stream>>>(*a, status);
  return cudaGetLastError();
}
