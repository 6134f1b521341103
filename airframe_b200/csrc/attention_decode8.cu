// Decode attention over the 8-bit cache (cache8.cuh): one new token per sequence.
#include "cache8.cuh"

namespace {

struct Decode8Args {
  __nv_bfloat16* out;
  long long out_stride;
  const __nv_bfloat16* q;
  long long q_stride;
  const uint8_t *k, *v, *k_exp, *v_exp;
  const int *page_table, *slots, *lens;
  int max_pages, nq, nkv;
  float scale, cap;
  int window, keep, ring_rows;
  const float* sinks;
};

// A block a (sequence, head), a warp every fourth key, online softmax per warp, joined at the end.
template <int HD>
__global__ void __launch_bounds__(128) decode8_kernel(Decode8Args a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int E = HD / 32;
  __shared__ float o_s[4][HD], ml_s[4][2];
  const int b = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = a.slots[b], len = slot >= 0 ? a.lens[b] : 0, kvh = h / (a.nq / a.nkv);
  __nv_bfloat16* dst = a.out + (size_t)b * a.out_stride + (size_t)h * HD;
  if (len <= 0) {
    for (int d = threadIdx.x; d < HD; d += 128) dst[d] = __float2bfloat16_rn(0.f);
    return;
  }
  const int pos = len - 1;
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : (a.window < 0 ? pos - pos % (-a.window) : 0);
  const int kept = min(a.keep, lo);
  float q[E], o[E], m = -INFINITY, l = 0.f;
  for (int i = 0; i < E; ++i) q[i] = to_f32(a.q[(size_t)b * a.q_stride + (size_t)h * HD + lane * E + i]), o[i] = 0.f;
  for (int i = warp; i < kept + pos + 1 - lo; i += 4) {
    const int j = i < kept ? i : lo + i - kept;
    const int row = af_cache_row(j, a.ring_rows, a.keep);
    const int page = a.page_table[(size_t)slot * a.max_pages + row / AF_PAGE];
    if (page < 0) continue;
    const size_t at = ((size_t)page * a.nkv + kvh) * AF_PAGE + row % AF_PAGE;
    float s = 0.f;
    for (int e = 0; e < E; ++e) {
      __nv_fp8_e4m3 c;
      c.__x = a.k[at * HD + lane * E + e];
      s += q[e] * (float)c;
    }
    s = softcap_f32(warp_sum(s) * ldexpf(1.f, (int)a.k_exp[at] - 127) * a.scale, a.cap);
    const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
    const float pv = p * ldexpf(1.f, (int)a.v_exp[at] - 127);
    for (int e = 0; e < E; ++e) {
      __nv_fp8_e4m3 c;
      c.__x = a.v[at * HD + lane * E + e];
      o[e] = o[e] * f + pv * (float)c;
    }
    l = l * f + p, m = mn;
  }
  for (int e = 0; e < E; ++e) o_s[warp][lane * E + e] = o[e];
  if (lane == 0) ml_s[warp][0] = m, ml_s[warp][1] = l;
  __syncthreads();
  float M = a.sinks ? a.sinks[h] : -INFINITY;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, ml_s[w][0]);
  float L = a.sinks ? expf(a.sinks[h] - M) : 0.f;
  for (int w = 0; w < 4; ++w) L += ml_s[w][1] * expf(ml_s[w][0] - M);
  for (int d = threadIdx.x; d < HD; d += 128) {
    float v = 0.f;
    for (int w = 0; w < 4; ++w) v += o_s[w][d] * expf(ml_s[w][0] - M);
    dst[d] = __float2bfloat16_rn(L == 0.f ? 0.f : v / L);
  }
}

}  // namespace

// out [batch, nq * hd] = attention of one new token per sequence over its rows of the 8-bit cache.  window > 0: the last
// `window` positions; < 0: the position's own chunk of -window; the first `keep` stay visible beside either.
AF_EXPORT int af_attn_decode8(void* out, long long out_stride, const void* q, long long q_stride, const void* k, const void* v,
                              const void* k_exp, const void* v_exp, const int* page_table, int max_pages, const int* slots,
                              const int* lens, int batch, int nq, int nkv, int hd, float scale, float cap, int window, int keep,
                              int ring_rows, const float* sinks, cudaStream_t stream) {
  if (batch == 0) return 0;
  AF_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "af_attn_decode8: heads %d, groups %d", nq, nkv);
  AF_REQUIRE(keep >= 0 && (keep == 0 || window != 0), "af_attn_decode8: %d kept tokens with window %d", keep, window);
  AF_REQUIRE(ring_rows % AF_PAGE == 0 && (ring_rows == 0 || (window != 0 && abs(window) <= ring_rows)),
             "af_attn_decode8: window %d (negative: a chunk), ring rows %d", window, ring_rows);
  Decode8Args a{(__nv_bfloat16*)out, out_stride, (const __nv_bfloat16*)q, q_stride, (const uint8_t*)k, (const uint8_t*)v,
                (const uint8_t*)k_exp, (const uint8_t*)v_exp, page_table, slots, lens, max_pages, nq, nkv, scale, cap, window, keep,
                ring_rows, sinks};
  if (hd == 64) af_launch(decode8_kernel<64>, dim3(batch, nq), dim3(128), 0, stream, a);
  else if (hd == 128) af_launch(decode8_kernel<128>, dim3(batch, nq), dim3(128), 0, stream, a);
  else if (hd == 256) af_launch(decode8_kernel<256>, dim3(batch, nq), dim3(128), 0, stream, a);
  else return af_fail(-1, "af_attn_decode8: head_dim %d (takes 64, 128, 256)", hd);
  AF_CHECK_LAUNCH("af_attn_decode8");
}
