// Keys and values of a step's tokens into the 8-bit cache (the formats: cache8.cuh).
//
// A row takes hd / 8 lanes, 16 bytes (8 bfloat16) each, so a warp holds one, two or four rows; the row's maximum is an integer
// maximum over the magnitudes' bits (infinities and NaN left out: they become NaN codes and the rest of their row keeps
// its scale).  With `rounded` the values as they are kept go out as bfloat16 rows [k | v] too: a prompt's own attention then
// sees the keys that the single tokens behind it will see.
// Bound by the bytes: 2 read and 1 written a value (5 in all with the rounded rows).
#include "cache8.cuh"

namespace {

constexpr int S8_THREADS = 256;

struct Store8Args {
  const __nv_bfloat16* qkv;
  long long ld;
  __nv_bfloat16* rounded;      // null: not wanted
  long long rounded_ld;
  const int *positions, *seq_of_token, *slots, *len_after, *page_table;
  int max_pages, T, nq, nkv, ring_rows, keep;
  long long n_pages;
  uint8_t *k, *v, *k_exp, *v_exp;
};

template <int HD>
__global__ void __launch_bounds__(S8_THREADS) store_kv8_kernel(Store8Args a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int LANES = HD / 8;
  const long long item = ((long long)blockIdx.x * S8_THREADS + threadIdx.x) / LANES;
  const int l = threadIdx.x % LANES;
  const int per_token = 2 * a.nkv;                       // rows of a token: its keys, then its values
  const bool live = item < (long long)a.T * per_token;
  const int t = live ? (int)(item / per_token) : 0, r = live ? (int)(item - (long long)t * per_token) : 0;
  // where it goes
  bool stores = false;
  size_t row = 0;
  if (live) {
    const int s = a.seq_of_token[t], slot = a.slots[s], pos = a.positions[t];
    if (slot >= 0 && af_cache_stores(pos, a.len_after[s], a.ring_rows, a.keep)) {
      const int cr = af_cache_row(pos, a.ring_rows, a.keep), entry = cr / AF_PAGE;
      const int page = AF_INDEX_OK(entry < a.max_pages, entry) && entry < a.max_pages ? a.page_table[(size_t)slot * a.max_pages + entry] : -1;
      stores = AF_INDEX_OK(page >= 0 && page < a.n_pages, page) && page >= 0 && page < a.n_pages;      // (a bad page is not written)
      row = stores ? ((size_t)page * a.nkv + (r < a.nkv ? r : r - a.nkv)) * AF_PAGE + cr % AF_PAGE : 0;
    }
  }
  const bool reads = stores || (live && a.rounded != nullptr);
  uint4 w = make_uint4(0u, 0u, 0u, 0u);
  if (reads) w = *reinterpret_cast<const uint4*>(a.qkv + (size_t)t * a.ld + (size_t)(a.nq + r) * HD + l * 8);
  const uint32_t p[4] = {w.x, w.y, w.z, w.w};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = (p[i] & 0x7fffu) << 16, hi = p[i] & 0x7fff0000u;
    top = max(top, lo < 0x7f800000u ? lo : 0u);
    top = max(top, hi < 0x7f800000u ? hi : 0u);
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int e = c8_exponent(top);
  const float inv = c8_pow2(-e);
  uint32_t codes[2];
  uint32_t back[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = __uint_as_float(p[i] << 16), y = __uint_as_float(p[i] & 0xffff0000u);
    x = isfinite(x) ? x * inv : __uint_as_float(0x7fc00000u);
    y = isfinite(y) ? y * inv : __uint_as_float(0x7fc00000u);
    const uint32_t c = c8_pack2(x, y);
    if (i & 1) codes[i >> 1] |= c << 16; else codes[i >> 1] = c;
    if (a.rounded != nullptr) {
      const uint32_t h = c8_half2(c);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      const float s = c8_pow2(e);
      const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * s, f.y * s);
      back[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  if (stores) {
    uint8_t* dst = r < a.nkv ? a.k : a.v;
    *reinterpret_cast<uint2*>(dst + row * HD + l * 8) = make_uint2(codes[0], codes[1]);
    if (l == 0) (r < a.nkv ? a.k_exp : a.v_exp)[row] = (uint8_t)(e + 127);
  }
  if (live && a.rounded != nullptr)
    *reinterpret_cast<uint4*>(a.rounded + (size_t)t * a.rounded_ld + (size_t)r * HD + l * 8) = make_uint4(back[0], back[1], back[2], back[3]);
}

template <int HD>
int launch_store8(const Store8Args& a, cudaStream_t stream) {
  const long long blocks = ((long long)a.T * 2 * a.nkv * (HD / 8) + S8_THREADS - 1) / S8_THREADS;
  AF_REQUIRE(blocks < (1ll << 31), "af_store_kv8: %d tokens of %d kv heads", a.T, a.nkv);
  af_launch(store_kv8_kernel<HD>, dim3((unsigned)blocks), dim3(S8_THREADS), 0, stream, a);
  AF_CHECK_LAUNCH("af_store_kv8");
}

}  // namespace

// 1 when the 8-bit cache takes this head size.
AF_EXPORT int af_cache8_supported(int hd) { return hd == 64 || hd == 128 || hd == 256 ? 1 : 0; }

// What af_store_kv8 is given, as one block of 64-bit words.
struct AfStore8 {
  const void *qkv, *rounded, *positions, *seq_of_token, *slots, *len_after, *page_table, *k, *v, *k_exp, *v_exp;
  cudaStream_t stream;
  long long ld, rounded_ld, n_pages, max_pages, ring_rows, keep, T, nq, nkv, hd;
};

// The k and v heads of the packed bfloat16 rows [q | k | v] (T of them, ld elements apart) into the 8-bit pages of their
// sequences; `rounded` (null, or rows [k | v], rounded_ld elements apart): the values as they are kept.
AF_EXPORT int af_store_kv8(const AfStore8* c) {
  if (c->T == 0) return 0;
  AF_REQUIRE(c->T > 0 && c->T < (1ll << 31) && c->nq > 0 && c->nkv > 0, "af_store_kv8: %lld tokens, %lld heads, %lld kv heads", c->T, c->nq, c->nkv);
  AF_REQUIRE(af_cache8_supported((int)c->hd), "af_store_kv8: head_dim %lld (takes 64, 128, 256)", c->hd);
  AF_REQUIRE(c->ring_rows >= 0 && c->ring_rows % AF_PAGE == 0 && c->keep >= 0 && c->max_pages > 0 && c->n_pages > 0,
             "af_store_kv8: ring rows %lld, %lld kept, %lld page entries", c->ring_rows, c->keep, c->max_pages);
  AF_REQUIRE(c->ld % 8 == 0 && c->rounded_ld % 8 == 0 &&
                 (((uintptr_t)c->qkv | (uintptr_t)c->rounded | (uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0,
             "af_store_kv8: rows must be 16-byte aligned");
  Store8Args a{(const __nv_bfloat16*)c->qkv, c->ld, (__nv_bfloat16*)c->rounded, c->rounded_ld, (const int*)c->positions,
               (const int*)c->seq_of_token, (const int*)c->slots, (const int*)c->len_after, (const int*)c->page_table, (int)c->max_pages,
               (int)c->T, (int)c->nq, (int)c->nkv, (int)c->ring_rows, (int)c->keep, c->n_pages, (uint8_t*)c->k, (uint8_t*)c->v,
               (uint8_t*)c->k_exp, (uint8_t*)c->v_exp};
  if (c->hd == 64) return launch_store8<64>(a, c->stream);
  if (c->hd == 128) return launch_store8<128>(a, c->stream);
  return launch_store8<256>(a, c->stream);
}
