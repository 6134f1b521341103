// Keys and values of a step's tokens into the 8-bit cache (the formats: cache8.cuh).
//
// A row takes hd / 8 lanes, 16 bytes (8 bfloat16) each, so a warp holds one, two or four rows; the row's maximum is an integer
// maximum over the magnitudes' bits (infinities and NaN left out: they become NaN codes and the rest of their row keeps
// its scale).  With `rounded` the values as they are kept go out as bfloat16 rows [k | v] too: a prompt's own attention then
// sees the keys that the single tokens behind it will see.
// 2 bytes read and 1 written a value (5 in all with the rounded rows).  14,334 tokens of 16 kv heads of 128 with the rounded rows, the
// last 4,096 rows of each prompt kept: 59.7 us, 4.5 TB/s, bound by issue (75% of the slots; a value goes to its code and back); 2,048
// tokens of 4 heads of 256 7.8 us; the 8 tokens of a decode step 2.4 us, a launch and its chain of loads.
#include "cache8.cuh"

namespace {

constexpr int S8_THREADS = 256;
// Blocks of one row a thread from which on a thread takes two, and four.  8 tokens of 4 heads of 256: 2.4 us with one row, 3.0 with
// two; 2,048 tokens with the rounded rows: 8.6, 7.8 and 10.9; 14,334 tokens of 16 heads of 128: 78.7, 65.1 and 59.7.
constexpr int S8_TWO = 4 * 148, S8_FOUR = 48 * 148;

struct Store8Args {
  const __nv_bfloat16* qkv;
  long long ld;
  __nv_bfloat16* rounded;      // null: not wanted
  long long rounded_ld;
  const int *positions, *seq_of_token, *slots, *len_after, *page_table;
  int max_pages, T, nq, nkv, ring_rows, keep;
  long long n_pages;
  uint8_t *k, *v, *k_exp, *v_exp;
  int n_seqs;
  uint32_t by_token;           // 2^32 / (2 nkv), rounded up: x / (2 nkv) is the high word of x times it (x below 2^16)
};

// A thread takes U rows' pieces, S8_THREADS apart in the block's run of them: their loads go out together, before the block's first
// threads work out where its tokens' rows go (a chain of four loads a token).
template <int HD, int U>
__global__ void __launch_bounds__(S8_THREADS) store_kv8_kernel(Store8Args a) {
  // (the attention behind a decode step's store reads all pages but the new tokens' before it waits for this kernel: more tokens than
  // sequences fill earlier pages too, and it may not start before they are there)
  if (a.T <= a.n_seqs) pdl_launch_dependents();
  pdl_wait();
  constexpr int LANES = HD / 8, ROWS = S8_THREADS / LANES;       // rows that the block takes at a time
  __shared__ long long row_s[U * ROWS / 2 + 2];                  // the block's tokens' rows of a page's first head (-1: not stored)
  const int per_token = 2 * a.nkv;                               // rows of a token: its keys, then its values
  const long long total = (long long)a.T * per_token, row0 = (long long)blockIdx.x * (U * ROWS);
  const int token0 = (int)(row0 / per_token), first = (int)(row0 - (long long)token0 * per_token);      // (first: row0's place in its token)
  const int n_rows = (int)min((long long)(U * ROWS), total - row0);
  const int lr = threadIdx.x / LANES, l = threadIdx.x % LANES;
  uint4 w[U];
  if (a.rounded != nullptr) {                                    // (else only what is stored is read)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = first + u * ROWS + lr, tok = (int)__umulhi((uint32_t)x, a.by_token);
      w[u] = make_uint4(0u, 0u, 0u, 0u);
      if (u * ROWS + lr < n_rows)
        w[u] = *reinterpret_cast<const uint4*>(a.qkv + (size_t)(token0 + tok) * a.ld + (size_t)(a.nq + x - tok * per_token) * HD + l * 8);
    }
  }
  const int n_tokens = (first + n_rows - 1) / per_token + 1;
  for (int i = threadIdx.x; i < n_tokens; i += S8_THREADS) {
    const int t = token0 + i, s = a.seq_of_token[t], pos = a.positions[t], slot = a.slots[s];
    long long row = -1;
    if (slot >= 0 && af_cache_stores(pos, a.len_after[s], a.ring_rows, a.keep)) {
      const int cr = af_cache_row(pos, a.ring_rows, a.keep), entry = cr / AF_PAGE;
      const bool inside = pos >= 0 && entry < a.max_pages;
      const int page = AF_INDEX_OK(inside, pos) && inside ? a.page_table[(size_t)slot * a.max_pages + entry] : -1;
      if (AF_INDEX_OK(page >= 0 && page < a.n_pages, page) && page >= 0 && page < a.n_pages)      // (a bad page is not written)
        row = (long long)page * a.nkv * AF_PAGE + cr % AF_PAGE;
    }
    row_s[i] = row;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool live = u * ROWS + lr < n_rows;
    const int x = first + u * ROWS + lr, tok = live ? (int)__umulhi((uint32_t)x, a.by_token) : 0, r = x - tok * per_token;
    const long long at = live ? row_s[tok] : -1;
    if (a.rounded == nullptr) {
      w[u] = make_uint4(0u, 0u, 0u, 0u);
      if (at >= 0) w[u] = *reinterpret_cast<const uint4*>(a.qkv + (size_t)(token0 + tok) * a.ld + (size_t)(a.nq + r) * HD + l * 8);
    }
    const uint32_t p[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
    // the magnitudes as whole numbers, two to a word: infinities and NaN are the largest
    const uint32_t m0 = __vmaxu2(p[0] & 0x7fff7fffu, p[1] & 0x7fff7fffu), m1 = __vmaxu2(p[2] & 0x7fff7fffu, p[3] & 0x7fff7fffu);
    const uint32_t mm = __vmaxu2(m0, m1);
    uint32_t top = max(mm & 0xffffu, mm >> 16);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool fine = top < 0x7f80u;
    if (__any_sync(0xffffffffu, !fine)) {                        // (rare: the maximum again, of the finite ones alone)
      uint32_t t2 = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = p[i] & 0x7fffu, hi = (p[i] >> 16) & 0x7fffu;
        t2 = max(t2, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) t2 = max(t2, __shfl_xor_sync(0xffffffffu, t2, o));
      top = t2;
    }
    const int e = c8_exponent(top << 16);
    const float inv = c8_pow2(-e), s = c8_pow2(e);
    uint32_t codes[2];
    uint32_t back[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f = __uint_as_float(p[i] << 16) * inv, g = __uint_as_float(p[i] & 0xffff0000u) * inv;
      if (!fine) {                                               // (an infinity would be taken for the largest code)
        f = isfinite(f) ? f : __uint_as_float(0x7fc00000u);
        g = isfinite(g) ? g : __uint_as_float(0x7fc00000u);
      }
      const uint32_t c = c8_pack2(f, g);
      if (i & 1) codes[i >> 1] |= c << 16; else codes[i >> 1] = c;
      if (a.rounded != nullptr) {
        const uint32_t h = c8_half2(c);
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
        const __nv_bfloat162 b = __floats2bfloat162_rn(v.x * s, v.y * s);
        back[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
    if (at >= 0) {
      const bool key = r < a.nkv;
      const size_t row = (size_t)at + (size_t)(key ? r : r - a.nkv) * AF_PAGE;
      *reinterpret_cast<uint2*>((key ? a.k : a.v) + row * HD + l * 8) = make_uint2(codes[0], codes[1]);
      if (l == 0) (key ? a.k_exp : a.v_exp)[row] = (uint8_t)(e + 127);
    }
    if (live && a.rounded != nullptr)
      *reinterpret_cast<uint4*>(a.rounded + (size_t)(token0 + tok) * a.rounded_ld + (size_t)r * HD + l * 8) =
          make_uint4(back[0], back[1], back[2], back[3]);
  }
}

template <int HD, int U>
int launch_store8(const Store8Args& a, cudaStream_t stream) {
  constexpr int ROWS = U * (S8_THREADS / (HD / 8));
  const long long blocks = ((long long)a.T * 2 * a.nkv + ROWS - 1) / ROWS;
  AF_REQUIRE(blocks < (1ll << 31), "af_store_kv8: %d tokens of %d kv heads", a.T, a.nkv);
  af_launch(store_kv8_kernel<HD, U>, dim3((unsigned)blocks), dim3(S8_THREADS), 0, stream, a);
  AF_CHECK_LAUNCH("af_store_kv8");
}

template <int HD>
int launch_store8(const Store8Args& a, cudaStream_t stream) {
  const long long blocks = (long long)a.T * 2 * a.nkv / (S8_THREADS / (HD / 8));
  if (blocks < S8_TWO) return launch_store8<HD, 1>(a, stream);
  return blocks < S8_FOUR ? launch_store8<HD, 2>(a, stream) : launch_store8<HD, 4>(a, stream);
}

}  // namespace

// 1 when the 8-bit cache takes this head size.
AF_EXPORT int af_cache8_supported(int hd) { return hd == 64 || hd == 128 || hd == 256 ? 1 : 0; }

// What af_store_kv8 is given, as one block of 64-bit words.
struct AfStore8 {
  const void *qkv, *rounded, *positions, *seq_of_token, *slots, *len_after, *page_table, *k, *v, *k_exp, *v_exp;
  cudaStream_t stream;
  long long ld, rounded_ld, n_pages, max_pages, ring_rows, keep, T, nq, nkv, hd, n_seqs;
};

// The k and v heads of the packed bfloat16 rows [q | k | v] (T of them, ld elements apart) into the 8-bit pages of their
// sequences; `rounded` (null, or rows [k | v], rounded_ld elements apart): the values as they are kept.
AF_EXPORT int af_store_kv8(const AfStore8* c) {
  if (c->T == 0) return 0;
  AF_REQUIRE(c->T > 0 && c->T < (1ll << 31) && c->nq > 0 && c->nkv > 0 && c->nkv < (1 << 14), "af_store_kv8: %lld tokens, %lld heads, %lld kv heads", c->T, c->nq, c->nkv);
  AF_REQUIRE(af_cache8_supported((int)c->hd), "af_store_kv8: head_dim %lld (takes 64, 128, 256)", c->hd);
  AF_REQUIRE(c->ring_rows >= 0 && c->ring_rows % AF_PAGE == 0 && c->keep >= 0 && c->max_pages > 0 && c->n_pages > 0,
             "af_store_kv8: ring rows %lld, %lld kept, %lld page entries", c->ring_rows, c->keep, c->max_pages);
  AF_REQUIRE(c->ld % 8 == 0 && c->rounded_ld % 8 == 0 &&
                 (((uintptr_t)c->qkv | (uintptr_t)c->rounded | (uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0,
             "af_store_kv8: rows must be 16-byte aligned");
  Store8Args a{(const __nv_bfloat16*)c->qkv, c->ld, (__nv_bfloat16*)c->rounded, c->rounded_ld, (const int*)c->positions,
               (const int*)c->seq_of_token, (const int*)c->slots, (const int*)c->len_after, (const int*)c->page_table, (int)c->max_pages,
               (int)c->T, (int)c->nq, (int)c->nkv, (int)c->ring_rows, (int)c->keep, c->n_pages, (uint8_t*)c->k, (uint8_t*)c->v,
               (uint8_t*)c->k_exp, (uint8_t*)c->v_exp, (int)c->n_seqs, (uint32_t)(((1ull << 32) + 2 * c->nkv - 1) / (2 * c->nkv))};
  if (c->hd == 64) return launch_store8<64>(a, c->stream);
  if (c->hd == 128) return launch_store8<128>(a, c->stream);
  return launch_store8<256>(a, c->stream);
}
