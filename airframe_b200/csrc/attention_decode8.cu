// Decode attention over the 8-bit cache (cache8.cuh): one new token per sequence, bound by the bytes of codes it reads (every
// byte is read once; half of the 16-bit cache's).
//
// The work is cut as for the 16-bit cache (decode_split.cuh): one block an SM, units of a (sequence, kv head), their pages in
// equal splits or runs, by the step's plan.  A page's codes come in by TMA (swizzled) and its exponents by two bulk copies,
// through a ring of shared-memory stages; groups of four warps take the pages in turn, a warp 16 of a page's 64 keys.
//
// Products.  With a query group of few heads the keys are the rows of the m16n8k16 tiles and the heads their 8 columns:
//   S^T = K Q^T (16 keys x 8 heads), O^T += V^T P^T (16 dims x 8 heads)
// which wastes nothing for groups of up to 8 heads (16 rows of heads would waste half of both the instructions and the
// accumulators).  Codes become halves (cvt, exact) on their way from shared memory into the fragments, so the two factors of
// a row never touch its elements: 2^ek multiplies the key's score, and 2^ev goes into the key's weight.  The order of the
// contracted indices is free, so a lane takes 16 consecutive bytes of a row as four steps' fragments: K needs no ldmatrix, and
// V (whose fragments pair two keys) a byte permutation of four rows.  P's fragments are transposed by movmatrix.
//   The key with row r of a tile is r's permuted one (d8_perm), which keeps the 16-byte loads of both free of bank conflicts.
//
// Numbers.  Halves hold 11 bits (bfloat16: 8) but little range.  A head's query is brought to [2^14, 2^15) by a power of two
// (exact down to 2^-29 of its largest element; 2^-39 of it is the most that is lost below).  A weight's half holds
// 2^(s + ev) relative to the largest such sum of the warp's keys so far, times 2^6, which leaves 2^-20 of the largest weight a
// normal half; the softmax's own sum is kept in 32 bits against the scores' maximum.  Both references move only when one is
// passed by more than 8 (base 2).  The softcap is tanh by the exponential, exact to 2^-22 of the cap (tanh.approx: 2^-11).
#include "airframe_b200.h"
#include "cache8.cuh"
#include "decode_split.cuh"

namespace {

constexpr float D8_NONE = -3.0e38f;      // a reference before the first key (finite: exp2(-inf - it) is 0)
constexpr float D8_MOVES = 8.f;          // a reference moves when it is passed by more than this
constexpr float D8_SHIFT = 6.f;          // weights are kept times 2^6

template <int HD, int NT>
struct D8 {
  // (the accumulators of 16 heads of 256 take 128 registers, those of 8 heads 64 beside 32 of queries: fewer warps)
  static constexpr int THREADS = HD * NT == 512 ? 256 : (HD * NT == 256 ? 384 : 512);
  static constexpr int WARPS = THREADS / 32;
  // keys of a piece: half a page where heads are large, so that all warps have pieces in shared memory
  static constexpr int KEYS = HD == 256 ? 32 : 64, PER_PAGE = AF_PAGE / KEYS, TILES = KEYS / 16;
  static constexpr int AT_ONCE = NT == 2 && TILES == 4 ? 2 : TILES;      // tiles of a piece that are worked together
  static constexpr int CODES = KEYS * HD;                                // bytes of a piece's keys, and of its values
  static constexpr int SUB = KEYS * 128;                                 // bytes of a sub-tile of 128 dims
  static constexpr int STAGES = HD == 64 ? 16 : 12;
  // barriers: a piece's must not be met by another warp's pieces (a multiple of WARPS), nor be armed before the piece in the
  // same stage was consumed (a multiple of STAGES)
  static constexpr int NBAR = HD == 64 ? 16 : (WARPS == 16 ? 48 : (WARPS == 12 ? 12 : 24));
  static constexpr int RING = STAGES * 2 * CODES;
  static constexpr int SMEM = RING + STAGES * 2 * KEYS + 1024;
  static_assert(NBAR % WARPS == 0 && NBAR % STAGES == 0, "barriers");
  static_assert(WARPS * 8 * NT * HD * 4 <= RING, "the merge's buffer");
};

struct Decode8Args {
  const __nv_bfloat16* q;
  long long q_stride;
  const uint8_t *k_exp, *v_exp;
  long long n_pages;
  const int *page_table, *slots, *lens, *shared, *plan;
  int max_pages, nq, nkv;
  float scale, cap;
  int window, keep, ring_rows, n_splits, batch;
  float *part_o, *part_ml;
  int* err;
};

__device__ __forceinline__ int d8_perm(int r) { return (r >> 1) | ((r & 1) << 2); }

__device__ __forceinline__ void d8_mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t d8_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 d8_lds4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 d8_lds2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ int d8_lds_u8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
  return (int)v;
}
__device__ __forceinline__ void d8_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// S^T, softmax and O^T of N tiles of 16 keys (all of a piece, or one), beginning with tile `t0`.
template <int HD, int NT, int N>
struct D8Step {
  using C = D8<HD, NT>;
  // k_l, v_l, e_l: this lane's addresses of the piece's keys, values and exponents (tile 0); swap: what the odd halves' addresses
  // differ by (the swizzle); lo, hi, keep: the visible keys, counted from the piece's first
  __device__ static __forceinline__ void run(uint32_t k_l, uint32_t v_l, uint32_t ke_l, int t0, bool whole, int lo, int hi, int keep,
                                             int g, int t, bool capped, float ecap, float capl, const uint32_t (&qf)[NT][HD / 16][2],
                                             const float (&cq)[NT][2], float (&o)[HD / 16][NT][4], float (&rs)[NT][2], float (&ra)[NT][2],
                                             float (&l)[NT][2]) {
    constexpr int ROW = HD == 64 ? 64 : 128;              // bytes between rows of a sub-tile
    k_l += t0 * 16 * ROW;
    v_l += t0 * 16 * ROW;
    ke_l += t0 * 16;
    float sc[N][NT][4], wt[N][NT][4];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) sc[i][n][0] = sc[i][n][1] = sc[i][n][2] = sc[i][n][3] = 0.f;
    // ---- S^T = K Q^T
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t at = (c & 1 ? k_l ^ 64u : k_l) + (c >> 1) * C::SUB + i * 16 * ROW;
        const uint4 x = d8_lds4(at), y = d8_lds4(at + 8 * ROW);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a0, a1, a2, a3;
          c8_half4(xs[j], a0, a2);
          c8_half4(ys[j], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) d8_mma(sc[i][n], a0, a1, a2, a3, qf[n][c * 4 + j][0], qf[n][c * 4 + j][1]);
        }
      }
    }
    // ---- scale, softcap, mask; the weights' exponents; whether a reference moves
    const int kr = t0 * 16 + d8_perm(g);                  // this lane's keys: kr + 16 i, and 8 behind
    bool moves = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float ks[2], lv[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ks[h] = __uint_as_float((uint32_t)d8_lds_u8(ke_l + i * 16 + 8 * h) << 23);
        lv[h] = (float)(d8_lds_u8(ke_l + C::KEYS + i * 16 + 8 * h) - 127);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[i][n][e] *= cq[n][e & 1] * ks[e >> 1];
      if (capped) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][n][e] = capl - 2.f * capl * __fdividef(1.f, 1.f + fast_exp2(sc[i][n][e] * ecap));
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = kr + 16 * i + 8 * (e >> 1);
          const bool on = (j >= lo || j < keep) && j <= hi;
#pragma unroll
          for (int n = 0; n < NT; ++n) sc[i][n][e] = on ? sc[i][n][e] : -INFINITY;
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) wt[i][n][e] = sc[i][n][e] + lv[e >> 1];
    }
    float ms[NT][2], ma[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x = fmaxf(sc[0][n][h], sc[0][n][h + 2]), y = fmaxf(wt[0][n][h], wt[0][n][h + 2]);
#pragma unroll
        for (int i = 1; i < N; ++i) {
          x = fmaxf(x, fmaxf(sc[i][n][h], sc[i][n][h + 2]));
          y = fmaxf(y, fmaxf(wt[i][n][h], wt[i][n][h + 2]));
        }
        ms[n][h] = x, ma[n][h] = y;
        moves = moves || x > rs[n][h] + D8_MOVES || y > ra[n][h] + D8_MOVES;
      }
    if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x = ms[n][h], y = ma[n][h];
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) {
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, w));
          }
          x = fmaxf(x, rs[n][h]), y = fmaxf(y, ra[n][h]);
          l[n][h] *= fast_exp2(rs[n][h] - x);
          const float f = fast_exp2(ra[n][h] - y);
          rs[n][h] = x, ra[n][h] = y;
#pragma unroll
          for (int m = 0; m < HD / 16; ++m) o[m][n][h] *= f, o[m][n][h + 2] *= f;
        }
    }
    uint32_t pb[N][NT][2];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          l[n][e & 1] += fast_exp2(sc[i][n][e] - rs[n][e & 1]);
          w[e] = fast_exp2(wt[i][n][e] - (ra[n][e & 1] - D8_SHIFT));
        }
        const __half2 p0 = __floats2half2_rn(w[0], w[1]), p1 = __floats2half2_rn(w[2], w[3]);
        pb[i][n][0] = d8_transpose(*reinterpret_cast<const uint32_t*>(&p0));
        pb[i][n][1] = d8_transpose(*reinterpret_cast<const uint32_t*>(&p1));
      }
    // ---- O^T += V^T P^T: this lane's fragments hold the keys t, t + 4, t + 8, t + 12 of a tile
    constexpr int VW = HD == 64 ? 2 : 4;                  // words of a row that a lane takes at a time
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int c = 0; c < HD / (32 * VW); ++c) {
        uint32_t w[4][VW];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t at = (x & 1 ? v_l ^ (HD == 64 ? 32u : 64u) : v_l) + c * C::SUB + (i * 16 + 4 * x) * ROW;
          if constexpr (HD == 64) {
            const uint2 v = d8_lds2(at);
            w[x][0] = v.x, w[x][1] = v.y;
          } else {
            const uint4 v = d8_lds4(at);
            w[x][0] = v.x, w[x][1] = v.y, w[x][2] = v.z, w[x][3] = v.w;
          }
          if (!whole) {
            // (a hidden key's codes may be any bytes, NaN among them: its weight of 0 does not make them 0)
            const int j = (t0 + i) * 16 + t + 4 * x;
            if (!((j >= lo || j < keep) && j <= hi)) {
#pragma unroll
              for (int k = 0; k < VW; ++k) w[x][k] = 0u;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < VW; ++j) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t sel = u ? 0x7362u : 0x5140u;
            uint32_t a0, a1, a2, a3;
            c8_half4(__byte_perm(w[0][j], w[1][j], sel), a0, a1);
            c8_half4(__byte_perm(w[2][j], w[3][j], sel), a2, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) d8_mma(o[c * 2 * VW + 2 * j + u][n], a0, a1, a2, a3, pb[i][n][0], pb[i][n][1]);
          }
        }
      }
    }
  }
};

template <int HD, int NT>
__global__ void __launch_bounds__(D8<HD, NT>::THREADS, 1)
decode8_split_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Decode8Args a) {
  using C = D8<HD, NT>;
  constexpr int STAGES = C::STAGES, WARPS = C::WARPS, NBAR = C::NBAR, PER = C::PER_PAGE;
  constexpr int ROWS = 8 * NT;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ unsigned char d8_raw[];
  unsigned char* ring = (unsigned char*)(((uintptr_t)d8_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* exps = ring + C::RING;                        // [stage][k exponents | v exponents]
  __shared__ uint64_t full[NBAR];
  __shared__ float rs_s[WARPS][ROWS], ra_s[WARPS][ROWS], l_s[WARPS][ROWS];
  __shared__ float f_s[WARPS][ROWS], ml_s[ROWS][2];
  __shared__ int give_up_s;
  volatile int* give_up = &give_up_s;

  pdl_launch_dependents();
  const int group = a.nq / a.nkv;
  const int tiles = (group + 15) / 16, units_per_seq = a.nkv * tiles;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  if (tid == 0) {
    for (int s = 0; s < NBAR; ++s) mbar_init(&full[s], 1);
    give_up_s = 0;
    mbar_fence_init();
  }
  // what the block begins with, from the step's plan
  const int4* rec = reinterpret_cast<const int4*>(a.plan + da_plan_records_at(a.batch, units_per_seq)) +
                    (size_t)blockIdx.x * (DA_PLAN_REC / 4);
  const uint64_t keep_policy = l2_policy_keep();
  const int4 head = ld_keep_int4(reinterpret_cast<const int4*>(a.plan), keep_policy);
  const int4 r0 = ld_keep_int4(rec, keep_policy), r1 = ld_keep_int4(rec + 1, keep_policy), r2 = ld_keep_int4(rec + 2, keep_policy);
  const int4 r3 = ld_keep_int4(rec + 3, keep_policy);
  if (head.x != a.n_splits || head.y != da_plan_mark((int)gridDim.x, D8_BREAK_PAGES) || head.z != a.batch || head.w != units_per_seq) {
    if (tid == 0 && a.err) atomicExch(a.err, 1);      // (a plan made for another launch: nothing is read or written by it)
    return;
  }
  __syncthreads();
  if (r0.x < 0) {                                     // (no work; a grid without any must not end before the kernel in front)
    if (blockIdx.x == 0) pdl_wait();
    return;
  }
  int left = r1.y;

  struct Segment {
    int b, kvh, row_head0, n_rows, z, n_pages, x_begin, kept, skip, last_pp, lo, pos, y;
    const int* pt;
  };
  auto of_unit = [&](Segment& sg, int b, int y, int p_in, int pos, int slot, int shared) {
    sg.b = b;
    sg.y = y;
    sg.kvh = y / tiles;
    sg.row_head0 = sg.kvh * group + (y % tiles) * 16;
    sg.n_rows = min(16, sg.kvh * group + group - sg.row_head0);
    sg.pos = pos;
    sg.lo = da_lo(pos, a.window);
    sg.last_pp = pos / AF_PAGE;
    const DaList l = da_list(pos, a.window, a.keep, shared);
    sg.kept = l.kept, sg.skip = l.skip;
    sg.x_begin = p_in;
    sg.pt = a.page_table + (size_t)slot * a.max_pages;
  };
  auto next_unit = [&](const Segment& sg) {           // (the run cut: see attention_decode.cu)
    Segment nx;
    int b = sg.b, y = sg.y + 1;
    if (y >= units_per_seq) {
      y = 0;
      do ++b; while (b < a.batch - 1 && da_pages(a.slots, a.lens, b, a.window, a.keep, a.shared) == 0);
    }
    const int P = da_pages(a.slots, a.lens, b, a.window, a.keep, a.shared);
    nx.z = 0;
    nx.n_pages = min(P, left - D8_BREAK_PAGES);
    left -= D8_BREAK_PAGES + P;
    of_unit(nx, b, y, 0, a.lens[b] - 1, a.slots[b], a.shared != nullptr ? a.shared[b] : 0);
    return nx;
  };
  auto page_of = [&](const Segment& sg, int i) { return da_page_of(sg.kept, sg.skip, sg.x_begin + i); };
  auto safe = [&](int page) { return AF_INDEX_OK(page >= 0 && page < a.n_pages, page) && page >= 0 && page < a.n_pages ? page : 0; };
  auto page_id = [&](const Segment& sg, int i) {
    const int entry = af_cache_row(page_of(sg, i) * AF_PAGE, a.ring_rows, a.keep) / AF_PAGE;
    return AF_INDEX_OK(entry < a.max_pages, entry) && entry < a.max_pages ? safe(sg.pt[entry]) : 0;
  };
  const uint64_t read_once = l2_policy_read_once();
  // piece `half` of cache page `page`, the block's piece number ii, into its stage
  auto issue = [&](int kvh, int page, int half, int ii) {
    const int s = ii % STAGES, row = (page * a.nkv + kvh) * AF_PAGE + half * C::KEYS;
    unsigned char* st = ring + (size_t)s * 2 * C::CODES;
    uint64_t* bar = &full[ii % NBAR];
    mbar_expect_tx(bar, 2 * C::CODES + 2 * C::KEYS);
#pragma unroll
    for (int c = 0; c < (HD + 127) / 128; ++c) {
      tma_load_2d_once(st + c * C::SUB, &map_k, c * 128, row, bar, read_once);
      tma_load_2d_once(st + C::CODES + c * C::SUB, &map_v, c * 128, row, bar, read_once);
    }
    d8_bulk(exps + s * 2 * C::KEYS, a.k_exp + row, C::KEYS, bar);
    d8_bulk(exps + s * 2 * C::KEYS + C::KEYS, a.v_exp + row, C::KEYS, bar);
  };
  auto issue_from = [&](const Segment& sg, int from, int to, int ii0, bool skip_last) {      // (pieces of the segment)
    int i = from;
    int page = -1, id = 0;
    for (; i < to; ++i) {
      if (skip_last && page_of(sg, i / PER) == sg.last_pp) break;
      if (i / PER != page) page = i / PER, id = page_id(sg, page);
      issue(sg.kvh, id, i % PER, ii0 + i);
    }
    return i;
  };

  int i_base = 0;
  Segment sg;
  sg.z = r0.w;
  sg.n_pages = r0.x;
  of_unit(sg, r0.y, r0.z, r1.x, r1.z, r1.w, r3.x);
  int issued = 0;
  if (tid == 0) {
    // pages of earlier tokens are on their way before the wait for the kernel in front; the new token's waits.  The first
    // four pages' ids are in the plan.
    const int ids0[4] = {r2.x, r2.y, r2.z, r2.w};
    bool go = true;
#pragma unroll
    for (int k = 0; k < 4 * PER; ++k) {
      go = go && k < STAGES && k < sg.n_pages * PER && page_of(sg, k / PER) != sg.last_pp;
      if (go) {
        issue(sg.kvh, safe(ids0[k / PER]), k % PER, k);
        ++issued;
      }
    }
    if (issued == 4 * PER) issued = issue_from(sg, issued, min(STAGES, sg.n_pages * PER), 0, true);
  }
  pdl_wait();
  while (true) {
    const int b = sg.b, n = sg.n_pages * PER, n_rows = sg.n_rows, row_head0 = sg.row_head0;
    if (tid == 0) issued = issue_from(sg, issued, min(STAGES, n), i_base, false);

    // ---- the queries as B fragments (head g of every tile of 8), halves brought to [2^14, 2^15)
    uint32_t qf[NT][HD / 16][2];
    float cq[NT][2];                     // per column (head) of this lane: the factor of its scores
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool on = n * 8 + g < n_rows;
      const __nv_bfloat16* qr = a.q + (size_t)b * a.q_stride + (size_t)(row_head0 + n * 8 + g) * HD + t * 16;
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t* p = reinterpret_cast<const uint32_t*>(qr + c * 64 + j * 4);
          const uint32_t x = on ? p[0] : 0u, y = on ? p[1] : 0u;
          qf[n][c * 4 + j][0] = x;
          qf[n][c * 4 + j][1] = y;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w = h ? y : x, lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
            top = max(top, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
          }
        }
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // (the scaling in two steps: 2^(14 - k) alone may pass the largest power of two)
      const int k = top == 0 ? 14 : max((int)(top >> 7) - 127, -126), up = 14 - k;
      const float f1 = c8_pow2(up / 2), f2 = c8_pow2(up - up / 2);
      // cq = scale 2^-up in two steps, too
      const float cs = (a.cap > 0.f ? a.scale : a.scale * LOG2E) * c8_pow2(-(up / 2)) * c8_pow2(-(up - up / 2));
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w = qf[n][i][h];
          const __half2 v = __floats2half2_rn(__uint_as_float(w << 16) * f1 * f2, __uint_as_float(w & 0xffff0000u) * f1 * f2);
          qf[n][i][h] = *reinterpret_cast<const uint32_t*>(&v);
        }
      cq[n][0] = __shfl_sync(0xffffffffu, cs, t * 8);
      cq[n][1] = __shfl_sync(0xffffffffu, cs, t * 8 + 4);
    }
    const float ecap = a.cap > 0.f ? 2.f * LOG2E / a.cap : 0.f, capl = a.cap * LOG2E;

    float o[HD / 16][NT][4];
#pragma unroll
    for (int m = 0; m < HD / 16; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
    float rs[NT][2], ra[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) rs[n][0] = rs[n][1] = ra[n][0] = ra[n][1] = D8_NONE, l[n][0] = l[n][1] = 0.f;

    // A warp takes a piece at a time; where the pieces are fewer than the warps, a tile of 16 keys.
    const bool few = n <= STAGES && n * C::TILES <= 2 * WARPS;
    const int items = few ? n * C::TILES : n;
    // this lane's place in a piece (see D8Step)
    const int pg = d8_perm(g);
    const uint32_t k_off = HD == 64 ? pg * 64 + ((t ^ ((pg >> 1) & 3)) << 4) : pg * 128 + ((t ^ pg) << 4);
    const uint32_t v_off = C::CODES + (HD == 64 ? t * 64 + (((g >> 1) ^ (t >> 1)) << 4) + (g & 1) * 8 : t * 128 + ((pg ^ t) << 4));
    for (int x = warp; x < items; x += WARPS) {
      const int i = few ? x / C::TILES : x, ii = i_base + i, s = ii % STAGES;
      const bool refill = lane == 0 && i + STAGES < n;
      const int refill_page = refill ? page_id(sg, (i + STAGES) / PER) : 0;
      if (!mbar_wait(&full[ii % NBAR], (ii / NBAR) & 1, give_up)) break;
      const uint32_t st = smem_u32(ring) + s * 2 * C::CODES, e_l = smem_u32(exps) + s * 2 * C::KEYS + pg;
      const int base = page_of(sg, i / PER) * AF_PAGE + (i % PER) * C::KEYS;
      const int lo = sg.lo - base, hi = sg.pos - base, keep = a.keep - base;       // (visible: [lo, hi] and what is before keep)
      const bool whole = C::KEYS - 1 <= hi && (lo <= 0 || C::KEYS - 1 < keep);
      if (few)
        D8Step<HD, NT, 1>::run(st + k_off, st + v_off, e_l, x % C::TILES, whole, lo, hi, keep, g, t, a.cap > 0.f, ecap, capl, qf, cq, o, rs, ra, l);
      else
#pragma unroll 1
        for (int t0 = 0; t0 < C::TILES; t0 += C::AT_ONCE)
          D8Step<HD, NT, C::AT_ONCE>::run(st + k_off, st + v_off, e_l, t0, whole, lo, hi, keep, g, t, a.cap > 0.f, ecap, capl, qf, cq, o, rs, ra, l);
      __syncwarp();
      if (refill && !*give_up) issue(sg.kvh, refill_page, (i + STAGES) % PER, ii + STAGES);
    }
    if (*give_up && tid == 0) grace_period();
    __syncthreads();
    const bool gave_up = *give_up != 0;

    // ---- merge the warps through shared memory (the stages that the next segment's first pages do not take)
    i_base += n;
    const bool more = left > D8_BREAK_PAGES && !gave_up;
    const int buf_bytes = WARPS * n_rows * HD * 4, buf_stages = (buf_bytes + 2 * C::CODES - 1) / (2 * C::CODES);
    Segment nx = sg;
    issued = 0;
    // The buffer is `buf_stages` stages in a row (they do not wrap): those just before the next page's stage, so that all
    // others can be filled, or where these are too few the last ones, and the pages up to them can.
    const int first = i_base % STAGES;
    const int buf0 = first >= buf_stages ? first - buf_stages : STAGES - buf_stages;
    const int room = first >= buf_stages ? STAGES - buf_stages : max(0, buf0 - first);
    if (more) {
      nx = next_unit(sg);
      if (tid == 0) issued = issue_from(nx, 0, min(room, nx.n_pages * PER), i_base, false);
    }
    float* o_s = reinterpret_cast<float*>(ring + (size_t)buf0 * 2 * C::CODES);     // [warp][row][HD]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v = l[n][h];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        const int row = n * 8 + 2 * t + h;
        if (g == 0) rs_s[warp][row] = rs[n][h], ra_s[warp][row] = ra[n][h], l_s[warp][row] = v;
        if (row < n_rows) {
          float* dst = o_s + ((size_t)warp * n_rows + row) * HD;
#pragma unroll
          for (int m = 0; m < HD / 16; ++m) {
            const int d = HD == 64 ? g * 8 + m * 2 : (m >> 3) * 128 + d8_perm(g) * 16 + (m & 7) * 2;
            *reinterpret_cast<float2*>(dst + d) = make_float2(o[m][n][h], o[m][n][h + 2]);
          }
        }
      }
    __syncthreads();
    if (tid < n_rows) {
      float M = D8_NONE, L = 0.f;
      for (int w = 0; w < WARPS; ++w) M = fmaxf(M, rs_s[w][tid]);
      for (int w = 0; w < WARPS; ++w) {
        L += l_s[w][tid] * fast_exp2(rs_s[w][tid] - M);
        f_s[w][tid] = fast_exp2(ra_s[w][tid] - D8_SHIFT - M);
      }
      ml_s[tid][0] = M == D8_NONE ? -INFINITY : M;
      ml_s[tid][1] = L;
    }
    __syncthreads();
    for (int i = tid; i < n_rows * (HD / 4); i += C::THREADS) {
      const int row = i / (HD / 4), d = (i - row * (HD / 4)) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int w = 0; w < WARPS; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(o_s + ((size_t)w * n_rows + row) * HD + d);
        const float f = f_s[w][row];
        v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
      }
      const size_t pidx = ((size_t)b * a.nq + row_head0 + row) * a.n_splits + sg.z;
      *reinterpret_cast<float4*>(a.part_o + pidx * HD + d) = v;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + pidx * 2) = make_float2(ml_s[row][0], ml_s[row][1]);
    }
    if (!more) break;
    // (the buffer is one of the next segment's stages; what was read and written here by the generic proxy comes before the
    // copies that follow)
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    sg = nx;
  }
  if (tid == 0 && give_up_s && a.err) atomicExch(a.err, 1);
}

// Tensor map of the codes as a matrix of bytes [rows, HD]: boxes of a piece's rows by up to 128 bytes, swizzled.
int d8_map(CUtensorMap* map, const void* base, long long rows, int hd) {
  AfEncodeTiledFn enc = af_encode_tiled();
  if (enc == nullptr) return af_fail(-1, "the driver has no cuTensorMapEncodeTiled");
  cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)hd};
  cuuint32_t box[2] = {hd < 128 ? 64u : 128u, hd == 256 ? 32u : (cuuint32_t)AF_PAGE};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         hd < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return af_fail(-1, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return 0;
}

template <int HD, int NT>
int launch_decode8(const CUtensorMap& mk, const CUtensorMap& mv, const Decode8Args& a, int blocks, cudaStream_t stream) {
  static bool configured[AF_MAX_DEVICES] = {};
  const int dev = af_current_device();
  if (dev < 0) return -1;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(decode8_split_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, D8<HD, NT>::SMEM);
    if (e != cudaSuccess) return af_fail((int)e, "af_attn_decode8: %s", cudaGetErrorString(e));
    configured[dev] = true;
  }
  af_launch(decode8_split_kernel<HD, NT>, dim3(blocks), dim3(D8<HD, NT>::THREADS), D8<HD, NT>::SMEM, stream, mk, mv, a);
  AF_CHECK_LAUNCH("af_attn_decode8 (split)");
}

}  // namespace

// The split pass: partial results of every (sequence, head) into `scratch` (af_attn_decode_scratch(...) floats), as the
// step's `plan` (af_attn_decode_plan_kept, or the shared one) cuts the work.
int af_decode8_split(const void* q, long long q_stride, const void* k, const void* v, const void* k_exp, const void* v_exp,
                     long long n_pages, const int* page_table, int max_pages, const int* slots, const int* lens, const int* shared,
                     int batch, int nq, int nkv, int hd, float scale, float cap, int window, int keep, int ring_rows, int n_splits,
                     float* scratch, const int* plan, int* err, cudaStream_t stream) {
  AF_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "af_attn_decode8: heads %d, groups %d", nq, nkv);
  AF_REQUIRE(hd == 64 || hd == 128 || hd == 256, "af_attn_decode8: head_dim %d (takes 64, 128, 256)", hd);
  AF_REQUIRE(keep >= 0 && (keep == 0 || window != 0), "af_attn_decode8: %d kept tokens with window %d", keep, window);
  AF_REQUIRE(ring_rows >= 0 && ring_rows % AF_PAGE == 0 && (ring_rows == 0 || (window != 0 && abs(window) <= ring_rows)),
             "af_attn_decode8: window %d (negative: a chunk), ring rows %d", window, ring_rows);
  AF_REQUIRE(n_splits >= 1 && n_splits <= 65535 && scratch != nullptr && plan != nullptr && ((uintptr_t)plan & 15) == 0,
             "af_attn_decode8: splits %d, scratch and a 16-byte aligned plan", n_splits);
  AF_REQUIRE((((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_exp | (uintptr_t)v_exp | (uintptr_t)scratch) & 15) == 0,
             "af_attn_decode8: cache and scratch alignment");
  AF_REQUIRE(q_stride % 2 == 0 && ((uintptr_t)q & 3) == 0, "af_attn_decode8: queries must be 4-byte aligned");
  AF_REQUIRE(n_pages > 0 && n_pages * nkv * AF_PAGE < (1ll << 31), "af_attn_decode8: %lld cache pages", n_pages);
  const int group = nq / nkv, units_per_seq = nkv * ((group + 15) / 16);
  AF_REQUIRE(batch <= DA_MAX_BATCH && (long long)batch * (max_pages + 1 + D8_BREAK_PAGES) * units_per_seq < (1ll << 31),
             "af_attn_decode8: %d sequences of up to %d pages (takes %d sequences)", batch, max_pages, DA_MAX_BATCH);
  CUtensorMap mk, mv;
  int rc = d8_map(&mk, k, n_pages * nkv * AF_PAGE, hd);
  if (rc) return rc;
  rc = d8_map(&mv, v, n_pages * nkv * AF_PAGE, hd);
  if (rc) return rc;
  const int sms = af_sm_count();
  if (sms <= 0) return -1;
  Decode8Args a{(const __nv_bfloat16*)q, q_stride, (const uint8_t*)k_exp, (const uint8_t*)v_exp, n_pages, page_table, slots, lens, shared, plan,
                max_pages, nq, nkv, scale, cap, window, keep, ring_rows, n_splits, batch, scratch,
                scratch + (size_t)batch * nq * n_splits * hd, err};
  if (group <= 8) {
    if (hd == 64) return launch_decode8<64, 1>(mk, mv, a, sms, stream);
    if (hd == 128) return launch_decode8<128, 1>(mk, mv, a, sms, stream);
    return launch_decode8<256, 1>(mk, mv, a, sms, stream);
  }
  if (hd == 64) return launch_decode8<64, 2>(mk, mv, a, sms, stream);
  if (hd == 128) return launch_decode8<128, 2>(mk, mv, a, sms, stream);
  return launch_decode8<256, 2>(mk, mv, a, sms, stream);
}

// out [batch, nq * hd] bfloat16 = attention of one new token per sequence over its rows of the 8-bit cache (lens counts the new
// token, which the cache holds already; sequences with slot < 0 or no token give zeros).  window > 0: the last `window`
// positions; < 0: the position's own chunk of -window; the first `keep` stay visible beside either.
AF_EXPORT int af_attn_decode8(void* out, long long out_stride, const void* q, long long q_stride, const void* k, const void* v,
                              const void* k_exp, const void* v_exp, long long n_pages, const int* page_table, int max_pages,
                              const int* slots, const int* lens, int batch, int nq, int nkv, int hd, float scale, float cap, int window,
                              int keep, int ring_rows, int n_splits, float* scratch, const int* plan, const float* sinks, int* err,
                              cudaStream_t stream) {
  if (batch == 0) return 0;
  AF_REQUIRE(out_stride % 2 == 0 && ((uintptr_t)out & 3) == 0, "af_attn_decode8: out must be 4-byte aligned");
  const int rc = af_decode8_split(q, q_stride, k, v, k_exp, v_exp, n_pages, page_table, max_pages, slots, lens, nullptr, batch, nq, nkv, hd,
                                  scale, cap, window, keep, ring_rows, n_splits, scratch, plan, err, stream);
  if (rc) return rc;
  const int sms = af_sm_count();
  const float* part_ml = scratch + (size_t)batch * nq * n_splits * hd;
  const int threads = n_splits > DA_MERGE_FEW && batch * nq <= 32 ? DA_MERGE_THREADS : (hd < 128 ? hd : 128);
  const auto merge = hd == 64 ? attn_decode_merge_kernel<64> : (hd == 128 ? attn_decode_merge_kernel<128> : attn_decode_merge_kernel<256>);
  af_launch(merge, dim3(batch, nq), dim3(threads), 0, stream, (__nv_bfloat16*)out, out_stride, (const float*)scratch, part_ml, nq, nkv,
            n_splits, slots, lens, window, keep, sms, plan, sinks);
  AF_CHECK_LAUNCH("af_attn_decode8 (merge)");
}
