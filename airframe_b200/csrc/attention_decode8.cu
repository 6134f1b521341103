// Decode attention over the 8-bit cache (cache8.cuh): one new token per sequence, bound by the bytes of codes it reads (every
// byte is read once; half of the 16-bit cache's).
//
// The work is cut as for the 16-bit cache (decode_split.cuh): units of a (sequence, kv head), their pages in equal splits or runs, by the
// step's plan.  A block has a warp that brings codes in (TMA, swizzled, through a ring of stages; a row's exponents by plain loads) and
// warps that compute, each 8 KB of keys and values at a time, its running maximum, sum and output its own until the unit's end.  A
// warp's 8 KB are many products (of 16 keys by 8 heads, 16 by 16 by 8 at a time) in a dependent chain from score to output, so it is
// the number of warps with a chain at work that feeds the memory: two blocks of seven computing warps an SM, as the registers
// allow.  Measured (1 sequence of 131,072 tokens, 8 kv heads of 128, 4 heads each; 64 sequences of up to 8,192 tokens and a window of
// 4,096, 8 kv heads of 256, 2 heads each): 53 and 74 us, 5.1 and 4.2 TB/s; with one such block an SM 60 and 105.  Bound by the memory's rate at long lengths.  At short ones by the
// chain of a block: 8 sequences of 2,049 tokens, 4 kv heads of 256, take 14.3 us a layer of a step that has its plan (queries 1, four pages 4.5, the
// warps' join 2.3, the count of a unit's splits 1.5, their join 0.8, the boundary to the kernel before), 1 of 701 8.5.
// Groups of 9 to 16 heads take twice the accumulators and one block an SM: 8 sequences of 16,384 tokens, 2 kv heads of 16 heads each: 31% of
// a copy's rate with heads of 128, 40% with 256.
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
// The block that brings the last of a unit's splits merges them (a count per unit, which it puts back to zero for the next layer): the
// others' partial results come out of L2, and no kernel has to start behind this one.  A unit of one split is finished as it is.
//
// Numbers.  Halves hold 11 bits (bfloat16: 8) but little range.  A head's query is brought to [2^14, 2^15) by a power of two
// (exact down to 2^-29 of its largest element; 2^-39 of it is the most that is lost below).  A weight's half holds
// 2^(s + ev) relative to the largest such sum of the warp's keys so far, times 2^6, which leaves 2^-20 of the largest weight a
// normal half; the softmax's own sum is kept in 32 bits against the scores' maximum.  Both references move only when one is
// passed by more than 8 (base 2).  The softcap is tanh by the exponential, exact to 2^-22 of the cap (tanh.approx: 2^-11).
#include "airframe_b200.h"
#include "cache8.cuh"
#include "decode_split.cuh"

int af_decode8_plan(int* plan, long long plan_ints, const int* page_table, int max_pages, const int* slots, const int* lens, int batch,
                    int nq, int nkv, int window, int keep, int ring_rows, int n_splits, cudaStream_t stream);

namespace {

constexpr float D8_NONE = -3.0e38f;      // a reference before the first key (finite: exp2(-inf - it) is 0)
constexpr float D8_MOVES = 8.f;          // a reference moves when it is passed by more than this
constexpr float D8_SHIFT = 6.f;          // weights are kept times 2^6

template <int HD, int NT>
struct D8 {
  // Warps that compute (one more brings the pieces in) and blocks an SM (d8_blocks).  Groups of up to 8 heads: two blocks of eight warps,
  // 128 registers a thread (heads of 256: 64 of them accumulators, 32 queries); more heads have twice those: one block.
  static constexpr int BLOCKS = NT == 1 ? 2 : 1;
  static constexpr int WARPS = NT == 1 ? 7 : (HD == 256 ? 7 : (HD == 128 ? 11 : 15)), THREADS = (WARPS + 1) * 32;
  // A stage holds a page (heads of 256: half of one).  What a warp takes at a time is a piece of it, 8 KB of keys and values: a
  // stage's pieces are worked side by side, so that it is soon free again and as many bytes are on their way as are being worked.
  static constexpr int ROWS = HD == 256 ? 32 : 64, PER_PAGE = AF_PAGE / ROWS, STAGE_TILES = ROWS / 16;
  static constexpr int KEYS = 4096 / HD, TILES = KEYS / 16;              // keys of a piece, and its tiles of 16 keys
  static constexpr int AT_ONCE = NT == 2 && TILES == 4 ? 2 : TILES;      // tiles of a piece that are worked together
  static constexpr int CODES = ROWS * HD;                                // bytes of a stage's keys, and of its values
  static constexpr int SUB = ROWS * 128;                                 // bytes of a sub-tile of 128 dims
  static constexpr int STAGES = (HD == 64 ? 20 : 12) / BLOCKS;
  // Barriers of the stages' fillings: the producer fills in order, so one is only on its way when all STAGES before it are consumed; a
  // warp's next piece lies at most WARPS / (pieces of a stage) + 1 fillings behind its last one, and must not meet the barrier of one
  // that is still on its way.
  static constexpr int NBAR = 2 * STAGES;
  static constexpr int RING = STAGES * 2 * CODES;
  static constexpr int EXPS = STAGES + 8 <= 16 ? 16 : 32;                // fillings whose exponents are kept: eight more than stages
  static constexpr int MERGE = (24 << 10) / BLOCKS, ROUND = MERGE / (WARPS * HD * 4);       // the merge's buffer, and the rows it takes at a time
  static constexpr int SMEM = RING + MERGE + EXPS * 2 * ROWS + 1024;
  static_assert(NBAR >= STAGES + WARPS * TILES / STAGE_TILES + 2 && EXPS >= STAGES + 8 && NBAR >= 8 && ROUND >= 1, "barriers and buffers");
  static_assert(BLOCKS * (SMEM + 2304) <= 228 * 1024, "blocks an SM");
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
  __nv_bfloat16* out;              // null: the partial results are another kernel's to merge
  long long out_stride;
  int* counts;
  const float* sinks;
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
// Whether the barrier's phase is complete, without a wait.
__device__ __forceinline__ bool d8_is_complete(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// All of a stage's codes, keys or values: its rows, from `row` on, of every sub-tile of 128 dims (see d8_map).
__device__ __forceinline__ void d8_load(void* dst, const CUtensorMap* map, int row, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %3}], [%2], %5;" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(0), "r"(row), "l"(policy)
      : "memory");
}

// S^T, softmax and O^T of N tiles of 16 keys, beginning with tile `t0` of a stage.
template <int HD, int NT, int N>
struct D8Step {
  using C = D8<HD, NT>;
  // k_l, v_l, ke_l: this lane's addresses of the stage's keys, values and exponents (tile 0); lo, hi, keep: the visible keys, counted
  // from the stage's first
  __device__ static __forceinline__ void run(uint32_t k_l, uint32_t v_l, uint32_t ke_l, int t0, bool whole, int lo, int hi, int keep,
                                             int g, int t, bool capped, float ecap, float capl, const uint32_t (&qf)[NT][HD / 16][2],
                                             const float (&cq)[NT][2], float (&o)[HD / 16][NT][4], float (&rs)[NT][2], float (&ra)[NT][2],
                                             float (&l)[NT][2]) {
    constexpr int ROW = HD == 64 ? 64 : 128;              // bytes between rows of a sub-tile
    k_l += t0 * 16 * ROW;
    v_l += t0 * 16 * ROW;
    ke_l += t0 * 16;
    constexpr int CHAINS = N * NT == 1 ? 2 : 1;            // (a product waits for the one before it in its sum)
    float sc[N][NT][4], sc2[CHAINS == 2 ? N : 1][NT][4], wt[N][NT][4];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) sc[i][n][0] = sc[i][n][1] = sc[i][n][2] = sc[i][n][3] = 0.f;
    if constexpr (CHAINS == 2) sc2[0][0][0] = sc2[0][0][1] = sc2[0][0][2] = sc2[0][0][3] = 0.f;
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
          for (int n = 0; n < NT; ++n) d8_mma(CHAINS == 2 && (j & 1) ? sc2[CHAINS == 2 ? i : 0][n] : sc[i][n], a0, a1, a2, a3, qf[n][c * 4 + j][0], qf[n][c * 4 + j][1]);
        }
      }
    }
    if constexpr (CHAINS == 2) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][n][e] += sc2[CHAINS == 2 ? i : 0][n][e];
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
        lv[h] = (float)(d8_lds_u8(ke_l + C::ROWS + i * 16 + 8 * h) - 127);
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

// Four outputs from their sums: v and L relative to 2^ref; a head's sink joins L.
__device__ __forceinline__ void d8_finish(__nv_bfloat16* dst, float4 v, float ref, float L, const float* sinks, int head) {
  if (ref == D8_NONE) ref = 0.f;
  if (sinks != nullptr) {
    // (the larger of the two is the reference, so that neither passes the range)
    const float s = sinks[head] * 1.4426950408889634f, M = fmaxf(ref, s), f = fast_exp2(ref - M);
    L = L * f + fast_exp2(s - M);
    v.x *= f, v.y *= f, v.z *= f, v.w *= f;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const __nv_bfloat162 x = __floats2bfloat162_rn(v.x * inv, v.y * inv), y = __floats2bfloat162_rn(v.z * inv, v.w * inv);
  reinterpret_cast<__nv_bfloat162*>(dst)[0] = x;
  reinterpret_cast<__nv_bfloat162*>(dst)[1] = y;
}

// What a segment of a block's work is: some of the pages of one unit.  The producer warp works it out, the others read it.
struct D8Segment {
  int b, y, kvh, row_head0, n_rows, z, n_pages, x_begin, kept, skip, lo, pos, more;
};

template <int HD, int NT>
__global__ void __launch_bounds__(D8<HD, NT>::THREADS, D8<HD, NT>::BLOCKS)
decode8_split_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Decode8Args a) {
  using C = D8<HD, NT>;
  constexpr int STAGES = C::STAGES, WARPS = C::WARPS, NBAR = C::NBAR, PER = C::PER_PAGE, SEGS = 4;
  constexpr int ROWS = 8 * NT;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ unsigned char d8_raw[];
  unsigned char* ring = (unsigned char*)(((uintptr_t)d8_raw + 1023) & ~(uintptr_t)1023);
  float* o_s = reinterpret_cast<float*>(ring + C::RING);       // the merge's buffer: [warp][row of the round][HD]
  unsigned char* exps = ring + C::RING + C::MERGE;             // [filling modulo EXPS][k exponents | v exponents]
  __shared__ uint64_t full[NBAR], empty[STAGES], seg_full[SEGS], seg_empty[SEGS];
  __shared__ D8Segment seg_s[SEGS];
  __shared__ float rs_s[WARPS][ROWS], ra_s[WARPS][ROWS], l_s[WARPS][ROWS];
  __shared__ int give_up_s, last_s;
  volatile int* give_up = &give_up_s;

  pdl_launch_dependents();
  const int group = a.nq / a.nkv;
  const int tiles = (group + 15) / 16, units_per_seq = a.nkv * tiles;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int4 head = ld_keep_int4(reinterpret_cast<const int4*>(a.plan), l2_policy_keep());
  const int4* rec = reinterpret_cast<const int4*>(a.plan + da_plan_records_at(a.batch, units_per_seq)) +
                    (size_t)blockIdx.x * (DA_PLAN_REC / 4);
  const int4 r0 = ld_keep_int4(rec, l2_policy_keep());
  if (warp == 0) {
    for (int s = lane; s < NBAR; s += 32) mbar_init(&full[s], 2);      // (the copies, and the exponents)
    for (int s = lane; s < STAGES; s += 32) mbar_init(&empty[s], C::STAGE_TILES);
    if (lane < SEGS) {
      mbar_init(&seg_full[lane], 1);
      mbar_init(&seg_empty[lane], WARPS);
    }
    if (lane == 0) give_up_s = 0;
    mbar_fence_init();
  }
  if (head.x != a.n_splits || head.y != da_plan_mark((int)gridDim.x, D8_BREAK_PAGES) || head.z != a.batch || head.w != units_per_seq) {
    if (tid == 0 && a.err) atomicExch(a.err, 1);      // (a plan made for another launch: nothing is read or written by it)
    return;
  }
  __syncthreads();
  // Units without a page give zeros.
  auto zeros = [&]() {
    if (a.out == nullptr) return;
    for (int u = blockIdx.x; u < a.batch * units_per_seq; u += gridDim.x) {
      if (a.plan[DA_PLAN_HEAD + u] != 0) continue;
      const int b = u / units_per_seq, y = u - b * units_per_seq, h0 = y / tiles * group + y % tiles * 16, rows = min(16, y / tiles * group + group - h0);
      for (int i = lane; i < rows * HD / 2; i += 32)
        reinterpret_cast<uint32_t*>(a.out + (size_t)b * a.out_stride + (size_t)h0 * HD)[i] = 0u;
    }
  };
  if (r0.x < 0) {                                     // (no work; a grid without any must not end before the kernel in front)
    pdl_wait();
    if (warp == WARPS) zeros();
    return;
  }

  if (warp == WARPS) {
    // ---- the producer: segments, and their pieces through the ring without a pause between segments
    const int4 r1 = ld_keep_int4(rec + 1, l2_policy_keep()), r2 = ld_keep_int4(rec + 2, l2_policy_keep());
    const int4 r3 = ld_keep_int4(rec + 3, l2_policy_keep());
    int left = r1.y;                                  // what the block's run holds behind the segment's unit
    const int* pt;
    D8Segment sg;
    int y;
    auto of_unit = [&](int b, int y, int p_in, int pos, int slot, int shared) {
      sg.b = b;
      sg.y = y;
      sg.kvh = y / tiles;
      sg.row_head0 = sg.kvh * group + (y % tiles) * 16;
      sg.n_rows = min(16, sg.kvh * group + group - sg.row_head0);
      sg.pos = pos;
      sg.lo = da_lo(pos, a.window);
      const DaList l = da_list(pos, a.window, a.keep, shared);
      sg.kept = l.kept, sg.skip = l.skip;
      sg.x_begin = p_in;
      pt = a.page_table + (size_t)slot * a.max_pages;
    };
    auto safe = [&](int page) { return AF_INDEX_OK(page >= 0 && page < a.n_pages, page) && page >= 0 && page < a.n_pages ? page : 0; };
    auto page_id = [&](int i) {
      const int entry = af_cache_row(da_page_of(sg.kept, sg.skip, sg.x_begin + i) * AF_PAGE, a.ring_rows, a.keep) / AF_PAGE;
      return AF_INDEX_OK(entry < a.max_pages, entry) && entry < a.max_pages ? safe(pt[entry]) : 0;
    };
    const uint64_t read_once = l2_policy_read_once();
    sg.z = r0.w;
    sg.n_pages = r0.x;
    y = r0.z;
    of_unit(r0.y, y, r1.x, r1.z, r1.w, r3.x);
    bool waited = a.shared != nullptr;                // for the kernel in front (see below)
    int ii = 0, stage = 0, bar = 0;                   // fillings so far; their stage and barrier
    uint32_t phase = 0;
    for (int k = 0;; ++k) {
      sg.more = left > D8_BREAK_PAGES ? 1 : 0;        // (the even cut: one segment)
      if (k >= SEGS && !mbar_wait(&seg_empty[k % SEGS], ((k / SEGS) & 1) ^ 1, give_up)) break;
      if (lane == 0) {
        seg_s[k % SEGS] = sg;
        mbar_arrive(&seg_full[k % SEGS]);
      }
      if (waited && lane < sg.n_rows * (HD / 64))     // (the unit's queries: asked into L1 now, read when their segment begins)
        asm volatile("prefetch.global.L1 [%0];" ::"l"(a.q + (size_t)sg.b * a.q_stride + (size_t)(sg.row_head0 + lane / (HD / 64)) * HD +
                                                       (lane % (HD / 64)) * 64));
      const int last_pp = sg.pos / AF_PAGE;           // the page of the new token, which the kernel in front wrote
      // Eight fillings at a time (of a block's first segment first four, whose pages' ids are in the plan).  Four lanes have the filling's
      // exponents, 16 bytes each, asked for a round ahead; the first of them sends the copies off when the stage is free: as many
      // fillings as are free in a row go out at once.  The page of the new token, a segment's last, was written by the kernel in front.
      const int quarter = lane & 3, mine = lane >> 2;
      const bool has = quarter * 16 < C::ROWS;
      uint4 kx = make_uint4(0u, 0u, 0u, 0u), vx = kx;
      auto is_last = [&](int i) { return da_page_of(sg.kept, sg.skip, sg.x_begin + i / PER) == last_pp; };
      auto row_of = [&](int i, int page) { return (page * a.nkv + sg.kvh) * AF_PAGE + i % PER * C::ROWS; };
      auto load = [&](int row) {
        if (!has) return;
        kx = __ldcg(reinterpret_cast<const uint4*>(a.k_exp + row + quarter * 16));
        vx = __ldcg(reinterpret_cast<const uint4*>(a.v_exp + row + quarter * 16));
      };
      const int n = sg.n_pages * PER;
      int row = 0;
      auto ask = [&](int i) {
        if (i < n) {
          const int p = i / PER;
          row = row_of(i, k == 0 && p < 4 ? safe(p == 0 ? r2.x : (p == 1 ? r2.y : (p == 2 ? r2.z : r2.w))) : page_id(p));
          if (waited || !is_last(i)) load(row);
        }
      };
      int m = k == 0 ? 4 : 8;
      if (mine < m) ask(mine);
      bool ok = true;
      for (int i0 = 0; i0 < n && ok; i0 += m, m = 8) {
        m = min(m, n - i0);
        const int here = row;
        int late = 0;                                 // of the round, what lies in the new token's page
        if (!waited)
          while (late < min(m, PER) && is_last(i0 + m - 1 - late)) ++late;
        const int my_stage = (stage + mine) % STAGES;
        const uint32_t my_phase = phase ^ (uint32_t)((stage + mine) / STAGES & 1) ^ 1;
        const int my_bar = bar + mine >= NBAR ? bar + mine - NBAR : bar + mine;
        int done = 0;
        while (done < m) {
          if (late > 0 && done == m - late) {
            pdl_wait();
            waited = true;
            if (mine >= done && mine < m) load(here);
            late = 0;
          }
          __syncwarp();
          const bool open = ii + mine < STAGES || d8_is_complete(&empty[my_stage], my_phase);
          const int most = m - late;
          const uint32_t shut = __ballot_sync(0xffffffffu, mine >= done && !(open && mine < most));
          const int upto = shut ? (__ffs(shut) - 1) >> 2 : 8;
          if (upto > done) {
            if (quarter == 0 && mine >= done && mine < upto) {
              unsigned char* st = ring + (size_t)my_stage * 2 * C::CODES;
              mbar_expect_tx(&full[my_bar], 2 * C::CODES);
              d8_load(st, &map_k, here, &full[my_bar], read_once);
              d8_load(st + C::CODES, &map_v, here, &full[my_bar], read_once);
            }
            // (and their exponents: the round's later fillings may need these stages)
            if (has && mine >= done && mine < upto) {
              uint4* e = reinterpret_cast<uint4*>(exps + ((ii + mine) % C::EXPS) * 2 * C::ROWS) + quarter;
              e[0] = kx;
              e[C::ROWS / 16] = vx;
            }
            __syncwarp();
            if (quarter == 0 && mine >= done && mine < upto) mbar_arrive(&full[my_bar]);
            done = upto;
          } else if (done < most) {
            // nothing is free: the stage's wait, bounded in time (every lane the same barrier)
            ok = mbar_wait(&empty[(stage + done) % STAGES], phase ^ (uint32_t)((stage + done) / STAGES & 1) ^ 1, give_up);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
        }
        if (!ok) break;
        ask(i0 + m + mine);
        ii += m;
        stage += m;
        while (stage >= STAGES) stage -= STAGES, phase ^= 1;
        bar = bar + m >= NBAR ? bar + m - NBAR : bar + m;
      }
      if (!ok || !sg.more) break;
      // the run cut goes on with the unit behind: the same sequence's next, or the first of the next sequence that has pages
      int b = sg.b;
      if (++y >= units_per_seq) {
        y = 0;
        do ++b; while (b < a.batch - 1 && da_pages(a.slots, a.lens, b, a.window, a.keep, a.shared) == 0);
      }
      const int P = da_pages(a.slots, a.lens, b, a.window, a.keep, a.shared);
      sg.z = 0;
      sg.n_pages = min(P, left - D8_BREAK_PAGES);
      left -= D8_BREAK_PAGES + P;
      of_unit(b, y, 0, a.lens[b] - 1, a.slots[b], a.shared != nullptr ? a.shared[b] : 0);
    }
    if (*give_up && lane == 0) {
      grace_period();
      if (a.err) atomicExch(a.err, 1);
    }
    if (!waited || a.shared != nullptr) pdl_wait();
    zeros();
    return;
  }

  // ---- the other warps
  const int g = lane >> 2, t = lane & 3;
  const float ecap = a.cap > 0.f ? 2.f * LOG2E / a.cap : 0.f, capl = a.cap * LOG2E;
  // this lane's place in a piece (see D8Step)
  const int pg = d8_perm(g);
  const uint32_t k_off = HD == 64 ? pg * 64 + ((t ^ ((pg >> 1) & 3)) << 4) : pg * 128 + ((t ^ pg) << 4);
  const uint32_t v_off = C::CODES + (HD == 64 ? t * 64 + (((g >> 1) ^ (t >> 1)) << 4) + (g & 1) * 8 : t * 128 + ((pg ^ t) << 4));
  // a barrier of these warps with a vote: they go on or give up together
  auto all_of = [&](bool ok) {
    int all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "barrier.red.and.pred.aligned p, 1, %2, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(all)
        : "r"(ok ? 1 : 0), "n"(WARPS * 32)
        : "memory");
    return all != 0;
  };
  // (behind the prefix kernel all that came before it is complete already: it is waited for at the producer's end alone)
  if (a.shared == nullptr) pdl_wait();
  int i_base = 0;
  for (int k = 0;; ++k) {
    if (!all_of(mbar_wait(&seg_full[k % SEGS], (k / SEGS) & 1, give_up))) break;
    const D8Segment sg = seg_s[k % SEGS];
    __syncwarp();
    if (lane == 0) mbar_arrive(&seg_empty[k % SEGS]);
    const int n = sg.n_pages * PER, n_rows = sg.n_rows, row_head0 = sg.row_head0;
    const int unit = sg.b * units_per_seq + sg.y;
    const int n_parts = a.out != nullptr ? __ldcg(a.plan + DA_PLAN_HEAD + unit) : 0;       // (0: not merged here)

    // ---- the queries as B fragments (head g of every tile of 8), halves brought to [2^14, 2^15)
    uint32_t qf[NT][HD / 16][2];
    float cq[NT][2];                     // per column (head) of this lane: the factor of its scores
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8) {
      const bool on = n8 * 8 + g < n_rows;
      const __nv_bfloat16* qr = a.q + (size_t)sg.b * a.q_stride + (size_t)(row_head0 + n8 * 8 + g) * HD + t * 16;
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const uint4* p = reinterpret_cast<const uint4*>(qr + c * 64);
        const uint4 q0 = on ? p[0] : make_uint4(0u, 0u, 0u, 0u), q1 = on ? p[1] : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t words[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = words[2 * j], y = words[2 * j + 1];
          qf[n8][c * 4 + j][0] = x;
          qf[n8][c * 4 + j][1] = y;
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
      const int kx = top == 0 ? 14 : max((int)(top >> 7) - 127, -126), up = 14 - kx;
      const float f1 = c8_pow2(up / 2), f2 = c8_pow2(up - up / 2);
      const float cs = (a.cap > 0.f ? a.scale : a.scale * LOG2E) * c8_pow2(-(up / 2)) * c8_pow2(-(up - up / 2));
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w = qf[n8][i][h];
          const __half2 v = __floats2half2_rn(__uint_as_float(w << 16) * f1 * f2, __uint_as_float(w & 0xffff0000u) * f1 * f2);
          qf[n8][i][h] = *reinterpret_cast<const uint32_t*>(&v);
        }
      cq[n8][0] = __shfl_sync(0xffffffffu, cs, t * 8);
      cq[n8][1] = __shfl_sync(0xffffffffu, cs, t * 8 + 4);
    }
    float o[HD / 16][NT][4];
#pragma unroll
    for (int m = 0; m < HD / 16; ++m)
#pragma unroll
      for (int n8 = 0; n8 < NT; ++n8) o[m][n8][0] = o[m][n8][1] = o[m][n8][2] = o[m][n8][3] = 0.f;
    float rs[NT][2], ra[NT][2], l[NT][2];
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8) rs[n8][0] = rs[n8][1] = ra[n8][0] = ra[n8][1] = D8_NONE, l[n8][0] = l[n8][1] = 0.f;

    // A warp takes a piece at a time; where the keys are few, a tile of 16.
    const int each = n * C::STAGE_TILES <= 2 * WARPS ? 1 : C::TILES, items = n * C::STAGE_TILES / each;
    bool ok = true;
    for (int x = warp; x < items; x += WARPS) {
      const int tile = x * each % C::STAGE_TILES, i = x * each / C::STAGE_TILES, ii = i_base + i, s = ii % STAGES;
      ok = mbar_wait(&full[ii % NBAR], (ii / NBAR) & 1, give_up);
      if (!ok) break;
      const uint32_t st = smem_u32(ring) + s * 2 * C::CODES, e_l = smem_u32(exps) + ii % C::EXPS * 2 * C::ROWS + pg;
      const int base = da_page_of(sg.kept, sg.skip, sg.x_begin + i / PER) * AF_PAGE + i % PER * C::ROWS;
      const int lo = sg.lo - base, hi = sg.pos - base, keep = a.keep - base;       // (visible: [lo, hi] and what is before keep)
      const bool whole = C::ROWS - 1 <= hi && (lo <= 0 || C::ROWS - 1 < keep);
      if (C::AT_ONCE > 1 && each == 1) {
        D8Step<HD, NT, 1>::run(st + k_off, st + v_off, e_l, tile, whole, lo, hi, keep, g, t, a.cap > 0.f, ecap, capl, qf, cq, o, rs, ra, l);
      } else {
#pragma unroll 1
        for (int t0 = tile; t0 < tile + each; t0 += C::AT_ONCE)
          D8Step<HD, NT, C::AT_ONCE>::run(st + k_off, st + v_off, e_l, t0, whole, lo, hi, keep, g, t, a.cap > 0.f, ecap, capl, qf, cq, o, rs, ra, l);
      }
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&empty[s])), "r"(each) : "memory");
    }
    i_base += n;

    // ---- merge the warps through shared memory, some rows (heads) a round
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v = l[n8][h];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        const int row = n8 * 8 + 2 * t + h;
        if (g == 0) rs_s[warp][row] = rs[n8][h], ra_s[warp][row] = ra[n8][h], l_s[warp][row] = v;
      }
    bool going = true;
    for (int row0 = 0; row0 < n_rows; row0 += C::ROUND) {
      const int R = min(C::ROUND, n_rows - row0);
#pragma unroll
      for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = n8 * 8 + 2 * t + h - row0;
          if (r >= 0 && r < R) {
            float* dst = o_s + (warp * C::ROUND + r) * HD;
#pragma unroll
            for (int m = 0; m < HD / 16; ++m) {
              const int d = HD == 64 ? g * 8 + m * 2 : (m >> 3) * 128 + pg * 16 + (m & 7) * 2;
              *reinterpret_cast<float2*>(dst + d) = make_float2(o[m][n8][h], o[m][n8][h + 2]);
            }
          }
        }
      if (row0 == 0) {
        going = all_of(ok);
        if (!going) break;
      } else {
        all_of(true);
      }
      for (int i = tid; i < R * (HD / 4); i += WARPS * 32) {
        const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4, row = row0 + r;
        float M = D8_NONE;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, rs_s[w][row]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(o_s + (w * C::ROUND + r) * HD + d);
          const float f = fast_exp2(ra_s[w][row] - D8_SHIFT - M);
          L += l_s[w][row] * fast_exp2(rs_s[w][row] - M);
          v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
        }
        if (n_parts == 1) {
          d8_finish(a.out + (size_t)sg.b * a.out_stride + (size_t)(row_head0 + row) * HD + d, v, M, L, a.sinks, row_head0 + row);
        } else {
          const size_t pidx = ((size_t)sg.b * a.nq + row_head0 + row) * a.n_splits + sg.z;
          *reinterpret_cast<float4*>(a.part_o + pidx * HD + d) = v;
          if (d == 0) *reinterpret_cast<float2*>(a.part_ml + pidx * 2) = make_float2(M == D8_NONE ? -INFINITY : M, L);
        }
      }
      if (row0 + C::ROUND < n_rows) all_of(true);      // (the buffer is written again; a segment's first vote does it for the next segment)
    }
    if (!going) break;
    if (n_parts > 1) {
      // ---- the unit's last split merges them all
      all_of(true);
      if (tid == 0) {
        int before;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(a.counts + unit) : "memory");
        last_s = before == n_parts - 1;
        if (last_s) a.counts[unit] = 0;
      }
      all_of(true);
      constexpr int FEW = 16;
      if (last_s && n_parts <= FEW) {
        // few of them: maxima, sums and outputs all asked for at once
        for (int i = tid; i < n_rows * (HD / 4); i += WARPS * 32) {
          const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
          const size_t p0 = ((size_t)sg.b * a.nq + row_head0 + r) * a.n_splits;
          float2 ml[FEW];
          float4 x[FEW];
#pragma unroll
          for (int u = 0; u < FEW; ++u) {
            ml[u] = u < n_parts ? __ldcg(reinterpret_cast<const float2*>(a.part_ml) + p0 + u) : make_float2(-INFINITY, 0.f);
            x[u] = u < n_parts ? __ldcg(reinterpret_cast<const float4*>(a.part_o + (p0 + u) * HD + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
          float M = -INFINITY;
#pragma unroll
          for (int u = 0; u < FEW; ++u) M = fmaxf(M, ml[u].x);
          const float ref = M == -INFINITY ? 0.f : M;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          float L = 0.f;
#pragma unroll
          for (int u = 0; u < FEW; ++u) {
            const float f = fast_exp2(ml[u].x - ref);
            L += ml[u].y * f;
            v.x += x[u].x * f, v.y += x[u].y * f, v.z += x[u].z * f, v.w += x[u].w * f;
          }
          d8_finish(a.out + (size_t)sg.b * a.out_stride + (size_t)(row_head0 + r) * HD + d, v, ref, L, a.sinks, row_head0 + r);
        }
      } else if (last_s) {
        constexpr int MOST = C::MERGE / 8;               // (maximum, sum) pairs that the buffer holds
        float2* ml_s = reinterpret_cast<float2*>(o_s);
        const int R = max(1, min(n_rows, MOST / n_parts));
        for (int row0 = 0; row0 < n_rows; row0 += R) {
          const int rows = min(R, n_rows - row0);
          const size_t p0 = ((size_t)sg.b * a.nq + row_head0 + row0) * a.n_splits;
          for (int i = tid; i < rows * n_parts && i < MOST; i += WARPS * 32) {
            const int r = i / n_parts;
            ml_s[i] = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + p0 + (size_t)r * a.n_splits + (i - r * n_parts));
          }
          all_of(true);
          for (int i = tid; i < rows * (HD / 4); i += WARPS * 32) {
            const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
            const float2* ml = ml_s + r * n_parts;
            float M = -INFINITY;
            for (int x = 0; x < n_parts; ++x) M = fmaxf(M, ml[x].x);
            const float ref = M == -INFINITY ? 0.f : M;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float L = 0.f;
            const float* src = a.part_o + (p0 + (size_t)r * a.n_splits) * HD + d;
            for (int x0 = 0; x0 < n_parts; x0 += 8) {
              float4 t8[8];
#pragma unroll
              for (int u = 0; u < 8; ++u)
                t8[u] = x0 + u < n_parts ? __ldcg(reinterpret_cast<const float4*>(src + (size_t)(x0 + u) * HD)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                const float2 m = x0 + u < n_parts ? ml[x0 + u] : make_float2(-INFINITY, 0.f);
                const float f = fast_exp2(m.x - ref);
                L += m.y * f;
                v.x += t8[u].x * f, v.y += t8[u].y * f, v.z += t8[u].z * f, v.w += t8[u].w * f;
              }
            }
            d8_finish(a.out + (size_t)sg.b * a.out_stride + (size_t)(row_head0 + row0 + r) * HD + d, v, ref, L, a.sinks, row_head0 + row0 + r);
          }
          all_of(true);
        }
      }
    }
    if (!sg.more) break;
  }
}

// Tensor map of the codes: [HD / 128 sub-tiles][rows][128 bytes] (HD 64: one of 64 bytes), the sub-tiles of a row beside one
// another in memory; boxes of a stage's rows in all sub-tiles, swizzled.
int d8_map(CUtensorMap* map, const void* base, long long rows, int hd) {
  AfEncodeTiledFn enc = af_encode_tiled();
  if (enc == nullptr) return af_fail(-1, "the driver has no cuTensorMapEncodeTiled");
  const cuuint32_t width = hd < 128 ? 64u : 128u, subs = (cuuint32_t)hd / width;
  cuuint64_t dims[3] = {width, (cuuint64_t)rows, subs};
  cuuint64_t strides[2] = {(cuuint64_t)hd, width};
  cuuint32_t box[3] = {width, hd == 256 ? 32u : 64u, subs};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
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

// What the kernel cannot take, refused before anything is launched.
static int d8_refuses(const void* q, long long q_stride, const void* k, const void* v, const void* k_exp, const void* v_exp,
                      long long n_pages, int max_pages, int batch, int nq, int nkv, int hd, int window, int keep, int ring_rows,
                      int n_splits, const float* scratch, const int* plan) {
  AF_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "af_attn_decode8: heads %d, groups %d", nq, nkv);
  AF_REQUIRE(hd == 64 || hd == 128 || hd == 256, "af_attn_decode8: head_dim %d (takes 64, 128, 256)", hd);
  AF_REQUIRE(keep >= 0 && (keep == 0 || window != 0), "af_attn_decode8: %d kept tokens with window %d", keep, window);
  AF_REQUIRE(ring_rows >= 0 && ring_rows % AF_PAGE == 0 && (ring_rows == 0 || (window != 0 && abs(window) <= ring_rows)),
             "af_attn_decode8: window %d (negative: a chunk), ring rows %d", window, ring_rows);
  AF_REQUIRE(n_splits >= 1 && n_splits <= 65535 && scratch != nullptr && plan != nullptr && ((uintptr_t)plan & 15) == 0,
             "af_attn_decode8: splits %d, scratch and a 16-byte aligned plan", n_splits);
  AF_REQUIRE((((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_exp | (uintptr_t)v_exp | (uintptr_t)scratch) & 15) == 0,
             "af_attn_decode8: cache and scratch alignment");
  // (a row of queries is read in loads of 16 bytes)
  AF_REQUIRE((batch == 1 || q_stride % 8 == 0) && ((uintptr_t)q & 15) == 0, "af_attn_decode8: rows of queries must be 16-byte aligned");
  AF_REQUIRE(n_pages > 0 && n_pages * nkv * AF_PAGE < (1ll << 31), "af_attn_decode8: %lld cache pages", n_pages);
  const int group = nq / nkv, units_per_seq = nkv * ((group + 15) / 16);
  AF_REQUIRE(batch <= DA_MAX_BATCH && (long long)batch * (max_pages + 1 + D8_BREAK_PAGES) * units_per_seq < (1ll << 31),
             "af_attn_decode8: %d sequences of up to %d pages (takes %d sequences)", batch, max_pages, DA_MAX_BATCH);
  return 0;
}

// The attention into `out`, or where that is null the split pass alone: partial results of every (sequence, head) in `scratch`
// (af_attn_decode_scratch(...) floats), as the step's `plan` (af_decode8_plan, or the shared one) cuts the work.
int af_decode8_split(const void* q, long long q_stride, const void* k, const void* v, const void* k_exp, const void* v_exp,
                     long long n_pages, const int* page_table, int max_pages, const int* slots, const int* lens, const int* shared,
                     int batch, int nq, int nkv, int hd, float scale, float cap, int window, int keep, int ring_rows, int n_splits,
                     float* scratch, const int* plan, int* err, cudaStream_t stream, void* out, long long out_stride,
                     const float* sinks) {
  int rc = d8_refuses(q, q_stride, k, v, k_exp, v_exp, n_pages, max_pages, batch, nq, nkv, hd, window, keep, ring_rows, n_splits, scratch, plan);
  if (rc) return rc;
  const int group = nq / nkv, units_per_seq = nkv * ((group + 15) / 16);
  CUtensorMap mk, mv;
  rc = d8_map(&mk, k, n_pages * nkv * AF_PAGE, hd);
  if (rc) return rc;
  rc = d8_map(&mv, v, n_pages * nkv * AF_PAGE, hd);
  if (rc) return rc;
  const int sms = af_sm_count();
  if (sms <= 0) return -1;
  const int blocks = d8_blocks(sms, nq, nkv);
  Decode8Args a{(const __nv_bfloat16*)q, q_stride, (const uint8_t*)k_exp, (const uint8_t*)v_exp, n_pages, page_table, slots, lens, shared, plan,
                max_pages, nq, nkv, scale, cap, window, keep, ring_rows, n_splits, batch, scratch,
                scratch + (size_t)batch * nq * n_splits * hd, err, (__nv_bfloat16*)out, out_stride,
                (int*)plan + da_plan_records_at(batch, units_per_seq) + (size_t)blocks * DA_PLAN_REC, sinks};
  if (group <= 8) {
    if (hd == 64) return launch_decode8<64, 1>(mk, mv, a, blocks, stream);
    if (hd == 128) return launch_decode8<128, 1>(mk, mv, a, blocks, stream);
    return launch_decode8<256, 1>(mk, mv, a, blocks, stream);
  }
  if (hd == 64) return launch_decode8<64, 2>(mk, mv, a, blocks, stream);
  if (hd == 128) return launch_decode8<128, 2>(mk, mv, a, blocks, stream);
  return launch_decode8<256, 2>(mk, mv, a, blocks, stream);
}

// What af_attn_decode8 is given, as one block of 64-bit words.
struct AfDecode8 {
  void* out;
  const void *q, *k, *v, *k_exp, *v_exp, *page_table, *slots, *lens;
  float* scratch;
  int* plan;
  const void* sinks;
  int* err;
  cudaStream_t stream;
  long long out_stride, q_stride, n_pages, max_pages, batch, nq, nkv, hd, window, keep, ring_rows, n_splits, plan_ints;
  double scale, cap;
};

// out [batch, nq * hd] bfloat16 = attention of one new token per sequence over its rows of the 8-bit cache (lens counts the new
// token, which the cache holds already; sequences with slot < 0 or no token give zeros).  window > 0: the last `window`
// positions; < 0: the position's own chunk of -window; the first `keep` stay visible beside either.  plan_ints > 0: the step's plan
// is made first, into `plan`'s so many integers; 0: it holds the plan of a call for the same slots, lengths, page table, heads,
// window, ring and n_splits.
AF_EXPORT int af_attn_decode8(const AfDecode8* c) {
  if (c->batch == 0) return 0;
  AF_REQUIRE(c->out_stride % 2 == 0 && ((uintptr_t)c->out & 3) == 0, "af_attn_decode8: out must be 4-byte aligned");
  AF_REQUIRE(c->batch > 0 && c->batch <= DA_MAX_BATCH, "af_attn_decode8: %lld sequences (takes %d)", c->batch, DA_MAX_BATCH);
  const int batch = (int)c->batch, nq = (int)c->nq, nkv = (int)c->nkv, hd = (int)c->hd, n_splits = (int)c->n_splits;
  const int *page_table = (const int*)c->page_table, *slots = (const int*)c->slots, *lens = (const int*)c->lens;
  int rc = d8_refuses(c->q, c->q_stride, c->k, c->v, c->k_exp, c->v_exp, c->n_pages, (int)c->max_pages, batch, nq, nkv, hd, (int)c->window,
                      (int)c->keep, (int)c->ring_rows, n_splits, c->scratch, c->plan);
  if (rc) return rc;
  if (c->plan_ints > 0) {
    rc = af_decode8_plan(c->plan, c->plan_ints, page_table, (int)c->max_pages, slots, lens, batch, nq, nkv, (int)c->window, (int)c->keep,
                                   (int)c->ring_rows, n_splits, c->stream);
    if (rc) return rc;
  }
  return af_decode8_split(c->q, c->q_stride, c->k, c->v, c->k_exp, c->v_exp, c->n_pages, page_table, (int)c->max_pages, slots, lens, nullptr,
                          batch, nq, nkv, hd, (float)c->scale, (float)c->cap, (int)c->window, (int)c->keep, (int)c->ring_rows, n_splits,
                          c->scratch, c->plan, c->err, c->stream, c->out, c->out_stride, (const float*)c->sinks);
}
