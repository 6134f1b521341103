// Decode attention of sequences that share a prefix (completions of one prompt, requests behind one system prompt): the
// shared cache pages are read once for all of a group's sequences, and their products are one tensor-core product of many rows.
//
// Three kernels behind the step's plan (one small kernel a step for all layers), the first two of which run side by side where SMs are
// left: the prefix kernel lets the next one start when its own wait is over, so that all that came before is complete, and the next
// one waits for it at its end only:
//   prefix  the rows of a unit are the query heads of one kv head of all members of a group (up to 128 of them, more in several
//           units); the units' pages are cut into items, one a block; every row leaves (max, sum, output) of each item
//   rest    the split kernel of the cache at hand over each sequence's own pages (its plan leaves the shared ones out)
//   merge   of both, one block a (sequence, head)
//
// The prefix kernel.  A block holds its 128 rows' queries in tensor memory and walks its pages, 64 keys at a time:
//   S = Q K^T     tcgen05.mma, M = 128, N = 64, Q from TMEM, the K page from swizzled shared memory
//   softmax       two groups of eight warps take the pages in turn, two threads a row (32 keys each): all keys are visible (a shared
//                 page is full and older than every member's token), so there is no mask; P goes back into its S columns of TMEM
//   O += P V      tcgen05.mma, P from TMEM, O (128 x head_dim, 32 bits) in TMEM for the whole item
// A reference maximum moves only when it is passed by more than 2^8.  With heads of 64 and 128 each group has a reference and an O of its own
// (two of 128 columns), joined at the item's end; with heads of 256 TMEM holds one O, whose reference a group hands to the other with
// every page.  Products and softmax of neighbouring pages overlap.
//   warp 0        TMA producer (16-bit cache)         warp 1  issue of S, TMEM allocation      warp 2  issue of O += P V
//   warps 4..19   queries, softmax, rescaling, partial results
//   warps 20..    8-bit cache only: codes, brought into shared memory as they are by warp 0, to halves in the swizzled operand layout (four
//                 warps keys and values; with heads of 256, whose pages take twice the conversions, four the keys and four the values); warp 3 the
//                 rows' factors
// An item's partial results are gathered in the operands' memory and leave as one bulk copy (they are contiguous; 16-byte piece c of
// row r lies at piece c ^ (r & 7), for the banks' sake).
// In the 8-bit cache a key's factor multiplies its scores, a value's (2^ev) its weights.  The one reference of a row is then the largest
// s + max(ev, -60), so that the halves of the weights keep 2^-20 of the largest as normal numbers; sums and outputs are relative to it
// less 6.  (Weights of values below 2^-60 * 448 may vanish, and of sums what is below 2^-20 even where values are of 2^110.)
// Measured, a layer of 2 sequences behind 131,072 tokens: 8 kv heads of 128, bfloat16, 87.5 us (6.1 TB/s with all that belongs to it), bound by
// the prefix's bytes; 8 bits 118.9 us, 0.85 us a page and block, bound by the chain scores - softmax - weights of the two groups (a group's
// page takes some 3,400 cycles, of which 900 are waits on barriers that are complete); 4 kv heads of 256 96 us and 122 (8 bits: by the conversion
// and the single O).  32 sequences of 8 kv heads of 128, 4 heads each, behind 32,768 tokens in 8 bits: the kernel 46.7 us, 1.3 us a page with
// all 128 rows at work (half of the issue slots).  64 sequences of 4 kv heads of 256, 2 heads each, behind 7,168 tokens: the kernel 24 us.
// Every wait on a barrier is bounded in time; one that runs out sets the error word, and the block frees its TMEM and returns.
#include "airframe_b200.h"
#include "cache8.cuh"
#include "decode_split.cuh"
#include "umma.cuh"

int af_decode8_split(const void* q, long long q_stride, const void* k, const void* v, const void* k_exp, const void* v_exp,
                     long long n_pages, const int* page_table, int max_pages, const int* slots, const int* lens, const int* shared,
                     int batch, int nq, int nkv, int hd, float scale, float cap, int window, int keep, int ring_rows, int n_splits,
                     float* scratch, const int* plan, int* err, cudaStream_t stream, void* out, long long out_stride,
                     const float* sinks);
int af_decode16_split(const void* q, long long q_stride, const void* kcache, const void* vcache, long long n_pages,
                      const int* page_table, int max_pages, const int* slots, const int* lens, const int* shared, int batch, int nq,
                      int nkv, int hd, float scale, float cap, int n_splits, float* scratch, const int* plan, int blocks, int* err,
                      cudaStream_t stream);

namespace {

// ---------------------------------------------------------------- the plan
//
// 32-bit integers: [0, 16) items, units, sequences, heads, kv heads, blocks; then
//   shared [batch]      the pages of each sequence that the prefix kernel takes (0: none)
//   loc    [batch][2]   its group's first unit (-1: none), its place among the group's members
//   order  [batch]      the groups' members, group after group
//   units  [n][4]       members of its group, items, first partial row, 0
//   items  [n][8]       ShItem: what a block reads with two loads
constexpr int SH_HEAD = 16, SH_ROWS = 128, SH_MAX_BATCH = DA_MAX_BATCH;

__host__ __device__ inline int sh_max_units(int batch, int nq, int nkv) { return nkv * (batch * (nq / nkv) / SH_ROWS + batch / 2 + 1); }
struct ShPlan {
  int shared, loc, order, units, items, total;
};
__host__ __device__ inline ShPlan sh_layout(int batch, int nq, int nkv, int blocks) {
  ShPlan p;
  const int b4 = (batch + 3) / 4 * 4, units = sh_max_units(batch, nq, nkv);
  p.shared = SH_HEAD;
  p.loc = p.shared + b4;
  p.order = p.loc + 2 * b4;
  p.units = p.order + b4;       // (all of them multiples of four: read four integers at a time)
  p.items = p.units + 4 * units;
  p.total = p.items + 8 * (blocks + units);
  return p;
}

// Where the split kernel's plan begins.
__host__ __device__ inline int sh_own_plan(const ShPlan& p) { return (p.total + 3) / 4 * 4; }

// Items of a unit of `pages` shared pages, `units` of them and `rows` rows a kv head in its group: its share of the blocks, rounded
// down, so that no block gets a second one; but no more than pay.  s items take pages / s of a page's time each (some 0.8 us with heads
// of 256) and leave s partial results of every unit, written and read again at some 5 TB/s together: the sum is least for
// s^2 = pages * time of a page * rate / (bytes of a partial result of all units).  (64 sequences of 2 heads a kv head of 256, 112 pages: 20 items
// a unit instead of 37.)
__device__ __forceinline__ int sh_items(int pages, int units, int rows, int hd, int blocks, long long total) {
  const float page_us = 0.4f + 0.4f * (float)hd / 256.f;
  const float bytes = (float)units * (float)min(rows, SH_ROWS) * (float)hd * 8.f;
  const int pay = (int)ceilf(sqrtf((float)pages * page_us * 5.0e6f / bytes));
  return max(1, min(min(pages, pay), (int)min((long long)pages, (long long)pages * blocks / total)));
}

// A step's, for all layers: some 7 us with up to 64 sequences, 24 with 64 groups of 4, 50 to 70 with one of 2,048, 170 with 512 of 4 (a group's units and
// items by one warp).  Two blocks: the first writes the prefix kernel's plan, the second the split kernel's.  (Like attn_decode_plan_kernel they do not
// release their dependents early.)  A group is the live rows of one `lead` that share at least a page; alone in it a row keeps its pages.  Fewer
// pages than a row claims are taken where another of the group shares fewer, and never the page of its new token.
__global__ void __launch_bounds__(512)
attn_shared_plan_kernel(int* plan, const int* lead, const int* pages, const int* slots, const int* lens, const int* page_table, int max_pages,
                        int batch, int nq, int nkv, int hd, int blocks, int own_room, int own_blocks, int brk) {
  extern __shared__ int sp_smem[];
  int* gid = sp_smem;                  // [batch] the row's group, -1: none
  int* cnt = gid + batch;              // [batch] by group: members
  int* few = cnt + batch;              //           the pages all of them share
  int* unit0 = few + batch;            //           first unit
  int* item0 = unit0 + batch;          //           first item
  int* memb0 = item0 + batch;          //           first place in `order`
  int* row0 = memb0 + batch;           //           first partial row
  int* parts = row0 + batch;           //           items of a unit
  int* seen = parts + batch;           //           members met so far
  int* lead_row = seen + batch;        //           the first member
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = nq / nkv;
  const ShPlan L = sh_layout(batch, nq, nkv, blocks);
  for (int b = tid; b < batch; b += blockDim.x) cnt[b] = 0, few[b] = 0x7fffffff, seen[b] = 0;
  __syncthreads();
  for (int b = tid; b < batch; b += blockDim.x) {
    const int len = lens[b], p = slots[b] >= 0 && len > 0 ? min(pages[b], (len - 1) / AF_PAGE) : 0, g = lead[b];
    gid[b] = p > 0 && g >= 0 && g < batch ? g : -1;
    if (gid[b] >= 0) {
      atomicAdd(&cnt[g], 1);
      atomicMin(&few[g], p);
    }
  }
  __syncthreads();
  if (blockIdx.x == 1) {
    int* shared = unit0;
    for (int b = tid; b < batch; b += blockDim.x) shared[b] = gid[b] >= 0 && cnt[gid[b]] >= 2 ? few[gid[b]] : 0;
    __syncthreads();
    da_write_plan(plan + sh_own_plan(L), slots, lens, page_table, max_pages, batch, nq, nkv, 0, 0, 0, own_room, own_blocks, shared, brk,
                  parts + batch);
    return;
  }
  if (warp == 0) {
    // places of the groups: units first, then (their pages known) items and partial rows
    int units = 0, members = 0;
    long long total = 0;
    for (int base = 0; base < batch; base += 32) {
      const int g = base + lane;
      const bool on = g < batch && cnt[g] >= 2;
      const int c = on ? cnt[g] : 0, u = on ? nkv * ((c * group + SH_ROWS - 1) / SH_ROWS) : 0;
      int vu = u, vm = c;
      long long vt = on ? (long long)u * few[g] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, vu, o), m = __shfl_up_sync(0xffffffffu, vm, o);
        if (lane >= o) vu += a, vm += m;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) vt += __shfl_xor_sync(0xffffffffu, vt, o);
      if (on) unit0[g] = units + vu - u, memb0[g] = members + vm - c;
      units += __shfl_sync(0xffffffffu, vu, 31);
      members += __shfl_sync(0xffffffffu, vm, 31);
      total += vt;
    }
    int items = 0, rows = 0;
    for (int base = 0; base < batch; base += 32) {
      const int g = base + lane;
      const bool on = g < batch && cnt[g] >= 2;
      const int c = on ? cnt[g] : 0, u = on ? nkv * ((c * group + SH_ROWS - 1) / SH_ROWS) : 0;
      const int s = on ? sh_items(few[g], u, c * group, hd, blocks, total) : 0;
      int vi = u * s, vr = nkv * c * group * s;
      const int i1 = vi, r1 = vr;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, vi, o), m = __shfl_up_sync(0xffffffffu, vr, o);
        if (lane >= o) vi += a, vr += m;
      }
      if (on) item0[g] = items + vi - i1, row0[g] = rows + vr - r1, parts[g] = s;
      items += __shfl_sync(0xffffffffu, vi, 31);
      rows += __shfl_sync(0xffffffffu, vr, 31);
    }
    if (lane == 0) {
      plan[0] = items, plan[1] = units, plan[2] = batch, plan[3] = nq, plan[4] = nkv, plan[5] = blocks;
    }
  } else if (warp == 1) {
    // each row's place among its group's members, in the order of the rows: 32 rows at a time, a lane counts those of its group before it
    for (int base = 0; base < batch; base += 32) {
      const int b = base + lane, g = b < batch ? gid[b] : -1;
      const uint32_t same = __match_any_sync(0xffffffffu, g);
      const int place = g >= 0 ? seen[g] + __popc(same & ((1u << lane) - 1)) : 0;
      __syncwarp();
      if (g >= 0) {
        if (place == 0) lead_row[g] = b;
        if (lane == __ffs(same) - 1) seen[g] += __popc(same);
      }
      if (b < batch) plan[L.loc + 2 * b + 1] = place;
      __syncwarp();
    }
  }
  __syncthreads();
  for (int b = tid; b < batch; b += blockDim.x) {
    const int g = gid[b];
    const bool on = g >= 0 && cnt[g] >= 2;
    plan[L.shared + b] = on ? few[g] : 0;
    plan[L.loc + 2 * b] = on ? unit0[g] : -1;
    if (on) plan[L.order + memb0[g] + plan[L.loc + 2 * b + 1]] = b;
  }
  for (int g = warp; g < batch; g += (int)blockDim.x >> 5) {
    const int c = cnt[g];
    if (c < 2) continue;
    const int b = lead_row[g];                            // a member's slot: its page table holds the shared pages
    const int rows = c * group, tiles = (rows + SH_ROWS - 1) / SH_ROWS, u = nkv * tiles;
    const int s = parts[g];
    for (int x = lane; x < u; x += 32) {
      const int kvh = x / tiles, tile = x - kvh * tiles;
      reinterpret_cast<int4*>(plan + L.units)[unit0[g] + x] = make_int4(c, s, row0[g] + (kvh * rows + tile * SH_ROWS) * s, 0);
    }
    for (int x = lane; x < u * s; x += 32) {
      const int unit = x / s, z = x - unit * s, kvh = unit / tiles, tile = unit - kvh * tiles, r = min(SH_ROWS, rows - tile * SH_ROWS);
      const int first = (int)((long long)z * few[g] / s), end = (int)((long long)(z + 1) * few[g] / s);
      int4* it = reinterpret_cast<int4*>(plan + L.items + 8 * (item0[g] + x));
      it[0] = make_int4(r, first, end - first, row0[g] + (kvh * rows + tile * SH_ROWS) * s + z * r);
      it[1] = make_int4(memb0[g], tile * SH_ROWS, kvh, slots[b]);
    }
  }
}

// ---------------------------------------------------------------- the prefix kernel

constexpr float SH_NONE = -3.0e38f;      // a reference before the first key
constexpr float SH_MOVES = 8.f;          // the reference moves when it is passed by more than this
constexpr float SH_SHIFT = 6.f;          // (8 bits) halves of weights are kept times 2^6
constexpr int SH_EXPS = 16;              // (8 bits) pages whose factors are kept: more than the K stages and the two at work

template <int HD, int BITS>
struct Sh {
  // Warps that convert: four keys and four values, or four both.  (2 sequences behind 131,072 tokens: heads of 256 124 us with eight, 146 with four; heads of
  // 128 123 and 119: what the softmax loses in registers.)
  static constexpr int CONV = BITS == 16 ? 0 : (HD == 256 ? 8 : 4);
  static constexpr int WARPS = 20 + CONV, THREADS = WARPS * 32;
  static constexpr int TILE = AF_PAGE * HD * 2;                              // bytes of a page's keys, or values, as operand
  // pages in flight (16 bits), or converted (8 bits; beside them RAW pages of codes are in flight)
  static constexpr int STAGES = BITS == 16 ? (HD == 256 ? 3 : (HD == 128 ? 6 : 8)) : (HD == 256 ? 2 : (HD == 128 ? 4 : 6));
  static constexpr int CODES = BITS == 8 ? AF_PAGE * HD : 0, RAW = HD == 256 ? 2 : (HD == 128 ? 4 : 8);
  static constexpr int RAW_STAGE = 2 * CODES + (BITS == 8 ? 2 * AF_PAGE : 0);
  static constexpr int SMEM = 2 * STAGES * TILE + RAW * RAW_STAGE + 1024;
  static_assert(SH_ROWS * HD * 4 <= 2 * STAGES * TILE, "an item's results fit the operands' memory");
};

struct ShArgs {
  const __nv_bfloat16* q;
  long long q_stride;
  const uint8_t *k, *v, *k_exp, *v_exp;     // (8 bits)
  long long n_pages;
  const int *page_table, *plan;
  int max_pages, batch, nq, nkv;
  float scale, cap;
  float *part_o, *part_ml;                  // [partial row][HD], [partial row][2]
  int* err;
};

// f16 x f16 -> f32, as umma_idesc
__host__ __device__ constexpr uint32_t sh_idesc(int bn, bool f16, bool b_mn_major) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(bn >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void sh_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Two products (and sums) at a time.
struct ShPair {
  float x, y;
};
__device__ __forceinline__ ShPair sh_mul2(ShPair a, ShPair b) {
  ShPair d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ ShPair sh_add2(ShPair a, ShPair b) {
  ShPair d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ ShPair sh_fma2(ShPair a, ShPair b, ShPair c) {
  ShPair d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// What an item is: every role reads it from the plan.
struct ShItem {
  int rows, first, pages, row0, members0, group0, kvh, slot;      // rows of the tile; page range; partial row; ...
};

template <int HD, int BITS>
__global__ void __launch_bounds__(Sh<HD, BITS>::THREADS, 1)
attn_shared_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, ShArgs a) {
  using C = Sh<HD, BITS>;
  constexpr int SUB = HD / 64, STAGES = C::STAGES;
  // TMEM columns: S of the two groups [0, 64) [64, 128); where there is room P apart from it, [128, 160) [160, 192), and Q from 192 on (the
  // next scores are then made while a group's softmax still works); with heads of 256 P takes S's columns and Q is [128, 256); O from 256 on
  constexpr bool APART = HD <= 128;
  constexpr uint32_t P_COL = APART ? 128 : 0, P_STEP = APART ? 32 : 64, Q_COL = APART ? 192 : 128, O_COL = 256, O_STEP = APART ? HD : 0;
  constexpr uint32_t IDESC_S = sh_idesc(AF_PAGE, BITS == 8, false), IDESC_O = sh_idesc(HD, BITS == 8, true);
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ unsigned char sh_raw[];
  unsigned char* k_s = (unsigned char*)(((uintptr_t)sh_raw + 1023) & ~(uintptr_t)1023);      // [stage][sub-tile][64 keys][128 B]
  unsigned char* v_s = k_s + STAGES * C::TILE;
  unsigned char* raw_s = v_s + STAGES * C::TILE;     // [stage][codes of keys | of values | exponents of keys | of values]
  __shared__ uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[2], p_full[2], pv_done[2], m_ready[2], x_full[2], q_ready,
      l_full, staged, ring_free, raw_full[C::RAW], raw_empty[C::RAW];
  constexpr int W_PAGES = BITS == 8 ? SH_EXPS : 1;
  // by group: the reference after its page; by group, turn and part: the maxima of a page; by thread of a row: sums
  __shared__ float mref_s[2][SH_ROWS], mx_s[2][2][2][SH_ROWS], l_s[4][SH_ROWS];
  // the keys' factors, the values' exponents (no less than -60) and factors
  __shared__ __align__(16) float ks_s[W_PAGES][AF_PAGE], lv_s[W_PAGES][AF_PAGE], vs_s[W_PAGES][AF_PAGE];
  __shared__ uint32_t tmem_base_s;
  __shared__ int give_up_s;
  volatile int* give_up = &give_up_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.nq / a.nkv;
  const ShPlan L = sh_layout(a.batch, a.nq, a.nkv, (int)gridDim.x);
  const int4 head = *reinterpret_cast<const int4*>(a.plan);
  // (the block's first item is read beside the head: the plan holds as many places for items as the grid has blocks)
  const int4 it0 = *reinterpret_cast<const int4*>(a.plan + L.items + 8 * blockIdx.x);
  const int4 it1 = *reinterpret_cast<const int4*>(a.plan + L.items + 8 * blockIdx.x + 4);
  const int n_items = head.x;
  if (head.z != a.batch || head.w != a.nq || a.plan[4] != a.nkv || a.plan[5] != (int)gridDim.x) {
    if (threadIdx.x == 0 && a.err) atomicExch(a.err, 1);      // (a plan made for another launch)
    return;
  }
  if ((int)blockIdx.x >= n_items) {
    if (blockIdx.x == 0) pdl_wait();      // (without items the kernel must not end before the one in front: the next one waits for this one alone)
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&k_full[s], BITS == 8 ? 5 : 1);      // (one arrival a converting warp, and the factors')
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], BITS == 8 ? 4 : 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 8);
      mbar_init(&pv_done[s], 1);
      mbar_init(&m_ready[s], 8);
      mbar_init(&x_full[s], 8);
    }
    mbar_init(&q_ready, 16);
    mbar_init(&l_full, 16);
    mbar_init(&staged, 16);
    mbar_init(&ring_free, 1);
    for (int s = 0; s < C::RAW; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], C::CONV + 1);
    }
    give_up_s = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;

  auto item_of = [&](int w) {
    const int4* r = reinterpret_cast<const int4*>(a.plan + L.items + 8 * w);
    const int4 x = w == (int)blockIdx.x ? it0 : r[0], y = w == (int)blockIdx.x ? it1 : r[1];
    return ShItem{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  };
  auto page_id = [&](const ShItem& it, int j) {
    const int entry = it.first + j;
    const int page = AF_INDEX_OK(entry < a.max_pages, entry) && entry < a.max_pages ? a.page_table[(size_t)it.slot * a.max_pages + entry] : 0;
    return AF_INDEX_OK(page >= 0 && page < a.n_pages, page) && page >= 0 && page < a.n_pages ? page : 0;
  };

  // Pages are counted through over the block's items (`jj`): a page's group, stage and phases follow from its count.
  if (warp == 0) {
    // ---- the cache's pages, to the operands or (8 bits) as they are.  They are older than the kernels in front: nothing to wait for
    if (lane == 0) {
      int jj = 0, n = 0;
      for (int w = blockIdx.x; w < n_items && !*give_up; w += gridDim.x, ++n) {
        const ShItem it = item_of(w);
        int next = page_id(it, 0);
        if constexpr (BITS == 8) {
          for (int j = 0; j < it.pages; ++j, ++jj) {
            const int s = jj % C::RAW;
            const size_t at = (size_t)(next * a.nkv + it.kvh) * AF_PAGE;
            if (j + 1 < it.pages) next = page_id(it, j + 1);
            if (!mbar_wait(&raw_empty[s], ((jj / C::RAW) & 1) ^ 1, give_up)) break;
            unsigned char* st = raw_s + s * C::RAW_STAGE;
            mbar_expect_tx(&raw_full[s], C::RAW_STAGE);
            sh_bulk_load(st, a.k + at * HD, C::CODES, &raw_full[s]);
            sh_bulk_load(st + C::CODES, a.v + at * HD, C::CODES, &raw_full[s]);
            sh_bulk_load(st + 2 * C::CODES, a.k_exp + at, AF_PAGE, &raw_full[s]);
            sh_bulk_load(st + 2 * C::CODES + AF_PAGE, a.v_exp + at, AF_PAGE, &raw_full[s]);
          }
          continue;
        }
        if (n > 0 && !mbar_wait(&ring_free, (n - 1) & 1, give_up)) break;      // (the item before has left the operands' memory)
        for (int j = 0; j < it.pages; ++j, ++jj) {
          const int s = jj % STAGES, row = (next * a.nkv + it.kvh) * AF_PAGE;
          const uint32_t ph = ((jj / STAGES) & 1) ^ 1;
          if (j + 1 < it.pages) next = page_id(it, j + 1);
          if (!mbar_wait(&k_empty[s], ph, give_up)) break;
          mbar_expect_tx(&k_full[s], C::TILE);
#pragma unroll
          for (int c = 0; c < SUB; ++c) tma_load_2d(k_s + s * C::TILE + c * 8192, &map_k, c * 64, row, &k_full[s]);
          if (!mbar_wait(&v_empty[s], ph, give_up)) break;
          mbar_expect_tx(&v_full[s], C::TILE);
#pragma unroll
          for (int c = 0; c < SUB; ++c) tma_load_2d(v_s + s * C::TILE + c * 8192, &map_v, c * 64, row, &v_full[s]);
        }
      }
      if (*give_up) grace_period();
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int jj = 0, n = 0;
      bool ok = true;
      for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x, ++n) {
        const ShItem it = item_of(w);
        ok = mbar_wait(&q_ready, n & 1, give_up);       // (and everything of the item before is read)
        for (int j = 0; j < it.pages && ok; ++j, ++jj) {
          const int s = jj % STAGES;
          ok = mbar_wait(&k_full[s], (jj / STAGES) & 1, give_up);
          // the scores of two pages before are in registers (or, in whose columns P lies, P is consumed)
          if (ok && j >= 2) ok = mbar_wait(APART ? &x_full[jj & 1] : &pv_done[jj & 1], ((jj - 2) >> 1) & 1, give_up);
          if (!ok) break;
          tc_fence_after();
          const uint32_t kt = smem_u32(k_s + s * C::TILE);
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks)
            umma_f16_ts(tmem + (jj & 1) * 64, tmem + Q_COL + ks * 8, umma_desc(kt + (ks >> 2) * 8192) + 2 * (ks & 3), IDESC_S, ks > 0 ? 1u : 0u);
          umma_commit(&s_full[jj & 1]);
          umma_commit(&k_empty[s]);
        }
      }
    }
  } else if (warp == 2) {
    if (lane == 0) {
      int jj = 0;
      bool ok = true;
      for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x) {
        const ShItem it = item_of(w);
        for (int j = 0; j < it.pages && ok; ++j, ++jj) {
          const int s = jj % STAGES;
          ok = mbar_wait(&v_full[s], (jj / STAGES) & 1, give_up) && mbar_wait(&p_full[jj & 1], (jj >> 1) & 1, give_up);
          if (!ok) break;
          tc_fence_after();
          const uint32_t vt = smem_u32(v_s + s * C::TILE);
#pragma unroll
          for (int kk = 0; kk < AF_PAGE / 16; ++kk)
            umma_f16_ts(tmem + O_COL + (jj & 1) * O_STEP, tmem + P_COL + (jj & 1) * P_STEP + kk * 8, umma_desc_mn(vt + kk * 2048, 8192), IDESC_O, (j > (APART ? 1 : 0) || kk > 0) ? 1u : 0u);
          umma_commit(&v_empty[s]);
          umma_commit(&pv_done[jj & 1]);
        }
      }
    }
  } else if (warp >= 4 && warp < 20) {
    // ---- queries, softmax, partial results.  Group g takes the pages whose count is g modulo 2; two threads of a group have a row,
    // each 32 of the page's keys
    constexpr int W = AF_PAGE / 2;
    const int grp = (warp - 4) >> 3, part = ((warp - 4) >> 2) & 1, quad = grp * 2 + part, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    const float ecap = a.cap > 0.f ? 2.f * LOG2E / a.cap : 0.f, capl = a.cap * LOG2E;
    int jj = 0, n = 0;
    bool ok = true;
    pdl_wait();
    pdl_launch_dependents();      // (now, not before: the split kernel behind takes everything in front of this kernel for complete)
    for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x, ++n) {
      const ShItem it = item_of(w);
      const bool live = row < it.rows;
      const bool any = quarter * 32 < it.rows;             // (warps without a row only keep the barriers' count)
      float cs = fabsf(a.cap > 0.f ? a.scale : a.scale * LOG2E);        // (a scale's sign goes to the query)
      const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;
      if (any) {
        // ---- a quarter (heads of 64: half, by two threads) of the row's query into TMEM, two elements a column
        const int rr = it.group0 + row, member = rr / group;
        const int b = live ? a.plan[L.order + it.members0 + member] : 0;
        const __nv_bfloat16* qr = a.q + (size_t)b * a.q_stride + (size_t)(it.kvh * group + (live ? rr - member * group : 0)) * HD;
        constexpr int SHARE = HD == 64 ? 32 : HD / 4, PIECES = SHARE / 8;
        float f1 = 1.f, f2 = 1.f;
        if constexpr (BITS == 8) {
          uint32_t top = 0;
#pragma unroll 4
          for (int c = 0; c < HD / 8; ++c) {
            const uint4 x = live ? *reinterpret_cast<const uint4*>(qr + c * 8) : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t ws[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t lo = ws[e] & 0x7fffu, hi = (ws[e] >> 16) & 0x7fffu;
              top = max(top, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
            }
          }
          const int k = top == 0 ? 14 : max((int)(top >> 7) - 127, -126), up = 14 - k;
          f1 = c8_pow2(up / 2), f2 = c8_pow2(up - up / 2);
          cs *= c8_pow2(-(up / 2)) * c8_pow2(-(up - up / 2));
        }
        if (quad * SHARE < HD) {
#pragma unroll
          for (int c0 = 0; c0 < PIECES; c0 += 4) {
            uint32_t wd[16];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint4 x = live ? *reinterpret_cast<const uint4*>(qr + quad * SHARE + (c0 + c) * 8) : make_uint4(0u, 0u, 0u, 0u);
              wd[4 * c] = x.x, wd[4 * c + 1] = x.y, wd[4 * c + 2] = x.z, wd[4 * c + 3] = x.w;
            }
            if constexpr (BITS == 8) {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const __half2 h = __floats2half2_rn(__uint_as_float(wd[e] << 16) * f1 * f2, __uint_as_float(wd[e] & 0xffff0000u) * f1 * f2);
                wd[e] = *reinterpret_cast<const uint32_t*>(&h);
              }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) wd[e] ^= sign;
            tmem_st16(lane_addr + Q_COL + quad * (SHARE / 2) + c0 * 4, reinterpret_cast<const float*>(wd));
          }
          tmem_wait_st();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready);

      float m_known = SH_NONE, l = 0.f;                     // this thread's sum is relative to m_known
      for (int j = 0; j < it.pages && ok; ++j, ++jj) {
        if ((jj & 1) != grp) continue;
        ok = mbar_wait(&s_full[grp], (jj >> 1) & 1, give_up);
        if (!ok) break;
        if (!any) {
          // (not ahead of the group's other warps: their arrivals for the page before belong to the phase before)
          if (j >= 2) ok = mbar_wait(&p_full[grp], ((jj - 2) >> 1) & 1, give_up);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive(&x_full[grp]);
            if (!APART) mbar_arrive(&m_ready[grp]);
            mbar_arrive(&p_full[grp]);
          }
          continue;
        }
        tc_fence_after();
        float s[W];
        tmem_ld32(lane_addr + grp * 64 + part * W, s);
        tmem_wait_ld();
        const int fp = BITS == 8 ? jj % SH_EXPS : 0;
        const float4* ksp = reinterpret_cast<const float4*>(ks_s[fp] + part * W);
        const float4* lvp = reinterpret_cast<const float4*>(lv_s[fp] + part * W);
        const float4* vsp = reinterpret_cast<const float4*>(vs_s[fp] + part * W);
        // scores are s[c] * cx from here on
        if constexpr (BITS == 8) {
#pragma unroll
          for (int c = 0; c < W; c += 4) {
            const float4 f = ksp[c / 4];
            const ShPair t0 = sh_mul2({s[c], s[c + 1]}, {f.x, f.y}), t1 = sh_mul2({s[c + 2], s[c + 3]}, {f.z, f.w});
            s[c] = t0.x, s[c + 1] = t0.y, s[c + 2] = t1.x, s[c + 3] = t1.y;
          }
        }
        float cx = cs;
        if (a.cap > 0.f) {
          const float ec = ecap * cs;
#pragma unroll
          for (int c = 0; c < W; ++c) s[c] = capl - 2.f * capl * __fdividef(1.f, 1.f + fast_exp2(s[c] * ec));
          cx = 1.f;
        }
        float m4[4] = {SH_NONE, SH_NONE, SH_NONE, SH_NONE};
        float mx;
        if constexpr (BITS == 8) {
#pragma unroll
          for (int c = 0; c < W; c += 4) {
            const float4 f = lvp[c / 4];
            const ShPair t0 = sh_fma2({s[c], s[c + 1]}, {cx, cx}, {f.x, f.y}), t1 = sh_fma2({s[c + 2], s[c + 3]}, {cx, cx}, {f.z, f.w});
            m4[0] = fmaxf(m4[0], t0.x), m4[1] = fmaxf(m4[1], t0.y), m4[2] = fmaxf(m4[2], t1.x), m4[3] = fmaxf(m4[3], t1.y);
          }
          mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        } else {
#pragma unroll
          for (int c = 0; c < W; ++c) m4[c & 3] = fmaxf(m4[c & 3], s[c]);
          mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * cx;
        }
        // the row's maximum over the group's two threads (both have read their scores: the columns may be written again)
        const int turn = (jj >> 1) & 1;      // (a thread may be at its next page before the other one has read)
        mx_s[grp][turn][part][row] = mx;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&x_full[grp]);
        ok = mbar_wait(&x_full[grp], (jj >> 1) & 1, give_up);
        if (!ok) break;
        tc_fence_after();
        mx = fmaxf(mx, mx_s[grp][turn][part ^ 1][row]);
        // the reference after the page before, published by the other group; it moves only when it has to
        float m_prev = APART ? m_known : SH_NONE;
        if (!APART && j > 0) {
          ok = mbar_wait(&m_ready[grp ^ 1], ((jj - 1) >> 1) & 1, give_up);
          if (!ok) break;
          m_prev = mref_s[grp ^ 1][row];
        }
        const float m_new = mx > m_prev + SH_MOVES ? mx : m_prev;
        if constexpr (!APART) {
          if (part == 0) mref_s[grp][row] = m_new;
          __syncwarp();
          if (lane == 0) mbar_arrive(&m_ready[grp]);
        }
        // the group's P of two pages before is consumed (waited for here: it also pins the phase that the wait below looks at)
        if (APART && j >= 2) ok = mbar_wait(&pv_done[grp], ((jj - 2) >> 1) & 1, give_up);
        if (!ok) break;
        if (j > (APART ? 1 : 0) && __any_sync(0xffffffffu, m_new != m_prev)) {
          // O is rescaled once the product of the page before is complete (the next one waits for this page's P)
          if (!APART) ok = mbar_wait(&pv_done[grp ^ 1], ((jj - 1) >> 1) & 1, give_up);
          if (!ok) break;
          tc_fence_after();
          const float f = fast_exp2(m_prev - m_new);
#pragma unroll 1
          for (int c0 = 0; c0 < HD / 2; c0 += 16) {
            float o[16];
            tmem_ld16(lane_addr + O_COL + grp * O_STEP + part * (HD / 2) + c0, o);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] *= f;
            tmem_st16(lane_addr + O_COL + grp * O_STEP + part * (HD / 2) + c0, o);
          }
          tmem_wait_st();
        }
        ShPair sum0 = {0.f, 0.f}, sum1 = {0.f, 0.f};
        uint32_t packed[W / 2];
        if constexpr (BITS == 8) {
          const float ref = m_new - SH_SHIFT;
#pragma unroll
          for (int c = 0; c < W; c += 4) {
            const float4 f = vsp[c / 4];
            const ShPair t0 = sh_fma2({s[c], s[c + 1]}, {cx, cx}, {-ref, -ref}), t1 = sh_fma2({s[c + 2], s[c + 3]}, {cx, cx}, {-ref, -ref});
            const ShPair p0 = {fast_exp2(t0.x), fast_exp2(t0.y)}, p1 = {fast_exp2(t1.x), fast_exp2(t1.y)};
            sum0 = sh_add2(sum0, p0), sum1 = sh_add2(sum1, p1);
            const ShPair w0 = sh_mul2(p0, {f.x, f.y}), w1 = sh_mul2(p1, {f.z, f.w});
            const __half2 h0 = __floats2half2_rn(w0.x, w0.y), h1 = __floats2half2_rn(w1.x, w1.y);
            packed[c / 2] = *reinterpret_cast<const uint32_t*>(&h0);
            packed[c / 2 + 1] = *reinterpret_cast<const uint32_t*>(&h1);
          }
        } else {
#pragma unroll
          for (int c = 0; c < W; c += 2) {
            const ShPair t = sh_fma2({s[c], s[c + 1]}, {cx, cx}, {-m_new, -m_new});
            const __nv_bfloat162 pb = __floats2bfloat162_rn(fast_exp2(t.x), fast_exp2(t.y));
            ShPair& sum = (c >> 1) & 1 ? sum1 : sum0;
            sum = sh_add2(sum, {__low2float(pb), __high2float(pb)});      // (of the rounded weights that the product sees)
            packed[c / 2] = *reinterpret_cast<const uint32_t*>(&pb);
          }
        }
        l = l * fast_exp2(m_known - m_new) + ((sum0.x + sum0.y) + (sum1.x + sum1.y));
        m_known = m_new;
        tmem_st16(lane_addr + P_COL + grp * P_STEP + part * (W / 2), reinterpret_cast<const float*>(packed));
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[grp]);
      }
      if (!ok) break;
      // ---- the item's partial results
      // (First the page before the last: the group that does not own the last page has not seen that the barrier's phase before is
      // complete, and a wait one phase ahead returns at once.  Of that page's barrier it has, or has waited for a product behind it.)
      const int last = jj - 1;
      ok = it.pages < 2 || mbar_wait(&pv_done[(last - 1) & 1], ((last - 1) >> 1) & 1, give_up);
      ok = ok && mbar_wait(&pv_done[last & 1], (last >> 1) & 1, give_up);
      if (!ok) break;
      tc_fence_after();
      if constexpr (APART) {
        if (any) {
          l_s[quad][row] = l;
          if (part == 0) mref_s[grp][row] = m_known;      // (of a group without a page: SH_NONE)
        }
      } else if (any) {
        l_s[quad][row] = l * fast_exp2(m_known - mref_s[last & 1][row]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_full);
      ok = mbar_wait(&l_full, n & 1, give_up);
      if (!ok) break;
      if (any) {
        // the groups' two references become one
        const float m0 = mref_s[0][row], m1 = mref_s[1][row], m_fin = APART ? fmaxf(m0, m1) : mref_s[last & 1][row];
        const float f0 = APART ? fast_exp2(m0 - m_fin) : 1.f, f1 = APART ? fast_exp2(m1 - m_fin) : 1.f;
        const bool has0 = it.pages > 1 || (last & 1) == 0, has1 = it.pages > 1 || (last & 1) == 1;
#pragma unroll 1
        for (int c0 = 0; c0 < HD / 4; c0 += 16) {
          float o[16];
          const int col = quad * (HD / 4) + c0;
          tmem_ld16(lane_addr + O_COL + col, o);
          tmem_wait_ld();
          if constexpr (APART) {
            float o1[16];
            tmem_ld16(lane_addr + O_COL + O_STEP + col, o1);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = (has0 ? o[c] * f0 : 0.f) + (has1 ? o1[c] * f1 : 0.f);
          }
          if (live) {
            unsigned char* dst = k_s + row * (HD * 4);
#pragma unroll
            for (int c = 0; c < 16; c += 4)
              *reinterpret_cast<float4*>(dst + ((((col + c) >> 2) ^ (row & 7)) << 4)) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
          }
        }
        if (live && quad == 0)
          *reinterpret_cast<float2*>(a.part_ml + ((size_t)it.row0 + row) * 2) =
              make_float2(BITS == 8 ? m_fin - SH_SHIFT : m_fin, (l_s[0][row] + l_s[1][row]) * f0 + (l_s[2][row] + l_s[3][row]) * f1);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&staged);
      if (warp == 4) {
        ok = mbar_wait(&staged, n & 1, give_up);
        if (ok && lane == 0) {
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(a.part_o + (size_t)it.row0 * HD), "r"(smem_u32(k_s)),
                       "r"(it.rows * HD * 4)
                       : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          if (w + (int)gridDim.x < n_items) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            mbar_arrive(&ring_free);
          } else {
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
          }
        }
        __syncwarp();
      }
    }
  } else if (BITS == 8 && warp >= 20) {
    // ---- codes to halves.  A page's keys (and values) are 64 rows of HD / 16 pieces of 16 codes; a thread takes PER of them, their
    // codes read before the wait for the operand's place
    constexpr int P_ROW = HD / 16, PER = AF_PAGE * P_ROW / 128, KINDS = C::CONV == 8 ? 1 : 2;
    const int ct = (threadIdx.x - 20 * 32) & 127, kind0 = C::CONV == 8 ? (warp - 20) >> 2 : 0;
    int jj = 0, n = 0;
    bool ok = true;
    for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x, ++n) {
      const ShItem it = item_of(w);
      if (n > 0) ok = mbar_wait(&ring_free, (n - 1) & 1, give_up);      // (the item before has left the operands' memory)
      for (int j = 0; j < it.pages && ok; ++j, ++jj) {
        const int s = jj % STAGES, rs = jj % C::RAW;
        ok = mbar_wait(&raw_full[rs], (jj / C::RAW) & 1, give_up);
#pragma unroll
        for (int kind = kind0; kind < kind0 + KINDS && ok; ++kind) {      // 0: keys, 1: values
          const unsigned char* raw = raw_s + rs * C::RAW_STAGE + kind * C::CODES;
          uint4 w4[PER];
#pragma unroll
          for (int i = 0; i < PER; ++i) w4[i] = *reinterpret_cast<const uint4*>(raw + (ct + i * 128) * 16);
          ok = mbar_wait(kind ? &v_empty[s] : &k_empty[s], ((jj / STAGES) & 1) ^ 1, give_up);
          if (!ok) break;
          unsigned char* tile = (kind ? v_s : k_s) + s * C::TILE;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int x = ct + i * 128, r = x / P_ROW, p = x - r * P_ROW;
            uint4 h[2];
            c8_half4(w4[i].x, h[0].x, h[0].y);
            c8_half4(w4[i].y, h[0].z, h[0].w);
            c8_half4(w4[i].z, h[1].x, h[1].y);
            c8_half4(w4[i].w, h[1].z, h[1].w);
            unsigned char* base = tile + (p >> 2) * 8192 + r * 128;
            const int c = (p & 3) * 2, first = (p >> 2) & 1;        // (neighbouring sub-tiles begin with the other piece: other banks)
            *reinterpret_cast<uint4*>(base + (((c + first) ^ (r & 7)) << 4)) = first ? h[1] : h[0];
            *reinterpret_cast<uint4*>(base + (((c + 1 - first) ^ (r & 7)) << 4)) = first ? h[0] : h[1];
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(kind ? &v_full[s] : &k_full[s]);
            if (kind == kind0 + KINDS - 1) mbar_arrive(&raw_empty[rs]);
          }
        }
      }
    }
  } else if (BITS == 8 && warp == 3) {
    // ---- the factors of a page's rows
    int jj = 0;
    bool ok = true;
    for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x) {
      const ShItem it = item_of(w);
      for (int j = 0; j < it.pages && ok; ++j, ++jj) {
        const int s = jj % STAGES, rs = jj % C::RAW;
        const unsigned char* e = raw_s + rs * C::RAW_STAGE + 2 * C::CODES;
        // (behind the S of STAGES pages before: SH_EXPS pages before nobody reads factors any more, and the arrival is its phase's)
        ok = mbar_wait(&raw_full[rs], (jj / C::RAW) & 1, give_up) && mbar_wait(&k_empty[s], ((jj / STAGES) & 1) ^ 1, give_up);
        if (!ok) break;
#pragma unroll
        for (int c = lane; c < AF_PAGE; c += 32) {
          const uint32_t ke = e[c], ve = e[AF_PAGE + c];
          ks_s[jj % SH_EXPS][c] = __uint_as_float(ke << 23);
          vs_s[jj % SH_EXPS][c] = __uint_as_float(ve << 23);
          lv_s[jj % SH_EXPS][c] = (float)max((int)ve - 127, -60);
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&k_full[s]);
          mbar_arrive(&raw_empty[rs]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  if (threadIdx.x == 0 && give_up_s && a.err) atomicExch(a.err, 1);
}

// ---------------------------------------------------------------- merge

// Threads: four rows of partial results side by side (heads of 256: 256 threads, of 128: 128), with up to eight loads a thread on their way; with more
// blocks than the SMs hold of the large ones two side by side.  (A layer in all, us, 256 / 128 / 64 threads: 64 sequences of 8 heads of 256, 20 items each
// 45.4 / 46.0 / 48.2, 128 sequences of them 47.3 / 44.3 / -; 32 sequences of 32 heads of 128, 18 items 64.3 / 61.4 / 63.3, 128 sequences of
// them 67.3 / 58.6 / -.)
constexpr int SHM_LARGE_AN_SM = 4;
constexpr int SHM_MOST = 1024;     // partial results of a (sequence, head) that the block weighs

// out[b, h] from the items of the shared pages and the splits of the sequence's own.
template <int HD, int THREADS>
__global__ void __launch_bounds__(THREADS)
attn_shared_merge_kernel(__nv_bfloat16* __restrict__ out, long long out_stride, const float* pre_o, const float* pre_ml, const float* own_o,
                         const float* own_ml, int nq, int nkv, int own_room, const int* __restrict__ shared_plan, const int* __restrict__ own_plan,
                         int blocks, const float* __restrict__ sinks) {
  pdl_launch_dependents();
  const int b = blockIdx.x, h = blockIdx.y, batch = gridDim.x, tid = threadIdx.x, lane = tid & 31;
  const int group = nq / nkv, kvh = h / group, units_per_seq = nkv * ((group + 15) / 16);
  const ShPlan L = sh_layout(batch, nq, nkv, blocks);
  const int n_own = own_plan[DA_PLAN_HEAD + b * units_per_seq + kvh * ((group + 15) / 16) + (h % group) / 16];
  int n_pre = 0, rows = 0, turn = 0;
  size_t pre0 = 0;
  const int unit0 = shared_plan[L.loc + 2 * b];
  if (unit0 >= 0) {
    const int rr = shared_plan[L.loc + 2 * b + 1] * group + h % group;
    const int members = shared_plan[L.units + 4 * unit0], tiles = (members * group + SH_ROWS - 1) / SH_ROWS;
    const int* u = shared_plan + L.units + 4 * (unit0 + kvh * tiles + rr / SH_ROWS);
    rows = min(SH_ROWS, members * group - rr / SH_ROWS * SH_ROWS);
    n_pre = u[1];
    pre0 = (size_t)u[2] + rr % SH_ROWS;
    turn = rr & 7;                     // (how the row's pieces lie)
  }
  const size_t own0 = ((size_t)b * nq + h) * own_room;
  __shared__ float f_s[SHM_MOST], l_s[SHM_MOST];
  __shared__ float4 red_s[THREADS];
  pdl_wait();
  pre_o = pdl_fresh(pre_o), pre_ml = pdl_fresh(pre_ml), own_o = pdl_fresh(own_o), own_ml = pdl_fresh(own_ml);
  const int n = n_own + n_pre;         // (own splits first)
  constexpr int ROW = HD / 4, GROUPS = THREADS / ROW;
  const int grp = tid / ROW, d = (tid - grp * ROW) * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = sinks ? sinks[h] * 1.4426950408889634f : -INFINITY, Ls = sinks ? 1.f : 0.f;
  // (more partial results than the block weighs at a time: several rounds)
  for (int base = 0; base < n; base += SHM_MOST) {
    const int m = min(SHM_MOST, n - base);
    __syncthreads();
    float mine = -INFINITY;
    for (int i = tid; i < m; i += THREADS) {
      const int x = base + i;
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(x < n_own ? own_ml + (own0 + x) * 2 : pre_ml + (pre0 + (size_t)(x - n_own) * rows) * 2));
      f_s[i] = ml.x;
      l_s[i] = ml.y;
    }
    __syncthreads();
    for (int i = lane; i < m; i += 32) mine = fmaxf(mine, f_s[i]);
    const float now = fmaxf(M, warp_max(mine)), ref = now == -INFINITY ? 0.f : now;
    const float back = M == -INFINITY ? 0.f : fast_exp2(M - ref);
    acc.x *= back, acc.y *= back, acc.z *= back, acc.w *= back;
    float part = 0.f;
    for (int i = lane; i < m; i += 32) part += l_s[i] * fast_exp2(f_s[i] - ref);
    Ls = Ls * back + warp_sum(part);
    M = now;
    for (int i0 = grp; i0 < m; i0 += 8 * GROUPS) {
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * GROUPS, x = base + i;
        v[u] = i < m ? __ldcg(reinterpret_cast<const float4*>(x < n_own ? own_o + (own0 + x) * HD + d : pre_o + (pre0 + (size_t)(x - n_own) * rows) * HD + (((d >> 2) ^ turn) << 2)))
                     : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * GROUPS;
        const float f = i < m ? fast_exp2(f_s[i] - ref) : 0.f;
        acc.x += v[u].x * f, acc.y += v[u].y * f, acc.z += v[u].z * f, acc.w += v[u].w * f;
      }
    }
  }
  red_s[tid] = acc;
  __syncthreads();
  if (tid < ROW) {
    for (int u = 1; u < GROUPS; ++u) {
      const float4 x = red_s[u * ROW + tid];
      acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
    }
    const float inv = Ls == 0.f ? 0.f : 1.f / Ls;
    __nv_bfloat162* dst = reinterpret_cast<__nv_bfloat162*>(out + (size_t)b * out_stride + (size_t)h * HD + d);
    dst[0] = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
    dst[1] = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
  }
}

template <int HD, int BITS>
int launch_shared(const ShArgs& a, const void* k, const void* v, int blocks, cudaStream_t stream) {
  CUtensorMap mk = {}, mv = {};
  if (BITS == 16) {
    int rc = af_make_map_bf16(&mk, k, a.n_pages * a.nkv * AF_PAGE, HD, HD, AF_PAGE);
    if (rc) return rc;
    rc = af_make_map_bf16(&mv, v, a.n_pages * a.nkv * AF_PAGE, HD, HD, AF_PAGE);
    if (rc) return rc;
  }
  static bool configured[AF_MAX_DEVICES] = {};
  const int dev = af_current_device();
  if (dev < 0) return -1;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_shared_kernel<HD, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh<HD, BITS>::SMEM);
    if (e != cudaSuccess) return af_fail((int)e, "af_attn_decode_shared: %s", cudaGetErrorString(e));
    configured[dev] = true;
  }
  af_launch(attn_shared_kernel<HD, BITS>, dim3(blocks), dim3(Sh<HD, BITS>::THREADS), Sh<HD, BITS>::SMEM, stream, mk, mv, a);
  AF_CHECK_LAUNCH("af_attn_decode_shared (prefix)");
}

}  // namespace


// 32-bit integers of the two plans of a shared step (the prefix kernel's, then the split kernel's), 0 where the sizes are refused.
AF_EXPORT long long af_attn_shared_plan_ints(int batch, int nq, int nkv) {
  if (batch <= 0 || batch > SH_MAX_BATCH || nq <= 0 || nkv <= 0 || nq % nkv) return 0;
  const int sms = af_sm_count();
  if (sms <= 0) return 0;
  return sh_own_plan(sh_layout(batch, nq, nkv, sms)) + af_attn_decode_plan_ints(batch, nq, nkv) + (long long)sms * DA_PLAN_REC;      // (own_blocks: 2 sms at most)
}

// The most partial rows that the prefix kernel leaves (see af_attn_decode_shared).
AF_EXPORT long long af_attn_shared_rows(int batch, int nq, int nkv) {
  const int sms = af_sm_count();
  if (sms <= 0 || batch <= 0 || nq <= 0 || nkv <= 0) return 0;
  // units with several items have at most a block each and up to 128 rows, the others one item
  const int rows = batch * (nq / nkv) < SH_ROWS ? batch * (nq / nkv) : SH_ROWS;
  return (long long)rows * sms + (long long)batch * nq;
}

// Blocks of the split kernel: of the 16-bit cache's two an SM, one after the other: those of SMs that the prefix kernel leaves take more.
static int own_blocks(long long bits, int sms, int nq, int nkv) { return bits == 8 ? d8_blocks(sms, nq, nkv) : 2 * sms; }

// The plans of a step: row b's first pages[b] cache pages are those of row lead[b].
static int shared_plans(int* plan, long long plan_ints, const int* lead, const int* pages, const int* page_table, int max_pages,
                        const int* slots, const int* lens, int batch, int nq, int nkv, int hd, int n_splits, int bits, cudaStream_t stream) {
  const long long need = af_attn_shared_plan_ints(batch, nq, nkv);
  AF_REQUIRE(need > 0, "af_attn_decode_shared: %d sequences (takes %d), %d heads in %d groups", batch, SH_MAX_BATCH, nq, nkv);
  AF_REQUIRE(plan_ints >= need, "af_attn_decode_shared: a plan of %lld integers", need);
  const int sms = af_sm_count(), smem = (10 * batch + 2) * (int)sizeof(int);
  static bool configured[AF_MAX_DEVICES] = {};
  const int dev = af_current_device();
  if (dev < 0) return -1;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_shared_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (10 * SH_MAX_BATCH + 2) * (int)sizeof(int));
    if (e != cudaSuccess) return af_fail((int)e, "af_attn_decode_shared: %s", cudaGetErrorString(e));
    configured[dev] = true;
  }
  const int units_per_seq = nkv * ((nq / nkv + 15) / 16), brk = bits == 8 ? D8_BREAK_PAGES : DA_BREAK_PAGES;
  AF_REQUIRE((long long)batch * (max_pages + 1 + brk) * units_per_seq < (1ll << 31), "af_attn_decode_shared: %d sequences of up to %d pages", batch,
             max_pages);
  af_launch(attn_shared_plan_kernel, dim3(2), dim3(512), smem, stream, plan, lead, pages, slots, lens, page_table, max_pages, batch, nq, nkv, hd,
            sms, n_splits, own_blocks(bits, sms, nq, nkv), brk);
  AF_CHECK_LAUNCH("af_attn_decode_shared (plan)");
}

// What af_attn_decode_shared is given, as one block of 64-bit words.
struct AfShared {
  void* out;
  const void *q, *k, *v, *k_exp, *v_exp, *page_table, *slots, *lens, *lead, *pages;
  float *own_scratch, *pre_scratch;
  int* plan;
  const void* sinks;
  int* err;
  cudaStream_t stream;
  long long out_stride, q_stride, n_pages, max_pages, batch, nq, nkv, hd, n_splits, plan_ints, bits;
  double scale, cap;
};

// out [batch, nq * hd] bfloat16 = attention of one new token per sequence over all its keys, the shared pages read once a
// group.  bits 16: k, v are bfloat16 pages; 8: codes, with k_exp, v_exp.  own_scratch: af_attn_decode_scratch(batch, nq, hd,
// n_splits) floats; pre_scratch: af_attn_shared_rows(...) * (hd + 2) floats.  plan_ints > 0: the step's plans are made first, into
// `plan`'s so many integers; 0: it holds those of a call for the same lead, pages, slots, lengths, page table, heads and n_splits.
AF_EXPORT int af_attn_decode_shared(const AfShared* c) {
  if (c->batch == 0) return 0;
  AF_REQUIRE(c->bits == 8 || c->bits == 16, "af_attn_decode_shared: a cache of 8 or 16 bits, not %lld", c->bits);
  AF_REQUIRE(c->nq > 0 && c->nkv > 0 && c->nq % c->nkv == 0 && c->batch > 0 && c->batch <= SH_MAX_BATCH,
             "af_attn_decode_shared: %lld sequences, heads %lld, groups %lld", c->batch, c->nq, c->nkv);
  AF_REQUIRE(c->hd == 64 || c->hd == 128 || c->hd == 256, "af_attn_decode_shared: head_dim %lld (takes 64, 128, 256)", c->hd);
  AF_REQUIRE(c->q_stride % 8 == 0 && c->out_stride % 2 == 0 &&
                 (((uintptr_t)c->q | (uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->own_scratch | (uintptr_t)c->pre_scratch | (uintptr_t)c->plan) &
                  15) == 0 &&
                 ((uintptr_t)c->out & 3) == 0,
             "af_attn_decode_shared: rows must be 16-byte aligned (out: 4)");
  // (an 8-bit cache's exponents come into shared memory by copies of 16 bytes)
  AF_REQUIRE(c->bits == 16 || (c->k_exp != nullptr && c->v_exp != nullptr && (((uintptr_t)c->k_exp | (uintptr_t)c->v_exp) & 15) == 0),
             "af_attn_decode_shared: exponents must be 16-byte aligned");
  AF_REQUIRE(c->own_scratch != nullptr && c->pre_scratch != nullptr && c->plan != nullptr, "af_attn_decode_shared: scratch and plan");
  AF_REQUIRE(c->n_splits >= 1 && c->n_splits <= 65535, "af_attn_decode_shared: splits %lld", c->n_splits);
  AF_REQUIRE(c->n_pages > 0 && c->n_pages * c->nkv * AF_PAGE < (1ll << 31), "af_attn_decode_shared: %lld cache pages", c->n_pages);
  const int sms = af_sm_count();
  if (sms <= 0) return -1;
  const int batch = (int)c->batch, nq = (int)c->nq, nkv = (int)c->nkv, hd = (int)c->hd, n_splits = (int)c->n_splits, max_pages = (int)c->max_pages;
  const int *page_table = (const int*)c->page_table, *slots = (const int*)c->slots, *lens = (const int*)c->lens;
  int rc;
  if (c->plan_ints > 0) {
    rc = shared_plans(c->plan, c->plan_ints, (const int*)c->lead, (const int*)c->pages, page_table, max_pages, slots, lens, batch, nq, nkv, hd, n_splits,
                      (int)c->bits, c->stream);
    if (rc) return rc;
  }
  const ShPlan L = sh_layout(batch, nq, nkv, sms);
  const int at = sh_own_plan(L);
  const long long rows = af_attn_shared_rows(batch, nq, nkv);
  ShArgs a{(const __nv_bfloat16*)c->q, c->q_stride, (const uint8_t*)c->k, (const uint8_t*)c->v, (const uint8_t*)c->k_exp, (const uint8_t*)c->v_exp,
           c->n_pages, page_table, c->plan, max_pages, batch, nq, nkv, (float)c->scale, (float)c->cap, c->pre_scratch, c->pre_scratch + rows * hd,
           c->err};
  const bool eight = c->bits == 8;
  if (hd == 64)
    rc = eight ? launch_shared<64, 8>(a, c->k, c->v, sms, c->stream) : launch_shared<64, 16>(a, c->k, c->v, sms, c->stream);
  else if (hd == 128)
    rc = eight ? launch_shared<128, 8>(a, c->k, c->v, sms, c->stream) : launch_shared<128, 16>(a, c->k, c->v, sms, c->stream);
  else
    rc = eight ? launch_shared<256, 8>(a, c->k, c->v, sms, c->stream) : launch_shared<256, 16>(a, c->k, c->v, sms, c->stream);
  if (rc) return rc;
  if (eight)
    rc = af_decode8_split(c->q, c->q_stride, c->k, c->v, c->k_exp, c->v_exp, c->n_pages, page_table, max_pages, slots, lens, c->plan + L.shared,
                          batch, nq, nkv, hd, a.scale, a.cap, 0, 0, 0, n_splits, c->own_scratch, c->plan + at, c->err, c->stream, nullptr, 0, nullptr);
  else
    rc = af_decode16_split(c->q, c->q_stride, c->k, c->v, c->n_pages, page_table, max_pages, slots, lens, c->plan + L.shared, batch, nq, nkv, hd,
                           a.scale, a.cap, n_splits, c->own_scratch, c->plan + at, own_blocks(16, sms, nq, nkv), c->err, c->stream);
  if (rc) return rc;
  const bool large = hd == 256 && (long long)batch * nq <= (long long)SHM_LARGE_AN_SM * sms;
  const auto merge = hd == 64    ? attn_shared_merge_kernel<64, 128>
                     : hd == 128 ? attn_shared_merge_kernel<128, 128>
                     : large     ? attn_shared_merge_kernel<256, 256>
                                 : attn_shared_merge_kernel<256, 128>;
  af_launch(merge, dim3(batch, nq), dim3(large ? 256 : 128), 0, c->stream, (__nv_bfloat16*)c->out, c->out_stride, (const float*)a.part_o,
            (const float*)a.part_ml, (const float*)c->own_scratch, (const float*)c->own_scratch + (size_t)batch * nq * n_splits * hd, nq, nkv,
            n_splits, (const int*)c->plan, (const int*)c->plan + at, sms, (const float*)c->sinks);
  AF_CHECK_LAUNCH("af_attn_decode_shared (merge)");
}
