// What the split decode attentions share (attention_decode.cu: the 16-bit cache; attention_decode8.cu: the 8-bit one): how a
// step's work is cut among the blocks, the format of its plan, and (16 bits) the merge of the partial results.
#pragma once
#include "tma.cuh"

namespace {

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The first position that the token at `pos` sees.  window > 0: the last `window` positions, itself included;
// window < 0: those of its own chunk of -window positions (chunks counted from position 0); 0: all.
__device__ __forceinline__ int da_lo(int pos, int window) {
  return window > 0 ? max(0, pos - window + 1) : (window < 0 ? pos - pos % (-window) : 0);
}

// The pages of a sequence that its token at `pos` attends to: the pages of the kept first tokens, then the window's up to
// the token's own.  The pages count through; `skip` of them lie between the two parts.  `shared` (all keys visible): so many
// first pages are left to another kernel (attention_shared.cu); the token's own page never is.
struct DaList {
  int kept, skip, n;
};
__device__ __forceinline__ DaList da_list(int pos, int window, int keep, int shared) {
  DaList l;
  l.kept = af_kept_pages(keep);
  l.skip = max(max(0, da_lo(pos, window) / AF_PAGE - l.kept), shared);
  l.n = pos / AF_PAGE + 1 - l.skip;
  return l;
}
__device__ __forceinline__ int da_page_of(int kept, int skip, int x) { return x >= kept ? x + skip : x; }

// How many pages of the cache sequence b's new token attends to.
__device__ __forceinline__ int da_pages(const int* slots, const int* lens, int b, int window, int keep,
                                        const int* shared) {
  const int slot = slots[b], len_b = lens[b];   // (both loads at once: neither waits for the other)
  const int len = slot >= 0 ? len_b : 0;
  return len > 0 ? da_list(len - 1, window, keep, shared != nullptr ? shared[b] : 0).n : 0;
}

// ---------------------------------------------------------------- how the work is cut

constexpr int DA_MAX_BATCH = 2048;   // sequences whose page counts a block keeps in shared memory

// The blocks that share the work in the run cut.  A unit of P pages lies in at most P + 1 runs and in at most
// n_blocks / units_per_seq + 2 (a run is at least total / n_blocks pages, and the unit's sequence alone has
// units_per_seq * P): if the room for partial results, `room` a unit, is below both, fewer blocks work, so that
// no unit is cut more often than it has room for.
__device__ __forceinline__ int da_blocks_used(int n_blocks, int room, int units_per_seq, int most_pages) {
  if (room >= most_pages + 1 || room >= n_blocks / units_per_seq + 2) return n_blocks;
  return max(1, min(n_blocks, (room - 2) * units_per_seq));
}

// Splits of a unit of P pages in the even cut: pages / share, rounded to the nearest (how 1), down (how 2) or up (how 3).
__device__ __forceinline__ int da_even_splits(int P, int share, int room, int how) {
  return P > 0 ? max(1, min(room, (P + (how == 1 ? share / 2 : (how == 3 ? share - 1 : 0))) / share)) : 0;
}

// What a block loses at the end of a unit inside its run (merging, the next unit's queries, the first page's
// wait), in pages: the even cut is taken if its largest split is no more than this above the share, and in the run cut a unit
// of P pages takes P and a break of a run, the break first.  (Runs of equal pages left the blocks that met
// many short sequences behind.  Measured with heads of 256, two a tile: 64 sequences of 10 to 2,048 tokens, 256 units of which 88 have one page: a decode step of 26 layers
// 2,412 -> 2,267 us.)
constexpr int DA_BREAK_PAGES = 2;
// The same for the 8-bit cache, whose pages take half as long.  (64 sequences of up to 8,192 tokens, a window of 4,096, 8 kv heads of 256: with 2, 4 and
// 6 pages 88.4, 76.3 and 78.3 us.)
constexpr int D8_BREAK_PAGES = 4;
// Blocks of the 8-bit split kernel: two an SM (a block's end of a unit then falls into the other's work) where their registers fit.  (The same step
// with one an SM: 105 us.)
inline int d8_blocks(int sms, int nq, int nkv) { return nq / nkv <= 8 ? 2 * sms : sms; }
static_assert(DA_BREAK_PAGES != D8_BREAK_PAGES, "da_plan and the plans' marks tell the two caches apart by their breaks");
__device__ __forceinline__ int da_plan_mark(int blocks, int brk) { return blocks | (brk << 16); }

struct DaPlan {
  int share;        // pages a block should get (the run cut: with the units' breaks)
  int n_blocks;     // blocks that work in the run cut
  int brk;          // the break
  int even;         // 0: the run cut; else the even cut, and how it rounds (da_even_splits)
  int pages_before; // pages of the sequences before `b_query` (each counted once, not per unit; the run cut: with breaks)
};

// The plan, by one whole warp (every lane returns the same).  32-bit arithmetic all through: the launcher has
// checked that batch x (pages + break) x units stays below 2^31.  If `pages_s` is given it gets the pages of the sequences
// before b (the run cut: with a break for each that has any), and `splits_s` their splits in the even cut (b = 0 .. batch).
__device__ __forceinline__ DaPlan da_plan(const int* slots, const int* lens, int batch, int window, int keep,
                                          const int* shared, int brk, int units_per_seq, int grid_blocks, int room, int b_query, int* pages_s, int* splits_s) {
  const int lane = threadIdx.x & 31;
  int carry = 0, most = 0, before = 0, P_first = 0, live = 0, live_before = 0;
  if (pages_s && lane == 0) pages_s[0] = 0;
  for (int base = 0; base < batch; base += 32) {
    const int i = base + lane;
    const int P = i < batch ? da_pages(slots, lens, i, window, keep, shared) : 0;
    if (base == 0) P_first = P;
    most = max(most, P);
    if (i < b_query) before += P, live_before += P > 0 ? 1 : 0;
    live += P > 0 ? 1 : 0;
    int v = P;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    if (pages_s && i < batch) pages_s[i + 1] = carry + v;
    carry += __shfl_sync(0xffffffffu, v, 31);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  DaPlan pl;
  pl.brk = brk;
  pl.pages_before = __reduce_add_sync(0xffffffffu, before);
  const int total = carry * units_per_seq;
  pl.n_blocks = da_blocks_used(grid_blocks, room, units_per_seq, most);
  pl.share = max(1, (total + pl.n_blocks - 1) / pl.n_blocks);
  // the even cut, rounding either way: how many splits in all, and the most pages of one.  (Rounding up is the 8-bit cache's alone: its
  // blocks are small and many, so that where the splits still fit them no block has more than its share.  8 sequences of 2,049 tokens, 4 kv
  // heads, 296 blocks: 9 splits of up to 4 pages instead of 8 of up to 5,
  // a layer 15.1 -> 14.3 us.)
  const bool up = brk == D8_BREAK_PAGES;
  int items1 = 0, worst1 = 0, items2 = 0, worst2 = 0, items3 = 0, worst3 = 0;
  for (int base = 0; base < batch; base += 32) {
    const int i = base + lane;
    const int P = base == 0 ? P_first : (i < batch ? da_pages(slots, lens, i, window, keep, shared) : 0);
    const int sp1 = da_even_splits(P, pl.share, room, 1), sp2 = da_even_splits(P, pl.share, room, 2);
    const int sp3 = up ? da_even_splits(P, pl.share, room, 3) : 0;
    if (P > 0) {
      worst1 = max(worst1, (P + sp1 - 1) / sp1);
      worst2 = max(worst2, (P + sp2 - 1) / sp2);
      if (up) worst3 = max(worst3, (P + sp3 - 1) / sp3);
    }
    items1 += sp1;
    items2 += sp2;
    items3 += sp3;
  }
  items1 = __reduce_add_sync(0xffffffffu, items1);
  items2 = __reduce_add_sync(0xffffffffu, items2);
  worst1 = __reduce_max_sync(0xffffffffu, worst1);
  worst2 = __reduce_max_sync(0xffffffffu, worst2);
  const bool fits1 = items1 * units_per_seq <= grid_blocks, fits2 = items2 * units_per_seq <= grid_blocks;
  int how = 0, worst = 0;
  if (fits1 && (!fits2 || worst1 <= worst2)) how = 1, worst = worst1;
  else if (fits2) how = 2, worst = worst2;
  if (up) {
    items3 = __reduce_add_sync(0xffffffffu, items3);
    worst3 = __reduce_max_sync(0xffffffffu, worst3);
    if (items3 * units_per_seq <= grid_blocks && (how == 0 || worst3 < worst)) how = 3, worst = worst3;
  }
  pl.even = (how != 0 && worst <= pl.share + brk) ? how : 0;
  if (!pl.even) {
    live = __reduce_add_sync(0xffffffffu, live);
    pl.pages_before += brk * __reduce_add_sync(0xffffffffu, live_before);
    pl.share = max(1, ((carry + brk * live) * units_per_seq + pl.n_blocks - 1) / pl.n_blocks);
    if (pages_s) {
      int breaks = 0;
      for (int base = 0; base < batch; base += 32) {
        const int i = base + lane;
        const int P = base == 0 ? P_first : (i < batch ? da_pages(slots, lens, i, window, keep, shared) : 0);
        const uint32_t with = __ballot_sync(0xffffffffu, P > 0);
        if (i < batch) pages_s[i + 1] += brk * (breaks + __popc(with & (0xffffffffu >> (31 - lane))));
        breaks += __popc(with);
      }
    }
  }
  if (splits_s && pl.even) {
    int items = 0;
    if (lane == 0) splits_s[0] = 0;
    for (int base = 0; base < batch; base += 32) {
      const int i = base + lane;
      const int P = base == 0 ? P_first : (i < batch ? da_pages(slots, lens, i, window, keep, shared) : 0);
      int v = da_even_splits(P, pl.share, room, pl.even);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
      }
      if (i < batch) splits_s[i + 1] = items + v;
      items += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  return pl;
}

// The largest b in [0, n) with arr[b] * scale <= x (arr ascends, arr[0] = 0).
__device__ __forceinline__ int da_find(const int* arr, int n, int scale, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (arr[mid] * scale <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// What block w begins with: pages [p_in, p_in + n_pages) of unit y of sequence b, the unit's split z; run_left is what
// its run holds behind that unit, pages and breaks (in the run cut it goes on with the units that follow).  n_pages < 0: the
// block has no work.
struct DaFirst {
  int n_pages, b, y, z, p_in, run_left;
};

__device__ __forceinline__ DaFirst da_first_segment(const DaPlan& pl, const int* pages_s, const int* splits_s, int batch,
                                                    int units_per_seq, int w) {
  DaFirst fs;
  fs.n_pages = -1;
  fs.b = fs.y = fs.z = fs.p_in = fs.run_left = 0;
  if (pl.even) {
    // split z of unit y of sequence b, one of da_even_splits(...) equal parts of its pages
    if (w >= splits_s[batch] * units_per_seq) return fs;
    const int b = da_find(splits_s, batch, units_per_seq, w);
    const int sp = splits_s[b + 1] - splits_s[b], P = pages_s[b + 1] - pages_s[b];
    const int r = w - splits_s[b] * units_per_seq;
    const int per = (P + sp - 1) / sp;
    fs.b = b;
    fs.y = r / sp;
    fs.z = r - fs.y * sp;
    fs.p_in = fs.z * per;
    fs.n_pages = max(0, min(per, P - fs.p_in));   // (0: the unit has fewer pages than splits; an empty partial result)
    return fs;
  }
  // the run cut: [gpos, gend) of all units end to end, a unit's break and then its pages
  const int total = pages_s[batch] * units_per_seq;
  const int gpos = w * pl.share, gend = min(total, gpos + pl.share);
  if (w >= pl.n_blocks || gpos >= gend) return fs;
  const int b = da_find(pages_s, batch, units_per_seq, gpos);
  const int width = pages_s[b + 1] - pages_s[b];
  const int y = (gpos - pages_s[b] * units_per_seq) / width;
  const int unit0 = pages_s[b] * units_per_seq + y * width, page0 = unit0 + pl.brk;
  const int p_in = max(0, gpos - page0), n_pages = min(width - pl.brk, gend - page0) - p_in;
  if (n_pages <= 0) return fs;                // (the run lies in a break)
  fs.b = b;
  fs.y = y;
  fs.p_in = p_in;
  fs.n_pages = n_pages;
  fs.run_left = max(0, gend - unit0 - width);
  fs.z = w - page0 / pl.share;                // (the run may begin inside a unit: then it is not the unit's first split)
  return fs;
}
// The runs that hold pages of a unit whose break begins at unit0.
__device__ __forceinline__ int da_run_splits(int unit0, int P, int share, int brk) {
  return P > 0 ? (unit0 + brk + P - 1) / share - (unit0 + brk) / share + 1 : 0;
}

// ---------------------------------------------------------------- the plan of a step
//
// The cut depends on the step's lengths alone, so the layers that read the same caches the same way (one group of
// layers) can share it: a small kernel works it out once, and each layer's blocks read their first segment from
// it with one load, where otherwise each block loads slots and lengths, works out the cut and loads page ids,
// one after the other, before its first copy can start.  The plan, 32-bit integers:
//   [0, 8)                    room (splits a unit may have), grid blocks | break << 16, sequences, units a sequence, how cut
//   [8, 8 + sequences*units)  the splits of every unit, for the merge
//   then 16 a block           n_pages (< 0: no work), b, y, z, p_in, run_left, position of the new token, slot,
//                             the cache pages of the segment's first four pages, the sequence's pages left to another kernel
//   then (the 8-bit cache)    a zero for every unit: how many of its splits are there in the layer at hand
constexpr int DA_PLAN_HEAD = 8;
constexpr int DA_PLAN_REC = 16;

__host__ __device__ inline long long da_plan_records_at(int batch, int units_per_seq) {
  return DA_PLAN_HEAD + (((long long)batch * units_per_seq + 3) / 4) * 4;
}

// Writes the plan, by a whole block; smem: 2 (batch + 1) integers.
__device__ __forceinline__ void da_write_plan(int* plan, const int* slots, const int* lens, const int* page_table, int max_pages, int batch,
                                              int nq, int nkv, int window, int keep, int ring_rows, int room, int grid_blocks,
                                              const int* shared, int brk, int* dp_smem, bool counts = false) {
  int* pages_s = dp_smem;                 // [batch + 1]
  int* splits_s = dp_smem + batch + 1;    // [batch + 1]
  __shared__ DaPlan plan_s;
  const int group = nq / nkv, tiles = (group + 15) / 16, units_per_seq = nkv * tiles;
  if (threadIdx.x < 32) {
    const DaPlan pl = da_plan(slots, lens, batch, window, keep, shared, brk, units_per_seq, grid_blocks, room, 0, pages_s, splits_s);
    if (threadIdx.x == 0) plan_s = pl;
  }
  __syncthreads();
  const DaPlan pl = plan_s;
  if (threadIdx.x == 0) {
    plan[0] = room;
    plan[1] = da_plan_mark(grid_blocks, brk);
    plan[2] = batch;
    plan[3] = units_per_seq;
    plan[4] = pl.even;
    plan[5] = pl.share;
    plan[6] = pl.n_blocks;
    plan[7] = 0;
  }
  for (int u = threadIdx.x; u < batch * units_per_seq; u += blockDim.x) {
    const int b = u / units_per_seq, y = u - b * units_per_seq;
    const int width = pages_s[b + 1] - pages_s[b];      // (the run cut: with a break)
    plan[DA_PLAN_HEAD + u] = pl.even ? da_even_splits(width, pl.share, room, pl.even)
                                     : da_run_splits(pages_s[b] * units_per_seq + y * width, width - brk, pl.share, brk);
  }
  int* recs = plan + da_plan_records_at(batch, units_per_seq);
  if (counts)
    for (int u = threadIdx.x; u < batch * units_per_seq; u += blockDim.x) recs[grid_blocks * DA_PLAN_REC + u] = 0;
  for (int w = threadIdx.x; w < grid_blocks; w += blockDim.x) {
    const DaFirst fs = da_first_segment(pl, pages_s, splits_s, batch, units_per_seq, w);
    int* r = recs + (size_t)w * DA_PLAN_REC;
    int pos = 0, slot = 0, first = 0, ids[4] = {0, 0, 0, 0};
    if (fs.n_pages >= 0) {
      pos = lens[fs.b] - 1;
      slot = slots[fs.b];
      if (shared != nullptr) first = shared[fs.b];
      const DaList l = da_list(pos, window, keep, first);
      for (int i = 0; i < 4 && i < fs.n_pages; ++i) {
        const int entry = af_cache_row(da_page_of(l.kept, l.skip, fs.p_in + i) * AF_PAGE, ring_rows, keep) / AF_PAGE;
        int page = AF_INDEX_OK(entry < max_pages, entry) && entry < max_pages ? page_table[(size_t)slot * max_pages + entry] : 0;
        if (!AF_INDEX_OK(page >= 0, page) || page < 0) page = 0;
        ids[i] = page;
      }
    }
    reinterpret_cast<int4*>(r)[0] = make_int4(fs.n_pages, fs.b, fs.y, fs.z);
    reinterpret_cast<int4*>(r)[1] = make_int4(fs.p_in, fs.run_left, pos, slot);
    reinterpret_cast<int4*>(r)[2] = make_int4(ids[0], ids[1], ids[2], ids[3]);
    reinterpret_cast<int4*>(r)[3] = make_int4(first, 0, 0, 0);
  }
}

// ---------------------------------------------------------------- pass 2

constexpr int DA_MERGE_FEW = 8;        // up to this many splits: 128 threads, every load at once
constexpr int DA_MERGE_THREADS = 512;  // more, and few (sequence, head) pairs: groups of threads take the splits in turn
constexpr int DA_MERGE_MOST = 512;     // splits whose (max, sum) the block keeps in shared memory

// Merges the splits of (sequence, head), cut as the split kernel cut them (da_plan with that kernel's grid).
template <int HD>
__global__ void attn_decode_merge_kernel(__nv_bfloat16* __restrict__ out, long long out_stride,
                                         const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                         int nq, int nkv, int max_splits, const int* __restrict__ slots,
                                         const int* __restrict__ lens, int window, int keep, int grid_blocks,
                                         const int* __restrict__ plan, const float* __restrict__ sinks) {
  pdl_launch_dependents();
  const int b = blockIdx.x, h = blockIdx.y, batch = gridDim.x;
  // (the splits' maxima are base-2 exponents: the sink, a natural one, is brought there; a weight, not a result)
  const float sink2 = sinks ? sinks[h] * 1.4426950408889634f : -INFINITY;
  const size_t p0 = ((size_t)b * nq + h) * max_splits;
  __shared__ DaPlan plan_s;
  __shared__ float m_sh[DA_MERGE_MOST], l_sh[DA_MERGE_MOST];
  __shared__ float red_s[DA_MERGE_THREADS * 2];
  const int group = nq / nkv, tiles = (group + 15) / 16, units_per_seq = nkv * tiles;
  // (the plan, or slots and lengths, are inputs of the step: the cut is known before the wait)
  int n_splits;
  if (plan != nullptr) {
    n_splits = ld_keep_int(plan + DA_PLAN_HEAD + b * units_per_seq + (h / group) * tiles + (h % group) / 16, l2_policy_keep());
  } else {
    if (threadIdx.x < 32) {
      const DaPlan pl = da_plan(slots, lens, batch, window, keep, nullptr, DA_BREAK_PAGES, units_per_seq, grid_blocks, max_splits, b, nullptr,
                                nullptr);
      if (threadIdx.x == 0) plan_s = pl;
    }
    __syncthreads();
    const int P = da_pages(slots, lens, b, window, keep, nullptr);
    if (plan_s.even) {
      n_splits = da_even_splits(P, plan_s.share, max_splits, plan_s.even);
    } else {
      const int y = (h / group) * tiles + (h % group) / 16;
      n_splits = da_run_splits(plan_s.pages_before * units_per_seq + y * (P + DA_BREAK_PAGES), P, plan_s.share, DA_BREAK_PAGES);
    }
  }
  pdl_wait();
  // (the number of splits is known before the wait and the loads below depend on nothing else: without
  // this the compiler may move them, through the const __restrict__ pointers, above the wait)
  part_o = pdl_fresh(part_o);
  part_ml = pdl_fresh(part_ml);
  __nv_bfloat16* dst = out + (size_t)b * out_stride + (size_t)h * HD;
  if (n_splits <= DA_MERGE_FEW) {
    // few splits: every load (outputs, maxima, sums) is issued before the first use, one round trip
    constexpr int FEW = DA_MERGE_FEW;
    constexpr int PER = HD > 128 ? HD / 128 : 1;
    const int d = threadIdx.x;   // HD >= 128: threads 0..127 take d and d + 128 (HD 256)
    if (d >= 128 || d >= HD) return;
    float o[FEW][PER], m[FEW], l[FEW];
#pragma unroll
    for (int s = 0; s < FEW; ++s) {
      const bool on = s < n_splits;
      m[s] = on ? part_ml[(p0 + s) * 2] : -INFINITY;
      l[s] = on ? part_ml[(p0 + s) * 2 + 1] : 0.f;
#pragma unroll
      for (int e = 0; e < PER; ++e) o[s][e] = on ? part_o[(p0 + s) * HD + d + e * 128] : 0.f;
    }
    float M = -INFINITY;
#pragma unroll
    for (int s = 0; s < FEW; ++s) M = fmaxf(M, m[s]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, O[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) O[e] = 0.f;
#pragma unroll
    for (int s = 0; s < FEW; ++s) {
      const float f = fast_exp2(m[s] - ref);
      L += l[s] * f;
#pragma unroll
      for (int e = 0; e < PER; ++e) O[e] += o[s][e] * f;
    }
    if (sinks) L += exp2f(sink2 - ref);
    const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) dst[d + e * 128] = __float2bfloat16_rn(O[e] * inv);
    return;
  }
  if (n_splits <= DA_MERGE_MOST && blockDim.x % (HD / 2) == 0) {
    // many splits, three round trips: (max, sum) of every split at once; the outputs, the splits dealt to
    // groups of HD / 2 threads (two dims a thread), eight loads in flight each; the groups' sums through shared memory
    const int tid = threadIdx.x;
    for (int s = tid; s < n_splits; s += (int)blockDim.x) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml + (p0 + s) * 2));
      m_sh[s] = ml.x;
      l_sh[s] = ml.y;
    }
    __syncthreads();
    float M = -INFINITY;
    for (int s = tid & 31; s < n_splits; s += 32) M = fmaxf(M, m_sh[s]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    for (int s = tid & 31; s < n_splits; s += 32) L += l_sh[s] * fast_exp2(m_sh[s] - ref);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (sinks) L += exp2f(sink2 - ref);
    constexpr int ROW = HD / 2;                       // threads of a group
    const int GROUPS = (int)blockDim.x / ROW;         // (1 .. 16)
    const int grp = tid / ROW, dp = tid - grp * ROW;
    float2 acc = make_float2(0.f, 0.f);
    int s = grp;
    for (; s + 7 * GROUPS < n_splits; s += 8 * GROUPS) {
      float2 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = __ldcg(reinterpret_cast<const float2*>(part_o + (p0 + s + u * GROUPS) * HD) + dp);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float f = fast_exp2(m_sh[s + u * GROUPS] - ref);
        acc.x += v[u].x * f;
        acc.y += v[u].y * f;
      }
    }
    {
      float2 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = s + u * GROUPS < n_splits ? __ldcg(reinterpret_cast<const float2*>(part_o + (p0 + s + u * GROUPS) * HD) + dp)
                                         : make_float2(0.f, 0.f);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float f = s + u * GROUPS < n_splits ? fast_exp2(m_sh[s + u * GROUPS] - ref) : 0.f;
        acc.x += v[u].x * f;
        acc.y += v[u].y * f;
      }
    }
    red_s[tid * 2] = acc.x;
    red_s[tid * 2 + 1] = acc.y;
    __syncthreads();
    if (tid < ROW) {
      float2 O = make_float2(0.f, 0.f);
      for (int gq = 0; gq < GROUPS; ++gq) {
        O.x += red_s[(gq * ROW + tid) * 2];
        O.y += red_s[(gq * ROW + tid) * 2 + 1];
      }
      const float inv = L > 0.f ? 1.f / L : 0.f;
      *reinterpret_cast<__nv_bfloat162*>(dst + 2 * tid) = __floats2bfloat162_rn(O.x * inv, O.y * inv);
    }
    return;
  }
  // (more splits than the block keeps: one after the other)
  float M = -INFINITY;
  for (int s = 0; s < n_splits; ++s) M = fmaxf(M, part_ml[(p0 + s) * 2]);
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  for (int s = 0; s < n_splits; ++s) L += part_ml[(p0 + s) * 2 + 1] * fast_exp2(part_ml[(p0 + s) * 2] - ref);
  if (sinks) L += exp2f(sink2 - ref);
  const float inv = L > 0.f ? 1.f / L : 0.f;
  for (int dd = threadIdx.x; dd < HD; dd += blockDim.x) {
    float O = 0.f;
    for (int s = 0; s < n_splits; ++s) O += part_o[(p0 + s) * HD + dd] * fast_exp2(part_ml[(p0 + s) * 2] - ref);
    dst[dd] = __float2bfloat16_rn(O * inv);
  }
}

}  // namespace
