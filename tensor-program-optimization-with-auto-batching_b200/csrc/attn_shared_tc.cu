// Decode attention of a batch whose rows share long prefixes: the pages of a shared prefix are read once for all rows that have it
// (the page-sharing counterpart of attention_with_fused_qkv, tvm/llama_auto_batcher/llama_for_causal_lm.py:55-64).
//
// softmax(q K^T) V over the keys of a row falls into ranges: with m, l and O the maximum (or what is near it), the sum of exp(s - m) and the sum of
// exp(s - m) v of a range, two ranges make one with m = max(m1, m2), l = l1 e^(m1 - m) + l2 e^(m2 - m), O likewise.  So
//
//   prefix_plan_kernel     groups the rows of a step by the prefix their slot names (once a step, for all layers);
//   prefix_attn_kernel     the prefix: up to 128 (row, query head) pairs that share a key head are the M rows of one tcgen05 tile, a CTA
//                          takes a range of the prefix's keys and leaves m, l, O of its pairs in scratch;
//   tail_attn_kernel       what follows the prefix, row by row, and the join of everything.
//
// The prefix has 2 D 2 bytes per key and key head against 4 D 128 flops of a full tile: bound by HBM up to some 128 pairs (rows x query
// heads per key head) -- for few pairs by the chain scores, softmax, products of a block, which 32 of a tile's rows do not shorten --, by
// what comes through L2 beyond.  The tail is bound by HBM alone: its tiles have only the query heads of one key head, so it uses mma.sync with 16
// keys as the rows and up to eight heads as the columns, and a ring of TMA copies in every warp.  It is launched programmatically
// dependent on the prefix and waits for it only before the join.
// Measured (CUDA graph, three or four sets of inputs in turn): 32 rows x 32 heads behind 4096 tokens 60.5 us (3.9 TB/s of the keys and values
// read once), 72 rows x 40 heads in four groups 153 us (5.8 TB/s), 128 rows x 32 heads over 8 key heads behind 32768 tokens 138 us (498
// TFLOP/s; every tile reads the prefix through L2: 537 MB), 4 rows behind 512 tokens 12.2 us.  Call after call the second and third come to the
// power limit and take 158 and 147 us.  Exponentials partly on the FMA units (2 % more) and steps of 64 keys with two places for everything
// (18 % more) were no faster in the third.
#include <math.h>

#include <atomic>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace mlora {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 128;               // (row, query head) pairs of a tile = keys of a block
constexpr int kSub = kTile * 64 * 2;     // one [128 x 64] bf16 sub-tile: 16 KB
// A pair's scores are taken against a reference that follows their running maximum only when that is more than 2^kGrow above it: the
// reference cancels, fp32 sums and weights of 16 bits round those of up to 2^8 no more than those of up to 1, and O stays in TMEM (following
// every maximum takes 128 x 32768 5 % more).
constexpr float kGrow = 8.f;
constexpr int kPxThreads = 192;          // warps 0..3: one thread per pair; 4: MMA issue, copies of keys; 5: copies of values
constexpr int kPxRegs = 128;             // two CTAs per SM leave room for the tail's (72 rows x 40 heads: 10 % more time with 168)
constexpr int kPlanMaxRows = 1024;
constexpr int kPlanHeader = 8;           // int32: rows, tiles, items, parts
constexpr int kTickets = 1024;           // arrival counters at the start of the scratch, whatever the call's sizes: zero between calls
constexpr int kPlanMinRows = 2, kPlanMinKeys = 64;  // smaller groups and shorter prefixes are read row by row
// Groups that are taken together where the caller does not say what they have to save: the second kernel has a chain of blocks and a join to go
// through, so it takes rows enough to read a prefix again for, and a prefix that is long, or saves many reads ((rows - 1) x tokens x key
// heads).  Measured, shared and row by row, us, one group of rows x tokens, heads of 128 (8 key heads
// of 4 query heads | 32 of one | one of 8) and of 64 (8 of 4):
//    2 x 8192    21.5  21.0 |  44.1  37.1 |  21.1  22.4 |  17.6  16.3
//    2 x 32768   44.9  42.3 |   122   116 |  34.0  37.5 |  36.0  32.0
//    4 x 1024    13.2  15.1 |  17.3  16.7 |  12.5  14.5 |  11.5  13.3
//    4 x 8192    21.9  24.6 |  44.0  51.5 |  21.3  22.8 |  17.9  19.3
//    8 x 512     12.8  13.0 |  16.7  15.9 |  12.8  12.3 |  10.7  11.1
//    8 x 1024    13.3  16.1 |  18.2  28.2 |  12.9  14.5 |  11.3  14.0
//   32 x 512     15.8  15.8 |  28.6  40.5 |  14.3  12.6 |  12.5  12.9
//   32 x 8192    31.0   127 |  56.8   347 |  23.5  28.0 |  22.1  62.6
// Over 784 such cases (2 to 32 rows, 256 to 32768 tokens, 1 to 40 key heads) no group that is taken together loses more than 9 %.
constexpr int kPlanEnoughRows = 4, kPlanLongKeys = 1024, kPlanManyReads = 200000;
__host__ __device__ inline bool taken_together(int rows, int keys, int Hkv, long long least) {
  const long long saved = (long long)(rows - 1) * keys * Hkv;
  return rows >= kPlanMinRows && keys >= kPlanMinKeys &&
         (least >= 0 ? saved >= least : rows >= kPlanEnoughRows && (keys >= kPlanLongKeys || saved >= kPlanManyReads));
}
// Key ranges that a row's CTA joins in the time of a block, with kJoin of them on their way: some 0.15 us against 2.5 (2 rows behind 32768
// tokens of one key head, 256 blocks: in 256 ranges 178 us with one range after the other and 72 with kJoin, in some 50 ranges 35; ranges
// chosen with 6 here in place of 18 cost 5 to 12 % on average over 2 to 32 rows behind 2048 to 32768 tokens of 1 to 40 key heads).
constexpr int kBlockParts = 18;

// A plan in int32: header; per row a quad (first key of its own part, its first part, its parts, 0) and its entry of `list` (rows by group);
// then two quads per item, all that a CTA needs to begin: (slot whose pages are read, first block, blocks, keys of the prefix | first entry
// of `list`, rows, key head, key range).
struct PlanView {
  int32_t* head;
  int4* row;
  int32_t* list;
  int4* item;
};
__host__ __device__ inline PlanView plan_view(int32_t* p, int max_rows) {
  PlanView v;
  v.head = p;
  v.row = reinterpret_cast<int4*>(p + kPlanHeader);
  v.list = p + kPlanHeader + 4 * max_rows;
  v.item = reinterpret_cast<int4*>(v.list + (max_rows + 3) / 4 * 4);
  return v;
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = 148;
  }
  return n;
}

// Items of a call: a tile has at least kPlanMinRows rows, and more where it is full, so there are at most T / kPlanMinRows tiles.
int max_items_of(int T, int Hkv, int target) {
  const long long tiles = T / kPlanMinRows;
  return tiles == 0 ? 0 : (int)(tiles * Hkv > target ? tiles * Hkv : target);
}

// Rows of a tile; parts (a row's partial results over the key ranges of its prefix) that scratch has room for: an item is a tile's key
// range and key head, there are at most `target` of them or one per tile and key head.
int tile_rows(int rep) { return kTile / rep; }
long long max_parts(int T, int rep, int Hkv, int target) {
  const long long r = T < tile_rows(rep) ? T : tile_rows(rep), s = (target + Hkv - 1) / Hkv;
  return r * s > T ? r * s : T;
}

__device__ __forceinline__ int block_sum_int(int v, int* sm /*[33]*/) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  int s = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += sm[w];
  return s;
}

__device__ __forceinline__ int block_max_int(int v, int* sm /*[33]*/) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  int m = sm[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) m = max(m, sm[w]);
  return m;
}

// One CTA, a thread per row.  Rows of a group keep their order; groups are ordered by their first row.
__global__ void __launch_bounds__(kPlanMaxRows) prefix_plan_kernel(const int32_t* __restrict__ row_slot, const int32_t* __restrict__ row_pos, int T,
                                                                   const int32_t* __restrict__ prefix_id, const int32_t* __restrict__ prefix_len,
                                                                   int n_slots, int rt, int Hkv, int target, int cap_items, int cap_parts, long long least, int32_t* plan, int max_rows) {
  __shared__ int s_id[kPlanMaxRows];     // prefix of the row, -1: none
  __shared__ int s_len[kPlanMaxRows];    // its tokens
  __shared__ int s_lead[kPlanMaxRows];   // first row of its group, if the group is taken together
  __shared__ int s_tile[kPlanMaxRows / kPlanMinRows + 1][8];  // blocks, rows, key ranges, first item, slot, keys, first entry of the list
  __shared__ int s_red[33];
  pdl_launch_dependents();
  pdl_wait();
  const PlanView v = plan_view(plan, max_rows);
  const int t = threadIdx.x;
  int id = -1, len = 0, slot = 0;
  if (t < T) {
    slot = row_slot[t];
    if (slot >= 0 && slot < n_slots && (row_pos == nullptr || row_pos[t] >= 0)) id = prefix_id[slot], len = prefix_len[slot];
  }
  if (len < kPlanMinKeys) id = -1;
  s_id[t] = id;
  s_len[t] = len;
  __syncthreads();
  int rank = 0, count = 0, lead = t;
  if (id >= 0)
    for (int j = 0; j < T; ++j)
      if (s_id[j] == id) {
        if (j < lead) lead = j;
        len = min(len, s_len[j]);  // (of slots that say different things, what all of them share)
        rank += j < t;
        ++count;
      }
  const bool used = id >= 0 && taken_together(count, len, Hkv, least);
  s_lead[t] = used ? lead : -1;
  __syncthreads();
  const bool opens = used && rank % rt == 0;  // first row of a tile
  const int n_tiles = block_sum_int(opens, s_red);
  int place = 0, tile = 0;
  if (used) {
    for (int j = 0; j < T; ++j) place += s_lead[j] >= 0 && s_lead[j] < lead;
  }
  // tiles before this row's group: a group of n rows has ceil(n / rt); the group's first row knows n
  __shared__ int s_group_tiles[kPlanMaxRows];
  s_group_tiles[t] = used && rank == 0 ? (count + rt - 1) / rt : 0;
  __syncthreads();
  if (used) {
    for (int j = 0; j < lead; ++j) tile += s_group_tiles[j];
    tile += rank / rt;
    place += rank;
    v.list[place] = t;
  }
  int blocks = 0, rows = 0;
  if (opens) {
    rows = min(rt, count - rank);
    blocks = (len - 1) / kTile + 1;  // (any 32-bit length)
    s_tile[tile][0] = blocks;
    s_tile[tile][1] = rows;
  }
  const int total = block_sum_int(blocks, s_red);
  // Blocks per item: a candidate per thread, from a quarter of an equal share for `target` items -- two per SM -- upwards, and one item per
  // tile and key head, which always has room.  The best one has the shortest way through: rounds of `target` items times the longest item,
  // each with some two blocks' time before and behind, and then the join of a row's ranges.  (An equal
  // share alone gives 4 tiles x 256 blocks x 8 key heads 320 items of 26 blocks, a round and a bit; 288 of 29 are one.)
  __shared__ unsigned long long s_best;
  const int longest = block_max_int(blocks, s_red);
  if (t == 0) s_best = ~0ull;
  const int base = max(1, (int)(((long long)total * Hkv + 4LL * target - 1) / (4LL * target)));
  const auto candidate = [&](int i) { return i == 0 ? longest : base + (i - 1) * max(1, base / 16); };
  __syncthreads();
  {
    const int unit = candidate(t);
    long long items = 0, parts = 0;
    int length = 0, most = 0;
    for (int i = 0; i < n_tiles && unit <= longest; ++i) {
      const int n = s_tile[i][0], k = (n + unit - 1) / unit;
      items += k;
      parts += k * s_tile[i][1];
      length = max(length, (n + k - 1) / k);
      most = max(most, k);
    }
    items *= Hkv;
    if (n_tiles > 0 && unit <= longest && items <= cap_items && parts <= cap_parts) {
      const unsigned long long cost = (unsigned long long)((items + target - 1) / target) * (length + 2) * kBlockParts + most;
      atomicMin(&s_best, min(cost, (1ull << 29) - 1) << 34 | (unsigned long long)items << 10 | t);
    }
  }
  __syncthreads();
  const int unit = max(1, candidate((int)(s_best & 1023)));
  const int splits = opens ? (blocks + unit - 1) / unit : 0;
  if (opens) s_tile[tile][2] = splits;
  __syncthreads();
  int part_of_row = 0, n_part = 0;
  if (used) {
    int item = 0, part = 0;
    for (int i = 0; i < tile; ++i) {
      item += s_tile[i][2] * Hkv;
      part += s_tile[i][1] * s_tile[i][2];
    }
    n_part = s_tile[tile][2];
    part_of_row = part + (rank % rt) * n_part;
    if (opens) s_tile[tile][3] = item, s_tile[tile][4] = slot, s_tile[tile][5] = len, s_tile[tile][6] = place;
  }
  if (t < T) v.row[t] = make_int4(used ? len : 0, part_of_row, n_part, 0);
  const int items = block_sum_int(splits, s_red) * Hkv, parts = block_sum_int(splits * rows, s_red);
  if (t == 0) {
    v.head[0] = T;
    v.head[1] = n_tiles;
    v.head[2] = items;
    v.head[3] = parts;
  }
  for (int i = t; i < items; i += blockDim.x) {
    int lo = 0, hi = n_tiles - 1;  // the last tile whose first item is not behind this one
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (s_tile[mid][3] <= i) lo = mid; else hi = mid - 1;
    }
    const int* e = s_tile[lo];
    const int r = i - e[3], split = r % e[2], b0 = (int)((long long)e[0] * split / e[2]), b1 = (int)((long long)e[0] * (split + 1) / e[2]);
    v.item[2 * i] = make_int4(e[4], b0, b1 - b0, e[5]);
    v.item[2 * i + 1] = make_int4(e[6], e[1], r / e[2], split);
  }
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two weights as the sum of two pairs of bf16: what a truncation leaves is rounded, so that the products with the values see them to 2^-15
// and the sum l, which is taken before, fits them.  Decode attention without shared prefixes has fp32 weights; with bf16
// ones a row's error was 0.0019 of the result in place of 0.0017, which is the result's own rounding; twice the products and as many stores
// to TMEM cost 3 % at 32 x 4096, 5 % at four groups of 40 heads and, with the reference that lags behind, 4 to 10 % at 128 x 32768.  Truncating
// is a byte permutation; rounding the first part as well costs 6 % more there.
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
  const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  hi = __byte_perm(a, b, 0x7632);
  const __nv_bfloat162 r = __floats2bfloat162_rn(x - __uint_as_float(a & 0xffff0000u), y - __uint_as_float(b & 0xffff0000u));
  lo = *reinterpret_cast<const uint32_t*>(&r);
}

struct SharedArgs {
  const bf16* q;
  int64_t ld;
  const bf16* k_pages;
  const bf16* v_pages;
  const int32_t* block_table;
  int max_pages, n_pages;
  const int32_t* row_slot;
  const int32_t* row_pos;
  int T, Hq, Hkv, page_size;
  int32_t* plan;
  int plan_rows;
  float* parts;     // [part][Hq][D + 4]: O, m, l of a row's key range (base-2 logarithms)
  float* own;       // [T][Hq][n_splits][D + 4]
  int32_t* tickets; // [T][Hkv][head tiles], zero between calls
  int n_splits;
  bf16* out;
  int64_t ld_out;
  float scale;      // of the scores, times log2(e)
  int32_t* status;
};

// The matrix products multiply every value of a block with every pair's weight: a value that is infinite or none makes the sums NaN for pairs
// that do not see its key (weight 0) or whose weight has no second part.  A sum that has met one stays infinite or NaN, so that is looked at
// once, at the end, and the few pairs whose sums are not finite are weighed again by this function, a warp for a pair, key by key in fp32:
// keys that the pair does not see or scores -inf are left out, whatever their values are.  (Looking at the sums costs 1 %; one infinite value in
// 32768 tokens that 512 pairs share costs some 55 ms, in 4096 tokens of 32 pairs 8.)
// dst[c] = sum of exp2(scale q k - m) v[c] over the keys of [lo, hi) in the units of 16 from k0 on, every `step` keys.
template <int D>
__device__ __noinline__ void weigh_again(const bf16* q, const bf16* k_pages, const bf16* v_pages, int n_pages, const int32_t* bt, int Hkv, int kvh, int PS,
                                         int k0, int step, int lo, int hi, float scale, float m, float* dst) {
  constexpr int kCols = D / 32;
  const int lane = threadIdx.x & 31;
  float qf[kCols], o[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) qf[c] = __bfloat162float(q[lane * kCols + c]), o[c] = 0.f;
  for (int u = k0; u < hi; u += step) {
    const int page = bt[u / PS];
    const bool there = page >= 0 && page < n_pages;  // (else the copies have read zeros)
    const size_t at = (((size_t)(there ? page : 0) * Hkv + kvh) * PS + u % PS) * D + lane * kCols;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      if (u + i < lo || u + i >= hi) continue;
      float d = 0.f;
      if (there)
#pragma unroll
        for (int c = 0; c < kCols; ++c) d = fmaf(qf[c], __bfloat162float(k_pages[at + i * D + c]), d);
      d = warp_sum(d);
      if (d == -INFINITY) continue;
      const float w = fast_exp2(fmaf(d, scale, -m));
      if (there)
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[c] = fmaf(w, __bfloat162float(v_pages[at + i * D + c]), o[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < kCols; ++c) dst[lane * kCols + c] = o[c];
}

// One item: a tile's pairs x a range of the prefix's blocks of 128 keys x one key head.  As in the prompt attention, S = Q K^T and
// P V are tcgen05 products with S, P and O in TMEM, keys and values arrive page by page through the block table of the group's first
// row, and one thread per pair runs the softmax: 64 of a block's scores in registers at a time, and nothing else to be taken out of TMEM.
template <int ND, int PS>
__global__ void __maxnreg__(kPxRegs) prefix_attn_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                     const __grid_constant__ CUtensorMap map_v,
                                                                     const __grid_constant__ CUtensorMap map_kr,
                                                                     const __grid_constant__ CUtensorMap map_vr, SharedArgs a) {
  constexpr int D = ND * 64, kPages = kTile / PS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sq = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sk = sq + ND * kSub;
  uint8_t* sv = sk + ND * kSub;
  __shared__ uint64_t kbar, vbar;  // a block's keys / values have landed
  __shared__ uint64_t sbar;        // S = Q K^T has retired, and every P V before it
  __shared__ uint64_t pbar[2];     // the four softmax warps have written P of the block's first / last 64 keys; O is at its reference
  __shared__ uint64_t obar;        // P V has retired
  __shared__ uint64_t fbar;        // ... the last one
  __shared__ uint32_t tmem_slot;
  __shared__ int s_abort;

  pdl_wait();
  pdl_launch_dependents();  // (behind the wait: the tail may begin when everything before this kernel is done; its own keys do not depend on it)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PlanView pv = plan_view(a.plan, a.plan_rows);
  const int n_items = pv.head[2];
  const int4 i0 = pv.item[2 * blockIdx.x], i1 = pv.item[2 * blockIdx.x + 1];  // (there is room for as many as there are CTAs)
  if ((int)blockIdx.x >= n_items) return;  // (the whole CTA, before it has asked for anything)
  const int rep = a.Hq / a.Hkv, kvh = i1.z, split = i1.w;
  const int n_keys = min(i0.w, a.max_pages * PS), n_pages = (n_keys + PS - 1) / PS;
  const int b0 = i0.y, n_blocks = max(0, min(i0.y + i0.z, (n_keys + kTile - 1) / kTile) - i0.y);  // (a prefix longer than the block table is cut)
  const int32_t* bt = a.block_table + (size_t)i0.x * a.max_pages;
  if (tid == 0) {
    s_abort = 0;
    mbar_init(&kbar, 1);
    mbar_init(&vbar, 1);
    mbar_init(&sbar, 1);
    mbar_init(&pbar[0], 4);
    mbar_init(&pbar[1], 4);
    mbar_init(&obar, 1);
    mbar_init(&fbar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) {
    if (lane == 0) {
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
      tma_prefetch_desc(&map_kr);
      tma_prefetch_desc(&map_vr);
    }
    __syncwarp();
    tmem_alloc(&tmem_slot, 256);
  }

  // (the pairs' queries, as the tensor cores read them: rows of 128 bytes, 16-byte chunks XORed with the row)
  int row = -1, head = 0;
  if (tid < kTile) {
    if (tid < i1.y * rep) {
      row = pv.list[i1.x + tid / rep];
      head = kvh * rep + tid % rep;
    }
    const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)max(row, 0) * a.ld + (size_t)head * D);
#pragma unroll
    for (int c = 0; c < ND * 8; ++c)
      *reinterpret_cast<uint4*>(sq + (c >> 3) * kSub + tid * 128 + (((c & 7) ^ (tid & 7)) << 4)) = row >= 0 ? src[c] : make_uint4(0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot, tmem_o = tmem_base + kTile;

  if (warp >= 4) {
    auto wait = [&](uint64_t* bar, uint32_t par) {
      int w = 1;
      if (lane == 0) w = mbar_wait(bar, par, &s_abort) ? 1 : 0;
      w = __shfl_sync(0xffffffffu, w, 0);
      if (!w) s_abort = 1;
      return w != 0;
    };
    // Copies of a block's pages take some hundred cycles each to be issued: two warps share them, and the MMAs have time for half of them
    // while the softmax runs.
    auto page_of = [&](int kb) {  // read one block ahead
      const int pg = (b0 + kb) * kPages + lane;
      return lane < kPages && kb < n_blocks && pg < n_pages ? bt[pg] : -1;
    };
    auto copy = [&](int kb, int page, uint8_t* dst, const CUtensorMap* map, const CUtensorMap* map_run, uint64_t* bar) {
      const int valid = min(kPages, n_pages - (b0 + kb) * kPages);
      int pg[kPages];
#pragma unroll
      for (int i = 0; i < kPages; ++i) pg[i] = __shfl_sync(0xffffffffu, page, i);
      if (valid == kPages && __all_sync(0xffffffffu, lane >= kPages || page == pg[0] + lane)) {
        // pages that follow each other in the pool: one copy
        if (lane == 0) {
          mbar_expect_tx(bar, (uint32_t)(ND * kSub));
          tma_load_5d(dst, map_run, 0, 0, 0, kvh * (PS / 8), pg[0], bar);
        }
      } else if (lane == 0) {
        mbar_expect_tx(bar, (uint32_t)(valid * ND * PS * 128));
#pragma unroll
        for (int i = 0; i < kPages; ++i)
          if (i < valid) tma_load_5d(dst + i * (PS * D * 2), map, 0, 0, 0, kvh * (PS / 8), pg[i], bar);
      }
      __syncwarp();
    };
    int page = page_of(0), page_next = page_of(1);
    if (warp == 4) {
      // ---- MMAs, and copies of keys: the next block's once the scores are there -----------------------
      constexpr uint32_t idesc = make_idesc(kTile, kTile);
      constexpr uint32_t idesc_pv = make_idesc(kTile, D) | (1u << 16);  // B operand MN-major
      // (keys and values: atoms of 8 keys x 64 columns, those of the same keys beside each other)
      const uint64_t qdesc = make_smem_desc(smem_u32(sq)), kdesc = make_smem_desc(smem_u32(sk)) + ((uint64_t)((ND - 1) * 1024 >> 4) << 32);
      const uint64_t vdesc = make_smem_desc_mn(smem_u32(sv), 1024, ND * 1024);
      if (n_blocks > 0) copy(0, page, sk, &map_k, &map_kr, &kbar);
      for (int kb = 0; kb < n_blocks; ++kb) {
        const uint32_t par = kb & 1;
        if (!wait(&kbar, par)) break;
        if (lane == 0) {
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_bf16(tmem_base, qdesc + j * (kSub >> 4) + 2 * k, kdesc + j * (1024 >> 4) + 2 * k, idesc, (j > 0 || k > 0) ? 1u : 0u);
          umma_commit(&sbar);
        }
        __syncwarp();
        if (kb + 1 < n_blocks) {
          if (!wait(&sbar, par)) break;
          page = page_next;
          page_next = page_of(kb + 2);
          copy(kb + 1, page, sk, &map_k, &map_kr, &kbar);
        }
        if (!wait(&vbar, par)) break;
        bool ok = true;
        for (int half = 0; half < 2 && ok; ++half) {  // (the products of the first half run while the softmax is at the second)
          ok = wait(&pbar[half], par);
          if (ok && lane == 0) {
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 8; ++k)  // (both parts of 16 keys' weights, then the next 16)
              umma_bf16_ta(tmem_o, tmem_base + half * 64 + (k & 1) * 32 + (k >> 1) * 8, vdesc + (half * 4 + (k >> 1)) * (2 * ND * 1024 >> 4), idesc_pv,
                           kb + half + k > 0 ? 1u : 0u);
            if (half) umma_commit(&obar);
            if (half && kb + 1 == n_blocks) umma_commit(&fbar);
          }
        }
        if (!ok) break;
        __syncwarp();
      }
    } else {
      // ---- copies of values: a block's once the ones before are in O -------------------------------------------------------
      for (int kb = 0; kb < n_blocks; ++kb) {
        if (kb > 0 && !wait(&obar, (kb - 1) & 1)) break;
        copy(kb, page, sv, &map_v, &map_vr, &vbar);
        page = page_next;
        page_next = page_of(kb + 2);
      }
    }
    if (s_abort && lane == 0)  // copies may still be in flight: let them land before the shared memory goes to another CTA
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
  } else {
    // ---- softmax: one thread per pair; a warp without pairs only keeps step -------------------------------------------------
    const bool busy = warp * 32 < i1.y * rep;
    const int q_pos = row >= 0 ? a.row_pos[row] : -1;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int kb = 0; kb < n_blocks && ok; ++kb) {
      const uint32_t par = kb & 1;
      const int kstart = (b0 + kb) * kTile;
      ok = __all_sync(0xffffffffu, mbar_wait(&sbar, par, &s_abort));
      if (!ok) break;
      tc_fence_after();
      const uint32_t s_addr = tmem_base + lanes;
      if (n_keys - kstart < kTile) {
        // the prefix ends inside this block: values of keys that are not its own are zeroed (0 * NaN is not 0)
        ok = __all_sync(0xffffffffu, mbar_wait(&vbar, par, &s_abort));
        if (!ok) break;
        if (tid >= n_keys - kstart) {
#pragma unroll
          for (int half = 0; half < ND; ++half)
#pragma unroll
            for (int c = 0; c < 8; ++c) reinterpret_cast<uint4*>(sv + (tid >> 3) * (ND * 1024) + half * 1024 + (tid & 7) * 128)[c] = make_uint4(0u, 0u, 0u, 0u);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      const int hi = min(q_pos, n_keys - 1) - kstart;  // last key of the block that this pair sees
      if (busy) {
        float v[64];
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        const auto scores = [&](int half) {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld16_issue(s_addr + half * 64 + c * 16, v + c * 16);
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_wait_ld16(v + c * 16);
          if (__any_sync(0xffffffffu, hi < kTile - 1)) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (half * 64 + i > hi) v[i] = -INFINITY;
          }
        };
#pragma unroll
        for (int half = 1; half >= 0; --half) {
          scores(half);
#pragma unroll
          for (int i = 0; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], v[i]);
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale;
        const bool grows = top > m_run + kGrow;  // (with nothing seen yet: as soon as there is a score)
        if (__any_sync(0xffffffffu, grows)) {
          const float corr = !grows ? 1.f : m_run == -INFINITY ? 0.f : fast_exp2(m_run - top);
          if (grows) m_run = top;
          l_run *= corr;
          if (kb > 0)
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              float o[16];
              tmem_ld16_issue(tmem_o + lanes + c * 16, o);
              tmem_wait_ld16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= corr;
              tmem_st8_issue(tmem_o + lanes + c * 16, reinterpret_cast<const uint32_t*>(o));
              tmem_st8_issue(tmem_o + lanes + c * 16 + 8, reinterpret_cast<const uint32_t*>(o + 8));
            }
        }
        const float neg_m = m_run == -INFINITY ? 0.f : -m_run;  // (-inf: nothing seen yet)
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (half) scores(half);  // (the first half is still there; its weights go over scores that have been read)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float p0 = fast_exp2(fmaf(v[c * 16 + i], a.scale, neg_m)), p1 = fast_exp2(fmaf(v[c * 16 + i + 1], a.scale, neg_m));
              sum[i & 2] += p0;
              sum[(i & 2) + 1] += p1;
              split_pair(p0, p1, hi[i / 2], lo[i / 2]);
            }
            tmem_st8_issue(s_addr + half * 64 + c * 8, hi);
            tmem_st8_issue(s_addr + half * 64 + 32 + c * 8, lo);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pbar[half]);
        }
        l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      }
      if (!busy) {
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&pbar[0]);
          mbar_arrive(&pbar[1]);
        }
      }
    }
    if (ok && n_blocks > 0) ok = __all_sync(0xffffffffu, mbar_wait(&fbar, 0, &s_abort));
    tc_fence_after();
    if (!ok) s_abort = 1;
    if (busy) {
      float* dst = row < 0 ? nullptr : a.parts + ((size_t)(pv.row[row].y + split) * a.Hq + head) * (D + 4);
      const bool seen = ok && n_blocks > 0 && m_run > -INFINITY;  // (the sums of a pair that has seen nothing are 0, whatever the values are)
      float odd = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        float o[16] = {};
        if (ok && n_blocks > 0) {
          tmem_ld16_issue(tmem_o + lanes + c * 16, o);
          tmem_wait_ld16(o);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (!seen) o[i] = 0.f;
          odd = fmaf(o[i], 0.f, odd);
        }
        if (dst)
#pragma unroll
          for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(dst)[c * 4 + i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      }
      if (dst) *reinterpret_cast<float2*>(dst + D) = ok ? make_float2(m_run, l_run) : make_float2(-INFINITY, 0.f);
      for (uint32_t left = __ballot_sync(0xffffffffu, dst && odd != 0.f); left; left &= left - 1) {  // (NaN, where a sum is not finite)
        const int from = __ffs(left) - 1, r = __shfl_sync(0xffffffffu, row, from), h = __shfl_sync(0xffffffffu, head, from);
        const int end = min(__shfl_sync(0xffffffffu, q_pos, from) + 1, min(n_keys, (b0 + n_blocks) * kTile));
        const float m = __shfl_sync(0xffffffffu, m_run, from);
        __syncwarp();
        weigh_again<D>(a.q + (size_t)r * a.ld + (size_t)h * D, a.k_pages, a.v_pages, a.n_pages, bt, a.Hkv, kvh, PS, b0 * kTile, 16, 0, end, a.scale, m,
                       a.parts + ((size_t)(pv.row[r].y + split) * a.Hq + h) * (D + 4));
      }
    }
    if (!ok && tid == 0 && a.status) atomicOr(a.status, 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) tmem_dealloc(tmem_base, 256);
}

// ---- the tail -------------------------------------------------------------------------------------------------------------------
constexpr int kTlKeys = 16;  // keys a warp works on at a time
constexpr int kTlHeads = 8;  // query heads of a CTA
constexpr int kJoin = 8;     // ranges whose results a thread has on their way when it joins them

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {  // of 16-bit values, a pair per lane
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// grid (Hkv x head tiles, T, key ranges): up to eight query heads of a key head over the row's keys from `first` on (or a range of them).
template <int D, int STAGES, int W>
__global__ void __launch_bounds__(W * 32, 12 / W) tail_attn_kernel(const __grid_constant__ CUtensorMap map_k,
                                                               const __grid_constant__ CUtensorMap map_v, SharedArgs a) {
  constexpr int kTlWarps = W, kTlThreads = W * 32;
  constexpr int kHalf = kTlKeys * D * 2;               // bytes of 16 keys: D / 64 sub-tiles [16][64], 128-byte swizzle
  extern __shared__ uint8_t smem_raw[];                // [warp][stage][K | V]; then the warps' partial results
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[kTlWarps][STAGES];
  __shared__ float s_m[kTlWarps][kTlHeads], s_l[kTlWarps][kTlHeads];
  __shared__ float s_w[64][kTlHeads];                // factors of the ranges that are joined
  __shared__ int s_last, s_abort;

  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rep = a.Hq / a.Hkv, head_tiles = (rep + kTlHeads - 1) / kTlHeads;
  const int kvh = blockIdx.x / head_tiles, h0 = kvh * rep + (blockIdx.x % head_tiles) * kTlHeads, n_heads = min(kTlHeads, kvh * rep + rep - h0);
  const int t = blockIdx.y, split = blockIdx.z;
  const int slot = a.row_slot[t], pos = a.row_pos[t];
  const int4 plan = plan_view(a.plan, a.plan_rows).row[t];
  const int first = plan.x, n_part = plan.z;
  const int32_t* bt = a.block_table + (size_t)slot * a.max_pages;
  const int PS = a.page_size;
  const int n_tok = (int)min((long long)max(pos + 1, 0), (long long)a.max_pages * PS);
  // units of 16 keys; a range has at least 8 units a warp, else fewer CTAs work on the row
  const int u0 = min(first, n_tok) / kTlKeys, units = n_tok > first ? (n_tok + kTlKeys - 1) / kTlKeys - u0 : 0;
  const int ranges = max(1, min(a.n_splits, units / (8 * kTlWarps)));
  if (split >= ranges) return;
  const int ub = u0 + (int)((long long)units * split / ranges), ue = u0 + (int)((long long)units * (split + 1) / ranges);
  if (tid == 0) s_abort = 0;
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[warp][i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  uint8_t* mine = ring + warp * STAGES * 2 * kHalf;
  int page = 0;  // of the lane's unit among the 32 that come next: one read for them all, not one per unit in front of its copies
  auto fetch = [&](int i) {  // unit ub + warp + W i -> stage i % STAGES
    if ((i & 31) == 0) {
      const int u = ub + warp + (i + lane) * kTlWarps;
      page = u < ue ? bt[u * kTlKeys / PS] : 0;
    }
    const int u = ub + warp + i * kTlWarps, p = __shfl_sync(0xffffffffu, page, i & 31);
    if (u < ue && lane == 0) {
      uint64_t* bar = &full[warp][i % STAGES];
      uint8_t* dst = mine + (i % STAGES) * 2 * kHalf;
      mbar_expect_tx(bar, 2 * kHalf);
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        tma_load_4d(dst + j * 2048, &map_k, j * 64, u * kTlKeys % PS, kvh, p, bar);
        tma_load_4d(dst + kHalf + j * 2048, &map_v, j * 64, u * kTlKeys % PS, kvh, p, bar);
      }
    }
    __syncwarp();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(i);

  // queries as the B operand: column = head lane / 4, a register pair of columns 16 s + 2 (lane % 4) and + 8
  uint32_t qb[D / 16][2];
  {
    const int g = lane >> 2;
    const bf16* q = a.q + (size_t)t * a.ld + (size_t)(h0 + g) * D + (lane & 3) * 2;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      qb[s][0] = g < n_heads ? *reinterpret_cast<const uint32_t*>(q + s * 16) : 0u;
      qb[s][1] = g < n_heads ? *reinterpret_cast<const uint32_t*>(q + s * 16 + 8) : 0u;
    }
  }
  float o[D / 16][4];  // [column 16 i + lane / 4, + 8][head 2 (lane % 4), + 1]
#pragma unroll
  for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // of the lane's two heads (l: the lane's own keys)
  const int mr = lane & 7, mi = lane >> 3;  // row and matrix whose address this lane gives to ldmatrix

  bool ok = true;
  for (int i = 0; ub + warp + i * kTlWarps < ue; ++i) {
    fetch(i + STAGES - 1);
    ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][i % STAGES], (i / STAGES) & 1, &s_abort));
    if (!ok) break;
    const int key = (ub + warp + i * kTlWarps) * kTlKeys;
    uint8_t* stage = mine + (i % STAGES) * 2 * kHalf;
    const uint32_t sk = smem_u32(stage), sv = sk + kHalf;
    if (key < first || key + kTlKeys > n_tok) {  // what is not the row's own: its probabilities are 0, but 0 * NaN is not
      for (int c = lane; c < kTlKeys * D / 8; c += 32) {
        const int r = c % 128 / 8;  // (a sub-tile has 16 rows of eight pieces; a swizzled row stays inside its own 128 bytes)
        if (key + r < first || key + r >= n_tok) *reinterpret_cast<uint4*>(stage + kHalf + c * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    }
    float s[4] = {};  // [key lane / 4, + 8][head 2 (lane % 4), + 1]
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {  // matrices: keys 0-7 and 8-15 of columns 16 k, then of 16 k + 8
      uint32_t x[4];
      const int r = (mi & 1) * 8 + mr, ch = 2 * k + (mi >> 1);
      ldsm4(sk + (ch >> 3) * 2048 + r * 128 + (((ch & 7) ^ mr) << 4), x);
      mma16816(s, x, qb[k][0], qb[k][1]);
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int kk = key + (lane >> 2) + (e >> 1) * 8;
      s[e] = kk >= first && kk < n_tok ? s[e] * a.scale : -INFINITY;
      mx[e & 1] = fmaxf(mx[e & 1], s[e]);
    }
    float corr[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], x));
      const float mn = fmaxf(m[h], mx[h]);
      corr[h] = m[h] == -INFINITY ? 0.f : fast_exp2(m[h] - mn);
      l[h] *= corr[h];
      m[h] = mn;
    }
    uint32_t ph[2], pl[2];  // the lane's keys lane / 4 and + 8, a pair of heads each; then, transposed, a pair of keys of one head
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float x = s[2 * r] == -INFINITY ? 0.f : fast_exp2(s[2 * r] - m[0]), y = s[2 * r + 1] == -INFINITY ? 0.f : fast_exp2(s[2 * r + 1] - m[1]);
      l[0] += x, l[1] += y;
      split_pair(x, y, ph[r], pl[r]);
      ph[r] = transpose8x8(ph[r]), pl[r] = transpose8x8(pl[r]);
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {  // V transposed: rows = columns 16 c + lane / 4, + 8; matrices: keys 0-7 of both, then keys 8-15
      uint32_t x[4];
      const int r = (mi >> 1) * 8 + mr, ch = 2 * c + (mi & 1);
      ldsm4t(sv + (ch >> 3) * 2048 + r * 128 + (((ch & 7) ^ mr) << 4), x);
      o[c][0] *= corr[0], o[c][1] *= corr[1], o[c][2] *= corr[0], o[c][3] *= corr[1];
      mma16816(o[c], x, ph[0], ph[1]);
      mma16816(o[c], x, pl[0], pl[1]);
    }
    __syncwarp();  // (the next copy overwrites what was read here)
  }
  if (!ok) {
    s_abort = 1;
    for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies may still be in flight
  }
  __syncthreads();  // every warp is done with the ring
  if (s_abort && tid == 0 && a.status) atomicOr(a.status, 1);

  // ---- the warps' results, joined with what the prefix's key ranges left ---------------------------------------------------
  float* acc = reinterpret_cast<float*>(ring);  // [warp][head][D]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], x);
    const int hh = (lane & 3) * 2 + h;
    if (lane < 4) s_m[warp][hh] = m[h], s_l[warp][hh] = l[h];
    float odd = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      acc[(warp * kTlHeads + hh) * D + c * 16 + (lane >> 2)] = o[c][h];
      acc[(warp * kTlHeads + hh) * D + c * 16 + (lane >> 2) + 8] = o[c][2 + h];
      odd = fmaf(o[c][h], 0.f, fmaf(o[c][2 + h], 0.f, odd));
    }
    const uint32_t lanes = __ballot_sync(0xffffffffu, odd != 0.f);  // (NaN, where a sum is not finite)
    for (int x = 0; lanes && ok && x < 4 && 2 * x + h < n_heads; ++x) {
      if (!(lanes & (0x11111111u << x))) continue;
      const int hx = 2 * x + h;
      const float mx = __shfl_sync(0xffffffffu, m[h], x);
      __syncwarp();
      weigh_again<D>(a.q + (size_t)t * a.ld + (size_t)(h0 + hx) * D, a.k_pages, a.v_pages, a.n_pages, bt, a.Hkv, kvh, PS, (ub + warp) * kTlKeys,
                     kTlWarps * kTlKeys, first, mx > -INFINITY ? min(ue * kTlKeys, n_tok) : 0, a.scale, mx, acc + (warp * kTlHeads + hx) * D);
    }
  }
  __syncthreads();
  bool join = true;
  int32_t* ticket = a.tickets + ((size_t)t * a.Hkv + kvh) * head_tiles + blockIdx.x % head_tiles;
  if (ranges > 1) {  // this range's result into scratch; the last one of the row and key head joins them all
    for (int i = tid; i < n_heads * (D / 4); i += kTlThreads) {
      const int h = i / (D / 4), c = i % (D / 4);
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < kTlWarps; ++w) M = fmaxf(M, s_m[w][h]);
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kTlWarps; ++w) {
        const float f = s_m[w][h] == -INFINITY ? 0.f : fast_exp2(s_m[w][h] - M);
        const float4 x = reinterpret_cast<const float4*>(acc + (w * kTlHeads + h) * D)[c];
        L = fmaf(s_l[w][h], f, L);
        O.x = fmaf(x.x, f, O.x), O.y = fmaf(x.y, f, O.y), O.z = fmaf(x.z, f, O.z), O.w = fmaf(x.w, f, O.w);
      }
      float* dst = a.own + (((size_t)t * a.Hq + h0 + h) * a.n_splits + split) * (D + 4);
      reinterpret_cast<float4*>(dst)[c] = O;
      if (c == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(M, L);
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      const int before = atomicAdd(ticket, 1);
      s_last = before == ranges - 1;
      if (s_last) *ticket = 0;
    }
    __syncthreads();
    join = s_last;
    __threadfence();
  }
  if (!join) return;
  pdl_wait();  // the prefix's results (and, for whoever follows, that every kernel before this one is done)
  const int n_own = ranges > 1 ? ranges : kTlWarps;
  const auto own_ml = [&](int r, int h) {
    if (ranges == 1) return make_float2(s_m[r][h], s_l[r][h]);
    return __ldcg(reinterpret_cast<const float2*>(a.own + (((size_t)t * a.Hq + h0 + h) * a.n_splits + r) * (D + 4) + D));
  };
  const float* part0 = a.parts + ((size_t)plan.y * a.Hq + h0) * (D + 4);
  const size_t part_step = (size_t)a.Hq * (D + 4);
  // factors exp2(m - M) / L of every range, 64 prefix ranges at a time in shared memory; the totals first
  constexpr int kSubs = kTlThreads / kTlHeads;  // threads per head
  const int h = tid / kSubs, sub = tid % kSubs;
  float M = -INFINITY, L = 0.f;
  if (h < n_heads) {
    const auto take = [&](const float2& ml) {
      if (ml.x == -INFINITY) return;
      const float mn = fmaxf(M, ml.x);
      L = L * fast_exp2(M - mn) + ml.y * fast_exp2(ml.x - mn);
      M = mn;
    };
    for (int r = sub; r < n_own; r += kSubs) take(own_ml(r, h));
    const float* from = part0 + (size_t)h * (D + 4) + D;
    for (int r = sub; r < n_part; r += kSubs * kJoin) {
      float2 ml[kJoin];
#pragma unroll
      for (int j = 0; j < kJoin; ++j)
        ml[j] = r + j * kSubs < n_part ? __ldcg(reinterpret_cast<const float2*>(from + (size_t)(r + j * kSubs) * part_step)) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int j = 0; j < kJoin; ++j) take(ml[j]);
    }
  }
#pragma unroll
  for (int x = 1; x < kSubs; x <<= 1) {
    const float mo = __shfl_xor_sync(0xffffffffu, M, x), lo = __shfl_xor_sync(0xffffffffu, L, x), mn = fmaxf(M, mo);
    if (mn != -INFINITY) L = (M == -INFINITY ? 0.f : L * fast_exp2(M - mn)) + (mo == -INFINITY ? 0.f : lo * fast_exp2(mo - mn));
    M = mn;
  }
  const float inv = L > 0.f && !s_abort ? 1.f / L : 0.f;
  // outputs: 4 columns of a head per thread, D / 4 threads a head; where there are few heads, several threads share the ranges
  constexpr int kPer = kTlThreads / (D / 4);           // heads in work at once: 2, 4 or 8
  constexpr int kSets = kTlHeads / kPer;
  // (a part of them, a power of two, only where it has all heads: those are done in one set)
  const int hp = n_heads > kPer / 2 ? kPer : n_heads > 2 ? 4 : n_heads, slices = kPer / hp;
  float4 sum[kSets];
#pragma unroll
  for (int i = 0; i < kSets; ++i) sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  const int c = tid % (D / 4), hs = tid / (D / 4) % hp, slice = tid / (D / 4) / hp;
  for (int r0 = 0; r0 < n_own + n_part; r0 += 64) {
    const int n = min(64, n_own + n_part - r0);
    __syncthreads();
    if (h < n_heads)
      for (int r = sub; r < n; r += kSubs) {
        const int x = r0 + r;
        const float mx = x < n_own ? own_ml(x, h).x : __ldcg(part0 + (size_t)(x - n_own) * part_step + (size_t)h * (D + 4) + D);
        s_w[r][h] = mx == -INFINITY ? 0.f : fast_exp2(mx - M) * inv;
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      const int hh = i * hp + hs;
      if (hh >= n_heads || (i > 0 && hp < kPer)) continue;
      const auto add = [&](const float4& v, float f) {
        sum[i].x = fmaf(v.x, f, sum[i].x), sum[i].y = fmaf(v.y, f, sum[i].y), sum[i].z = fmaf(v.z, f, sum[i].z), sum[i].w = fmaf(v.w, f, sum[i].w);
      };
      int r = slice;
      for (; r < n && r0 + r < n_own; r += slices) {
        const int x = r0 + r;
        add(ranges == 1 ? reinterpret_cast<const float4*>(acc + (x * kTlHeads + hh) * D)[c]
                        : __ldcg(reinterpret_cast<const float4*>(a.own + (((size_t)t * a.Hq + h0 + hh) * a.n_splits + x) * (D + 4)) + c), s_w[r][hh]);
      }
      const float* from = part0 + (size_t)(r0 + r - n_own) * part_step + (size_t)hh * (D + 4) + 4 * c;
      for (; r < n; r += slices * kJoin, from += slices * kJoin * part_step) {
        float4 v[kJoin];
#pragma unroll
        for (int j = 0; j < kJoin; ++j)
          v[j] = r + j * slices < n ? __ldcg(reinterpret_cast<const float4*>(from + j * slices * part_step)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < kJoin; ++j) add(v[j], r + j * slices < n ? s_w[r + j * slices][hh] : 0.f);
      }
    }
  }
  if (slices > 1) {
    float4* share = reinterpret_cast<float4*>(ring) + kTlWarps * kTlHeads * D / 4;  // (behind the warps' results)
    if (slice > 0) share[tid] = sum[0];
    __syncthreads();
    if (slice > 0) return;
    for (int i = 1; i < slices; ++i) {
      const float4 v = share[tid + i * hp * (D / 4)];
      sum[0].x += v.x, sum[0].y += v.y, sum[0].z += v.z, sum[0].w += v.w;
    }
  }
#pragma unroll
  for (int i = 0; i < kSets; ++i) {
    const int hh = i * hp + hs;
    if (hh >= n_heads || (i > 0 && hp < kPer)) continue;
    __nv_bfloat162 b[2] = {__floats2bfloat162_rn(sum[i].x, sum[i].y), __floats2bfloat162_rn(sum[i].z, sum[i].w)};
    *reinterpret_cast<uint2*>(a.out + (size_t)t * a.ld_out + (size_t)(h0 + hh) * D + c * 4) = *reinterpret_cast<const uint2*>(b);
  }
}

// Pages [n_pages][Hkv][PS][D], a box of kTlKeys keys of one head, 64 columns: rows of 128 bytes, swizzled.
int page_map(CUtensorMap* m, const void* ptr, int n_pages, int Hkv, int PS, int D) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(MLORA_ECUDA, "paged_attention_shared: cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)PS, (cuuint64_t)Hkv, (cuuint64_t)n_pages};
  cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)PS * D * 2, (cuuint64_t)Hkv * PS * D * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)kTlKeys, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MLORA_ECUDA, "paged_attention_shared: cuTensorMapEncodeTiled failed with %d", (int)r);
  return MLORA_OK;
}

// The same, `pages` whole pages of one head as atoms of 8 keys x 64 columns, those of the same keys beside each other: one copy has it all.
int atom_map(CUtensorMap* m, const void* ptr, int n_pages, int Hkv, int PS, int D, int pages) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(MLORA_ECUDA, "paged_attention_shared: cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[5] = {64, 8, (cuuint64_t)D / 64, (cuuint64_t)Hkv * (PS / 8), (cuuint64_t)n_pages};
  cuuint64_t strides[4] = {(cuuint64_t)D * 2, 128, (cuuint64_t)8 * D * 2, (cuuint64_t)Hkv * PS * D * 2};
  cuuint32_t box[5] = {64, 8, (cuuint32_t)D / 64, (cuuint32_t)PS / 8, (cuuint32_t)pages};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MLORA_ECUDA, "paged_attention_shared: cuTensorMapEncodeTiled failed with %d", (int)r);
  return MLORA_OK;
}

template <typename K>
int allow_smem(K kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (!((done.load(std::memory_order_acquire) >> (dev & 63)) & 1ull)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return fail(MLORA_ECUDA, "paged_attention_shared: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done.fetch_or(1ull << (dev & 63), std::memory_order_release);
  }
  return MLORA_OK;
}

constexpr int kTlStages = 2;  // (twelve warps per SM, in three or six CTAs: 96 KB on the way, and another 96 at work)

template <int D, int W>
int launch_tail(const CUtensorMap& mk, const CUtensorMap& mv, const SharedArgs& a, bool behind_prefix, cudaStream_t st) {
  constexpr int smem = W * kTlStages * 2 * kTlKeys * D * 2 + 1024;
  static_assert(smem >= W * kTlHeads * D * 4 + W * 32 * 16 + 1024, "the warps' results lie in the ring");
  static std::atomic<unsigned long long> done{0};
  const int rc = allow_smem(tail_attn_kernel<D, kTlStages, W>, smem, done);
  if (rc) return rc;
  const int head_tiles = (a.Hq / a.Hkv + kTlHeads - 1) / kTlHeads;
  const cudaError_t e = launch_pdl_if(behind_prefix && pdl_enabled_tail(), tail_attn_kernel<D, kTlStages, W>,
                                      dim3((unsigned)(a.Hkv * head_tiles), (unsigned)a.T, (unsigned)a.n_splits), dim3(W * 32), smem, st, mk, mv, a);
  if (e != cudaSuccess) return fail(MLORA_ECUDA, "tail_attn_kernel: %s", cudaGetErrorString(e));
  count_launch();
  MLORA_CHECK_LAUNCH("tail_attn_kernel");
  return MLORA_OK;
}

template <int ND, int PS>
int launch_shared(const SharedArgs& a, int n_pages_total, int max_items, cudaStream_t st) {
  constexpr int D = ND * 64;
  CUtensorMap mk, mv, mkr, mvr, mkt, mvt;  // a page, a block of them, 16 keys
  int rc = atom_map(&mk, a.k_pages, n_pages_total, a.Hkv, PS, D, 1);
  if (!rc) rc = atom_map(&mv, a.v_pages, n_pages_total, a.Hkv, PS, D, 1);
  if (!rc) rc = atom_map(&mkr, a.k_pages, n_pages_total, a.Hkv, PS, D, kTile / PS);
  if (!rc) rc = atom_map(&mvr, a.v_pages, n_pages_total, a.Hkv, PS, D, kTile / PS);
  if (!rc) rc = page_map(&mkt, a.k_pages, n_pages_total, a.Hkv, PS, D);
  if (!rc) rc = page_map(&mvt, a.v_pages, n_pages_total, a.Hkv, PS, D);
  if (rc) return rc;
  constexpr int smem = 3 * ND * kSub + 1024;
  static std::atomic<unsigned long long> done{0};
  rc = allow_smem(prefix_attn_kernel<ND, PS>, smem, done);
  if (rc) return rc;
  if (max_items > 0) {
    const cudaError_t e = launch_pdl_if(pdl_enabled_tail(), prefix_attn_kernel<ND, PS>, dim3((unsigned)max_items), dim3(kPxThreads), smem, st, mk, mv, mkr, mvr, a);
    if (e != cudaSuccess) return fail(MLORA_ECUDA, "prefix_attn_kernel: %s", cudaGetErrorString(e));
    count_launch();
    MLORA_CHECK_LAUNCH("prefix_attn_kernel");
  }
  // Many (row, key head) pairs: CTAs of two warps, whose ends hold up less of an SM.  Against four warps, behind 1024 shared tokens: from 2048
  // pairs on 10 to 29 % less time with 48 tokens of the rows' own, 0 to 9 % with 400, and rows that share nothing take up to 9 % more (heads
  // of 128) or 19 % (64); at 1024 pairs 0 to 16 % less with 48 tokens, but 9 to 30 % more with 2000, and up to 18 or 44 % more without a prefix.
  return (long long)a.T * a.Hkv >= 2048 ? launch_tail<D, 2>(mkt, mvt, a, max_items > 0, st) : launch_tail<D, 4>(mkt, mvt, a, max_items > 0, st);
}

// How a call's scratch is laid out: tickets | own parts | prefix parts, in floats.
struct SharedSizes {
  int target, max_items, n_splits;
  long long tickets, own, parts, cap_parts;
};
SharedSizes sizes_of(int T, int Hq, int Hkv, int D) {
  SharedSizes s;
  const int rep = Hq / Hkv, ht = (rep + kTlHeads - 1) / kTlHeads;
  s.target = 2 * sm_count();
  s.max_items = max_items_of(T, Hkv, s.target);
  const long long ctas = (long long)T * Hkv * ht;
  s.n_splits = ctas >= s.target || ctas > kTickets ? 1 : (int)((s.target + ctas - 1) / (ctas > 0 ? ctas : 1));
  if (s.n_splits > 32) s.n_splits = 32;
  s.tickets = kTickets;
  s.own = s.n_splits > 1 ? (long long)T * Hq * s.n_splits * (D + 4) : 0;
  s.cap_parts = max_parts(T, rep, Hkv, s.target);
  s.parts = s.cap_parts * Hq * (D + 4);
  return s;
}

bool shared_sizes_fit(int T, int Hq, int Hkv, int D) {
  return T >= 0 && T <= kPlanMaxRows && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && kTile / (Hq / Hkv) > kPlanMinRows && Hq <= 1024 && (D == 64 || D == 128);
}

}  // namespace
}  // namespace mlora

using namespace mlora;

extern "C" size_t mlora_prefix_plan_bytes(int32_t max_rows, int32_t Hkv) {
  if (max_rows < 0 || max_rows > kPlanMaxRows || Hkv <= 0 || Hkv > 1024) return 0;
  return 4u * (size_t)(kPlanHeader + 4 * max_rows + (max_rows + 3) / 4 * 4 + 8 * max_items_of(max_rows, Hkv, 2 * sm_count()));
}

extern "C" int mlora_prefix_plan(const int32_t* d_row_slot, int32_t T, const int32_t* d_prefix_id, const int32_t* d_prefix_len, int32_t n_slots,
                                 int32_t Hq, int32_t Hkv, int64_t least, int32_t* d_plan, int32_t max_rows, void* stream) {
  return mlora_prefix_plan_rows(d_row_slot, nullptr, T, d_prefix_id, d_prefix_len, n_slots, Hq, Hkv, least, d_plan, max_rows, stream);
}

extern "C" int mlora_prefix_plan_rows(const int32_t* d_row_slot, const int32_t* d_row_pos, int32_t T, const int32_t* d_prefix_id,
                                      const int32_t* d_prefix_len, int32_t n_slots, int32_t Hq, int32_t Hkv, int64_t least, int32_t* d_plan,
                                      int32_t max_rows, void* stream) {
  MLORA_REQUIRE(shared_sizes_fit(T, Hq, Hkv, 64) && T <= max_rows && max_rows <= kPlanMaxRows && n_slots > 0,
                "prefix_plan: bad sizes T=%d of %d, %d heads over %d key heads", T, max_rows, Hq, Hkv);
  MLORA_REQUIRE(d_row_slot && d_prefix_id && d_prefix_len && d_plan && aligned16(d_plan), "prefix_plan: null pointer or unaligned plan");
  if (T == 0) return MLORA_OK;
  const int rep = Hq / Hkv, target = 2 * sm_count();
  const int threads = T <= 256 ? 256 : (T + 31) / 32 * 32;
  launch_pdl(prefix_plan_kernel, 1, threads, 0, (cudaStream_t)stream, d_row_slot, d_row_pos, T, d_prefix_id, d_prefix_len, n_slots, tile_rows(rep),
             Hkv, target, max_items_of(T, Hkv, target), (int)max_parts(T, rep, Hkv, target), (long long)least, d_plan, max_rows);
  count_launch();
  MLORA_CHECK_LAUNCH("prefix_plan_kernel");
  return MLORA_OK;
}

extern "C" int mlora_prefix_together(int32_t rows, int32_t tokens, int32_t Hkv, int64_t least) {
  MLORA_REQUIRE(rows >= 0 && tokens >= 0 && Hkv > 0, "prefix_together: bad sizes %d rows, %d tokens, %d key heads", rows, tokens, Hkv);
  return taken_together(rows, tokens, Hkv, least) ? 1 : 0;
}

extern "C" size_t mlora_paged_attention_shared_workspace(int32_t T, int32_t Hq, int32_t Hkv, int32_t D) {
  if (!shared_sizes_fit(T, Hq, Hkv, D)) return 0;
  const SharedSizes s = sizes_of(T, Hq, Hkv, D);
  return 4 * (size_t)(s.tickets + s.own + s.parts);
}

extern "C" int mlora_paged_attention_shared(const void* d_q, int64_t ld, const void* d_k_pages, const void* d_v_pages, int32_t n_pages_total,
                                            const int32_t* d_block_table, int32_t max_pages, const int32_t* d_row_slot,
                                            const int32_t* d_row_pos, int32_t T, int32_t Hq, int32_t Hkv, int32_t D, int32_t page_size,
                                            float scale, const int32_t* d_plan, int32_t plan_rows, void* d_out, int64_t ld_out, void* d_work,
                                            size_t work_bytes, int32_t* d_status, void* stream) {
  MLORA_REQUIRE((D == 64 || D == 128) && (page_size == 16 || page_size == 32),
                "paged_attention_shared: head_dim 64 or 128 and pages of 16 or 32 only (got %d, %d)", D, page_size);
  MLORA_REQUIRE(shared_sizes_fit(T, Hq, Hkv, D) && T <= plan_rows && plan_rows <= kPlanMaxRows && n_pages_total > 0 && max_pages > 0 &&
                    max_pages <= 2147483647 / page_size && scale > 0.f && ld >= (int64_t)Hq * D && ld_out >= (int64_t)Hq * D,
                "paged_attention_shared: bad sizes T=%d Hq=%d Hkv=%d", T, Hq, Hkv);
  MLORA_REQUIRE(d_q && d_k_pages && d_v_pages && d_block_table && d_row_slot && d_row_pos && d_plan && d_out, "paged_attention_shared: null pointer");
  MLORA_REQUIRE(aligned16(d_q) && aligned16(d_k_pages) && aligned16(d_v_pages) && aligned16(d_out) && aligned16(d_plan) && aligned16(d_work) &&
                    ld % 8 == 0 && ld_out % 8 == 0,
                "paged_attention_shared: 16-byte alignment of tensors and row pitches");
  if (T == 0) return MLORA_OK;
  const SharedSizes s = sizes_of(T, Hq, Hkv, D);
  if (!d_work || work_bytes < 4 * (size_t)(s.tickets + s.own + s.parts))
    return fail(MLORA_ESIZE, "paged_attention_shared: scratch of %zu bytes needed, %zu given", 4 * (size_t)(s.tickets + s.own + s.parts), work_bytes);
  float* w = (float*)d_work;
  SharedArgs a{(const bf16*)d_q, ld, (const bf16*)d_k_pages, (const bf16*)d_v_pages, d_block_table, max_pages, n_pages_total, d_row_slot, d_row_pos, T, Hq,
               Hkv, page_size, const_cast<int32_t*>(d_plan), plan_rows, w + s.tickets + s.own, w + s.tickets, (int32_t*)w, s.n_splits, (bf16*)d_out, ld_out,
               scale * kLog2e, d_status};
  cudaStream_t st = (cudaStream_t)stream;
  if (D == 64) return page_size == 16 ? launch_shared<1, 16>(a, n_pages_total, s.max_items, st) : launch_shared<1, 32>(a, n_pages_total, s.max_items, st);
  return page_size == 16 ? launch_shared<2, 16>(a, n_pages_total, s.max_items, st) : launch_shared<2, 32>(a, n_pages_total, s.max_items, st);
}
