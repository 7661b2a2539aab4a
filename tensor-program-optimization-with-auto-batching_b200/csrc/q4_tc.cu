// Projections with 4-bit weights on the 5th-generation tensor cores, for more than 16 rows (see q4.cuh for the layout).
//
// Tiles of 128 outputs x BN rows of x, in units of 128 inputs.  Eight warps take packed weights from rings of bulk copies, turn them into
// bf16 integers q - z and write them to TMEM (tcgen05.st.16x128b has the lanes where the packed order has them): weights go DRAM -> shared
// memory -> registers -> TMEM and are never written to shared memory as bf16, whose 32 KB per 8 KB of weights would be more than its
// bandwidth.  The MMA takes them from there as its A operand -- 16 cycles per m128n32k16, against 40 from shared memory -- and the rows of
// x (TMA, 128-byte swizzle) as B.  A group's sums have an accumulator of their own, which four or eight warps scale in fp32 registers
// while the next ones are filled: nothing but the output is rounded.
//
// Persistent, one CTA per SM; the units of all tiles are dealt out in equal ranges.  A tile that several CTAs share is summed by the last
// of them to arrive, in the order of the inputs, from the partial sums that each has left in scratch: no CTA waits for another.
#include "q4.cuh"
#include "tc_ptx.cuh"

#include <atomic>

namespace mlora {
namespace {

// Warps 0..7: weights; then four or eight (tiles of 128 rows of x: half of the columns each) for sums and outputs, MMA issue, copies of x.
constexpr int q4_threads(int bn) { return 32 * (8 + (bn == 128 ? 8 : 4) + 2); }
constexpr int kBufs = 4;                 // units of weights in TMEM, and of x in shared memory
constexpr int kWslots = 4;               // packed units in a weight warpgroup's ring
constexpr int kSlots = 8;                // units whose scales lie in shared memory
constexpr int kMaxCtas = 512;
constexpr int kHeader = 256;             // bytes: status word, then the caller's
constexpr int kScaleBytes = 4 * 512;     // scales of a unit's groups, at most
constexpr int kSlotBytes = 2 * kQ4TileBytes + kScaleBytes;  // a unit, and its groups' scales where there are zero points

struct TcArgs {
  Q4Args p;
  int32_t* status;
  int32_t* counters;  // [CTA that the tile begins in], zero between calls
  float* parts;       // [CTA][2][BN][128]: sums of the tile it ends and of the tile it begins
  int row_tiles, token_tiles, units;  // units of 128 inputs per tile
};

// One verdict of the N threads that sum; see bar_all.
template <int N>
__device__ __forceinline__ bool out_all(bool ok) {
  uint32_t r;
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.aligned.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok), "n"(N)
      : "memory");
  return r != 0;
}
// 16 lanes x 32 columns from registers laid out as A operands of mma.m16n8k16
__device__ __forceinline__ void tmem_st_16x128b_x8(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
               "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}

// The units of a CTA's range, one after the other.
struct Cursor {
  int left, u, row_tile, token_tile, units, row_tiles;
  __device__ Cursor(const TcArgs& t, long long a, long long b) : left((int)(b - a)), units(t.units), row_tiles(t.row_tiles) {
    const int tile = (int)(a / t.units);
    u = (int)(a % t.units);
    row_tile = tile % t.row_tiles;
    token_tile = tile / t.row_tiles;
  }
  __device__ void next() {
    --left;
    if (++u < units) return;
    u = 0;
    if (++row_tile == row_tiles) row_tile = 0, ++token_tile;
  }
};

template <int BN, bool ZERO, int G>
__global__ void __launch_bounds__(q4_threads(BN), 1) q4_tc_kernel(const __grid_constant__ CUtensorMap map_x, TcArgs t) {
  constexpr int kDbufs = BN == 128 ? 2 : 4;
  constexpr int kOutWarps = BN == 128 ? 8 : 4, kMma = 8 + kOutWarps;  // first of the two warps behind them
  constexpr int kCols = BN * 4 / kOutWarps;               // columns of a thread that sums
  constexpr int kSums = 128 / G;                          // groups of a unit
  constexpr int kEntry = ZERO ? 4 : 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sx = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sw = sx + kBufs * BN * 256;                    // [weight warpgroup][slot][kSlotBytes]
  uint8_t* ss = sw + 2 * kWslots * kSlotBytes;            // [slot][kScaleBytes]
  __shared__ uint64_t w_full[2 * kWslots], w_empty[2 * kWslots], x_full[kBufs], a_full[kBufs], empty[kBufs], d_full[kDbufs], d_empty[kDbufs],
      s_full[kSlots], s_empty[kSlots];
  __shared__ uint32_t tmem_slot;
  __shared__ int s_abort, s_last;

  pdl_launch_dependents();
  const LinearArgs& a = t.p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < 2 * kWslots; ++i) mbar_init(&w_full[i], 1), mbar_init(&w_empty[i], 4);
    for (int i = 0; i < kBufs; ++i) mbar_init(&x_full[i], 1), mbar_init(&a_full[i], 4), mbar_init(&empty[i], 1);
    for (int i = 0; i < kSlots; ++i) mbar_init(&s_full[i], 1), mbar_init(&s_empty[i], kOutWarps);
    for (int i = 0; i < kDbufs; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_empty[i], kOutWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_desc(&map_x);
  }
  if (warp == kMma) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_a = tmem_slot + kDbufs * BN, tmem_d = tmem_slot;
  const long long all = (long long)t.row_tiles * t.token_tiles * t.units;
  const long long u_begin = all * blockIdx.x / gridDim.x, u_end = all * (blockIdx.x + 1) / gridDim.x;
  const int n_kb = t.p.n_kb;
  volatile int* abort = &s_abort;

  if (warp < 8) {
    // ---- weights -> TMEM: a warpgroup takes every other block, a warp its 32 outputs of it -------------------------------------
    const int wg = warp >> 2, quarter = warp & 3;
    const uint8_t* weights = reinterpret_cast<const uint8_t*>(a.W);
    uint8_t* ring = sw + wg * kWslots * kSlotBytes;
    uint64_t *full = w_full + wg * kWslots, *freed = w_empty + wg * kWslots;
    Cursor ahead(t, u_begin, u_end), now(t, u_begin, u_end);
    if (wg == 1) ahead.next(), now.next();  // (a warpgroup takes every other unit)
    // One thread copies for the warpgroup: a unit's 8 KB lie one after the other, and so do its groups' scales.
    auto fetch = [&](int i) {
      if (ahead.left <= 0) return true;
      const int slot = i % kWslots;
      if (!mbar_wait(&freed[slot], ((i / kWslots) & 1) ^ 1, abort)) return false;
      const int blocks = min(2, n_kb - 2 * ahead.u), g = ahead.u * kSums, n_g = min(kSums, t.p.n_groups - g);
      mbar_expect_tx(&full[slot], blocks * kQ4TileBytes + (ZERO ? n_g * 512 : 0));
      bulk_load(ring + slot * kSlotBytes, weights + ((size_t)ahead.row_tile * n_kb + 2 * ahead.u) * kQ4TileBytes, blocks * kQ4TileBytes, &full[slot]);
      if (ZERO)
        bulk_load(ring + slot * kSlotBytes + 2 * kQ4TileBytes, t.p.table + ((size_t)ahead.row_tile * t.p.n_groups + g) * 512, n_g * 512, &full[slot]);
      ahead.next();
      ahead.next();
      return true;
    };
    const bool copies = quarter == 0 && lane == 0;
    // (weights and scales are never written by an earlier kernel of a step: the copies need not wait for it)
    if (copies)
      for (int i = 0; i < kWslots - 1; ++i) fetch(i);
    __syncwarp();
    int told = -1;  // unit whose stores are on their way to TMEM: told to the MMA warp while the next one is being expanded
    const auto tell = [&] {
      if (told < 0) return;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_full[told]);
      __syncwarp();
    };
    for (int i = 0; now.left > 0; ++i, now.next(), now.next()) {
      const int slot = i % kWslots;
      bool good = true;
      if (copies) good = fetch(i + kWslots - 1);
      if (!__all_sync(0xffffffffu, good && mbar_wait(&full[slot], (i / kWslots) & 1, abort))) {
        s_abort = 1;
        told = -1;
        break;
      }
      const uint8_t* sp = ring + slot * kSlotBytes + quarter * 1024 + lane * 16;
      const uint32_t* zp = reinterpret_cast<const uint32_t*>(ring + slot * kSlotBytes + 2 * kQ4TileBytes) + quarter * 32 + (lane >> 2);
      const int seq = 2 * i + wg, buf = seq % kBufs;
      uint4 w4[4];  // block, half of the warp's 32 outputs
#pragma unroll
      for (int h = 0; h < 4; ++h) w4[h] = *reinterpret_cast<const uint4*>(sp + (h >> 1) * kQ4TileBytes + (h & 1) * 512);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const uint32_t w[4] = {w4[h].x, w4[h].y, w4[h].z, w4[h].w};
        uint32_t r[16];
        uint32_t z0 = kQ4Middle, z1 = kQ4Middle;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (ZERO && (j == 0 || (G == 32 && j == 2))) {
            const uint32_t* e = zp + (G == 32 ? (h >> 1) * 2 + j / 2 : G == 64 ? (h >> 1) : 0) * 128 + (h & 1) * 16;
            z0 = __byte_perm(e[0], e[0], 0x3232), z1 = __byte_perm(e[8], e[8], 0x3232);
          }
          uint32_t q[4];
          q4_expand(w[j], z0, z1, q);
#pragma unroll
          for (int e = 0; e < 4; ++e) r[4 * j + e] = q[e];
        }
        if (h == 0) {
          tell();
          if (!__all_sync(0xffffffffu, mbar_wait(&empty[buf], ((seq / kBufs) & 1) ^ 1, abort))) {
            s_abort = 1;
            told = -1;
            break;
          }
          tc_fence_after();
          told = buf;
        }
        if (h == 3) {  // (everything of the slot has been read)
          __syncwarp();
          if (lane == 0) mbar_arrive(&freed[slot]);
          __syncwarp();
        }
        tmem_st_16x128b_x8(tmem_a + buf * 64 + (h >> 1) * 32 + ((uint32_t)(quarter * 32 + (h & 1) * 16) << 16), r);
      }
      if (told < 0) break;
    }
    tell();
    if (*abort && copies)  // copies may still be in flight: let them land before the shared memory goes to another CTA
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
  } else if (warp < kMma) {
    // ---- sums and outputs: one thread per output ---------------------------------------------------------------------------------
    const int row = tid & 127, col0 = (warp - 8) / 4 * kCols;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    float acc[kCols];
#pragma unroll
    for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
    pdl_wait();  // (scratch and outputs belong to earlier kernels until here)
    Cursor c(t, u_begin, u_end);
    long long unit = u_begin;
    int n = 0, seq = 0;  // accumulators and units taken
    bool ok = true;
    while (c.left > 0 && ok) {
      const int u0 = c.u, row_tile = c.row_tile, token0 = c.token_tile * BN + col0, n_units = min(c.left, t.units - u0);
      const long long seg_begin = unit, tile_begin = unit - u0, seg_end = unit + n_units;
      for (int k = 0; k < n_units && ok; ++k, ++seq) {
        const int slot = seq % kSlots, n_g = min(kSums, t.p.n_groups - (u0 + k) * kSums);
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[slot], (seq / kSlots) & 1, abort));
        const uint8_t* scales = ss + slot * kScaleBytes + row * kEntry;
#pragma unroll 1
        for (int g = 0; g < n_g && ok; ++g, ++n) {
          const float s = __uint_as_float((ZERO ? *reinterpret_cast<const uint32_t*>(scales + g * 512) : (uint32_t)*reinterpret_cast<const uint16_t*>(scales + g * 256)) << 16);
          const int d = n % kDbufs;
          ok = __all_sync(0xffffffffu, mbar_wait(&d_full[d], (n / kDbufs) & 1, abort));
          if (!ok) break;
          tc_fence_after();
          float v[2][16];
          const uint32_t from = tmem_d + d * BN + col0 + lanes;
          tmem_ld16_issue(from, v[0]);
#pragma unroll
          for (int b = 0; b < kCols / 16; ++b) {
            tmem_wait_ld16(v[b & 1]);
            if (b + 1 < kCols / 16) {
              tmem_ld16_issue(from + (b + 1) * 16, v[(b + 1) & 1]);
            } else {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&d_empty[d]);
              __syncwarp();
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[b * 16 + i] = fmaf(s, v[b & 1][i], acc[b * 16 + i]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[slot]);
        __syncwarp();
      }
      ok = out_all<32 * kOutWarps>(ok);
      if (!ok) break;
      // the segment is done: output, or a share of a tile that others have a part of
      const bool whole = seg_begin == tile_begin && seg_end == tile_begin + t.units;
      bool write = true;
      if (!whole) {
        // first and last CTA of the tile: the ones whose ranges hold its first and last unit
        auto cta_of = [&](long long unit) {
          int k = (int)(unit * gridDim.x / all);
          while (all * (k + 1) / gridDim.x <= unit) ++k;
          while (all * k / gridDim.x > unit) --k;
          return k;
        };
        const int c0 = cta_of(tile_begin), c1 = cta_of(tile_begin + t.units - 1);
        float* mine = t.parts + ((size_t)blockIdx.x * 2 + (seg_begin == tile_begin ? 1 : 0)) * (BN * kQ4Tile) + col0 * kQ4Tile + row;
#pragma unroll
        for (int i = 0; i < kCols; ++i) __stcg(mine + i * kQ4Tile, acc[i]);
        __threadfence();
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kOutWarps) : "memory");
        if (tid == 256) {
          const int before = atomicAdd(&t.counters[c0], 1);
          s_last = before == c1 - c0;
          if (before == c1 - c0) t.counters[c0] = 0;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kOutWarps) : "memory");
        write = s_last != 0;
        if (write) {
          __threadfence();
          const float* from = t.parts + ((size_t)c0 * 2 + 1) * (BN * kQ4Tile) + col0 * kQ4Tile + row;
#pragma unroll
          for (int i = 0; i < kCols; ++i) acc[i] = __ldcg(from + i * kQ4Tile);
          for (int k = c0 + 1; k <= c1; ++k) {
            from = t.parts + (size_t)k * 2 * (BN * kQ4Tile) + col0 * kQ4Tile + row;
#pragma unroll
            for (int i = 0; i < kCols; ++i) acc[i] += __ldcg(from + i * kQ4Tile);
          }
        }
      }
      if (write) {
        const int o = row_tile * kQ4Tile + row, n_tok = min(kCols, a.T - token0);
        if (a.u != nullptr && o < a.out) {
          const float* u = a.u + (size_t)token0 * (a.r_max * a.n_mod) + module_of(a, o) * a.r_max;
          for (int j = 0; j < a.r_max / 8; ++j) {
            int have = -1, sw;
            uint4 b = make_uint4(0u, 0u, 0u, 0u);
            float alpha = 0.f;
#pragma unroll
            for (int i = 0; i < kCols; ++i) {
              const int s = i < n_tok ? a.slots[token0 + i] : -1;
              if (s >= 0 && s < a.n_adapters) {
                if (s != have) {
                  b = ld_cached(q4_b_row(a, t.p.packed_b, s, o, j, sw));
                  alpha = a.scales[s];
                  have = s;
                }
                acc[i] = fmaf(alpha, dot8(b, u + (size_t)i * (a.r_max * a.n_mod) + 8 * j), acc[i]);
              }
            }
          }
        }
        const int act = a.flags & (MLORA_ACT_RELU2 | MLORA_ACT_GELU);
        if (a.flags & MLORA_SILU_MUL) {
#pragma unroll
          for (int i = 0; i < kCols; ++i) {
            const float up = __shfl_xor_sync(0xffffffffu, acc[i], 8);  // (8 gate outputs, then their 8 up outputs)
            if (!(lane & 8) && o < a.out && i < n_tok) store_out(a, token0 + i, o / 16 * 8 + (o & 7), silu_mul(acc[i], up));
          }
        } else if (o < a.out) {
#pragma unroll
          for (int i = 0; i < kCols; ++i)
            if (i < n_tok) store_out(a, token0 + i, o, act_one(acc[i], act));
        }
      }
#pragma unroll
      for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
      for (int k = 0; k < n_units; ++k) c.next();
      unit = seg_end;
    }
    if (!ok) s_abort = 1;
  } else {
    if (warp == kMma) {
      // ---- MMA issue -------------------------------------------------------------------------------------------------------------
      constexpr uint32_t idesc = make_idesc(kQ4Tile, BN);
      if (elect_one()) {  // (one thread: every instruction it spends per unit bounds the rate)
        const uint64_t b0 = make_smem_desc(smem_u32(sx));
        const uint32_t a_full0 = smem_u32(a_full), x_full0 = smem_u32(x_full), empty0 = smem_u32(empty), d_full0 = smem_u32(d_full),
                       d_empty0 = smem_u32(d_empty);
        uint32_t buf = 0, par = 0, d = 0, d_par = 1;
        bool ok = true;
        for (Cursor c(t, u_begin, u_end); c.left > 0 && ok; c.next()) {
          const int steps = min(8, (n_kb - 2 * c.u) * 4);  // of 16 inputs
          ok = mbar_wait_a(a_full0 + 8 * buf, par, abort) && mbar_wait_a(x_full0 + 8 * buf, par, abort);
          if (!ok) break;
          const uint64_t bdesc = b0 + (uint64_t)(buf * (BN * 256 >> 4));
          const uint32_t a_tmem = tmem_a + buf * 64;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (k < steps && ok) {
              const bool opens = k % (G / 16) == 0;
              if (opens) {
                ok = mbar_wait_a(d_empty0 + 8 * d, d_par, abort);
                tc_fence_after();
              }
              if (ok) umma_bf16_ta(tmem_d + d * BN, a_tmem + k * 8, bdesc + 2 * (k & 3) + (k >> 2) * (BN * 128 >> 4), idesc, opens ? 0u : 1u);
              if (ok && (k % (G / 16) == G / 16 - 1 || k + 1 == steps)) {
                umma_commit_a(d_full0 + 8 * d);
                if (++d == kDbufs) d = 0, d_par ^= 1;
              }
            }
          }
          if (!ok) break;
          umma_commit_a(empty0 + 8 * buf);
          if (++buf == kBufs) buf = 0, par ^= 1;
        }
        if (!ok) s_abort = 1;
      }
      __syncwarp();
    } else {
      // ---- rows of x, and the scales ------------------------------------------------------------------------------------------------
      pdl_wait();
      int seq = 0;
      for (Cursor c(t, u_begin, u_end); c.left > 0; c.next(), ++seq) {
        const int slot = seq % kBufs, s_slot = seq % kSlots;
        int good = 1;
        if (lane == 0) {
          good = mbar_wait(&empty[slot], ((seq / kBufs) & 1) ^ 1, abort);
          if (good) {
            const int blocks = min(2, n_kb - 2 * c.u);
            mbar_expect_tx(&x_full[slot], blocks * BN * 128);
            for (int b = 0; b < blocks; ++b)
              tma_load_2d(sx + (slot * 2 + b) * BN * 128, &map_x, (2 * c.u + b) * kQ4Block, c.token_tile * BN, &x_full[slot]);
            good = mbar_wait(&s_empty[s_slot], ((seq / kSlots) & 1) ^ 1, abort);
          }
          if (good) {
            const int g = c.u * kSums, bytes = min(kSums, t.p.n_groups - g) * kQ4Tile * kEntry;
            mbar_expect_tx(&s_full[s_slot], bytes);
            bulk_load(ss + s_slot * kScaleBytes, t.p.table + ((size_t)c.row_tile * t.p.n_groups + g) * kQ4Tile * kEntry, bytes, &s_full[s_slot]);
          }
        }
        good = __shfl_sync(0xffffffffu, good, 0);
        if (!good) {
          s_abort = 1;
          break;
        }
      }
      // commits arrive at these barriers until the last block's: nobody leaves before
      for (int k = max(seq - kBufs, 0); k < seq && !*abort; ++k)
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[k % kBufs], (k / kBufs) & 1, abort))) s_abort = 1;
      if (*abort && lane == 0)  // copies may still be in flight: let them land before the shared memory goes to another CTA
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && s_abort) atomicOr(t.status, 2);
  if (warp == kMma) tmem_dealloc(tmem_slot, 512);
}

int q4_ctas(long long units) {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = 148;
  }
  n = n < kMaxCtas ? n : kMaxCtas;
  return (int)(units < n ? units : n);
}
int rows_per_tile(int T) { return T <= 32 ? 32 : T <= 64 ? 64 : 128; }

template <int BN, bool ZERO, int G>
int launch_tc_as(const TcArgs& t, int grid, cudaStream_t st) {
  CUtensorMap mx;
  const int rc = make_map(&mx, t.p.a.x, t.p.a.T, t.p.a.in, t.p.a.ldx, BN, kQ4Block);
  if (rc) return rc;
  constexpr int smem = 1024 + kBufs * BN * 256 + 2 * kWslots * kSlotBytes + kSlots * kScaleBytes;
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!((done.load(std::memory_order_acquire) >> (dev & 63)) & 1ull)) {
    const cudaError_t e = cudaFuncSetAttribute(q4_tc_kernel<BN, ZERO, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(MLORA_ECUDA, "q4_linear: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done.fetch_or(1ull << (dev & 63), std::memory_order_release);
  }
  const cudaError_t e = launch_pdl_if(pdl_enabled_gemm(), q4_tc_kernel<BN, ZERO, G>, dim3((unsigned)grid), dim3(q4_threads(BN)), smem, st, mx, t);
  if (e != cudaSuccess) return fail(MLORA_ECUDA, "q4_tc_kernel: %s", cudaGetErrorString(e));
  count_launch();
  MLORA_CHECK_LAUNCH("q4_tc_kernel");
  return MLORA_OK;
}
template <int BN>
int launch_tc_for(const TcArgs& t, int grid, cudaStream_t st) {
  const bool zero = (t.p.a.flags & MLORA_Q4_ZEROS) != 0;
  switch (t.p.group) {
    case 32: return zero ? launch_tc_as<BN, true, 32>(t, grid, st) : launch_tc_as<BN, false, 32>(t, grid, st);
    case 64: return zero ? launch_tc_as<BN, true, 64>(t, grid, st) : launch_tc_as<BN, false, 64>(t, grid, st);
    default: return zero ? launch_tc_as<BN, true, 128>(t, grid, st) : launch_tc_as<BN, false, 128>(t, grid, st);
  }
}

}  // namespace

size_t q4_tc_workspace(int T, int in, int out) {
  // (the largest tile and every CTA, whatever the sizes: one buffer serves them all)
  (void)in, (void)out;
  return kHeader + kMaxCtas * 4 + (size_t)q4_ctas(kMaxCtas) * 2 * rows_per_tile(T) * kQ4Tile * 4;
}

int launch_q4_tc(const Q4Args& p, void* work, size_t work_bytes, cudaStream_t st) {
  const size_t need = q4_tc_workspace(p.a.T, p.a.in, p.a.out);
  if (!work || work_bytes < need) return fail(MLORA_ESIZE, "q4_linear: scratch of %zu bytes needed, %zu given", need, work_bytes);
  if (!aligned16(work)) return fail(MLORA_EINVAL, "q4_linear: the scratch must be 16-byte aligned");
  TcArgs t{};
  t.p = p;
  t.status = (int32_t*)work;
  t.counters = (int32_t*)((uint8_t*)work + kHeader);
  t.parts = (float*)((uint8_t*)work + kHeader + kMaxCtas * 4);
  const int bn = rows_per_tile(p.a.T);
  t.row_tiles = (p.a.out + kQ4Tile - 1) / kQ4Tile;
  t.token_tiles = (p.a.T + bn - 1) / bn;
  t.units = (p.n_kb + 1) / 2;
  if ((long long)t.row_tiles * t.token_tiles > 2147483647ll) return fail(MLORA_ESIZE, "q4_linear: too many tiles");
  const int grid = q4_ctas((long long)t.row_tiles * t.token_tiles * t.units);
  return bn == 32 ? launch_tc_for<32>(t, grid, st) : bn == 64 ? launch_tc_for<64>(t, grid, st) : launch_tc_for<128>(t, grid, st);
}

}  // namespace mlora
