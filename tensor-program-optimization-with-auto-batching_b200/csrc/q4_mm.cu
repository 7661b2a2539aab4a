// Projections with 4-bit weights for up to 16 rows (see q4.cuh for the layout): y = x W^T is bound by the weights' out in / 2 bytes, and on
// the way there by the integer pipe: shifts and masks of the eight weights of a word are seven instructions of two cycles, 224 cycles per
// 8 KB and SM sub-core against the 350 in which HBM delivers them.  So weights go from bulk copies in shared memory to registers and from
// there, as the A operand, straight into mma.m16n8k16, whose fragments the packed order has (8.3 cycles each and sub-core: 134 per 8 KB
// at up to eight rows); no TMEM, no hand-over between warps.  From 17 rows on the products of this path would cost more than the weights.
//
// A CTA's tile is 128 outputs x 8 or 16 rows; stages of 256 inputs -- 16 KB of weights, their scales, the rows of x -- arrive by bulk and
// TMA copies.  Eight warps: four ranges of 32 outputs x two sets of blocks of 64 inputs.  Persistent, two CTAs per SM, the stages of all
// tiles dealt out in equal ranges; a tile that several CTAs share is finished by the one that begins it, from the sums that the others
// have left in scratch -- the first thing each of them does.
//
// Measured (weights from HBM, CUDA graph, groups of 128): 1 x 4096 x 22016 17.8 us, 8 rows 18.0, 16 rows 21.3; 1 x 4096 x 4096 7.4; 7 x 11008 x
// 4096 in groups of 32 with zero points 14.2.  Without the products the copies alone take 13.4 us of the first, of which 5.7 are the
// launch, the first copy and the last sums.  16 or 24 warps, or one CTA per SM, are no faster (18.8, 19.9, 19.0).
#include "q4.cuh"
#include "tc_ptx.cuh"

#include <atomic>

namespace mlora {
namespace {

constexpr int kMmWarps = 8, kMmThreads = 32 * (kMmWarps + 1);  // and one warp for the copies
constexpr int kMmBlocks = 4;                                    // of 64 inputs per stage
constexpr int kMmSplit = 2;                                     // warps that share a range of outputs
constexpr int kMmPitch = 132;                                   // floats between rows of x in the sums

struct MmArgs {
  Q4Args p;
  Q4Work w;
  int row_tiles, token_tiles, units;  // stages per tile
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_more(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// One verdict of the 256 threads that multiply; see bar_all.
__device__ __forceinline__ bool mm_all(bool ok) {
  uint32_t r;
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.aligned.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

// N8: rows of x in eights; ZERO: zero points; G: inputs per group
template <int N8, bool ZERO, int G>
struct MmStage {
  static constexpr int kEntry = ZERO ? 4 : 2, kGroups = kMmBlocks * kQ4Block / G;
  static constexpr int kW = kMmBlocks * kQ4TileBytes, kX = kMmBlocks * N8 * 1024, kS = kGroups * kQ4Tile * kEntry;
  static constexpr int kBytes = (kW + kX + kS + 1023) / 1024 * 1024;  // (x is swizzled: 1024-byte places)
  static constexpr int kSums = kMmSplit * N8 * 8 * kMmPitch * 4;
  static constexpr int kStages = (227 * 1024 / 2 - 1024 - 1536 - kSums) / kBytes;  // (two CTAs per SM)
  static constexpr int kSmem = 1024 + kStages * kBytes + kSums;
};

template <int N8, bool ZERO, int G>
__global__ void __launch_bounds__(kMmThreads, 2) q4_mm_kernel(const __grid_constant__ CUtensorMap map_x, MmArgs t) {
  using S = MmStage<N8, ZERO, G>;
  constexpr int kStages = S::kStages, kEntry = S::kEntry;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);  // [stage][x | W | scales]
  float* sums = reinterpret_cast<float*>(ring + kStages * S::kBytes);                                            // [split][row of x][kMmPitch]
  __shared__ uint64_t bars[2 * kStages];
  uint64_t *const full = bars, *const empty = bars + kStages;
  __shared__ int s_abort;

  pdl_launch_dependents();
  const LinearArgs& a = t.p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], kMmWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_desc(&map_x);
  }
  __syncthreads();
  const long long all = (long long)t.row_tiles * t.token_tiles * t.units;
  const long long u_begin = all * blockIdx.x / gridDim.x, u_end = all * (blockIdx.x + 1) / gridDim.x;
  const int n_kb = t.p.n_kb, left = (int)(u_end - u_begin);
  volatile int* abort = &s_abort;
  int tile = (int)(u_begin / t.units), u = (int)(u_begin % t.units);  // of the unit at work

  if (warp == kMmWarps) {
    // ---- copies --------------------------------------------------------------------------------------------------------------------
    if (lane == 0) {
      // (one thread's instructions come one after the other: counters and running pointers instead of remainders and products; weights
      // and scales lie one stage after the other, whole tiles and all)
      struct Place {
        int u, row_tile, token;
        const uint8_t *weights, *table;
      };
      const uint8_t* weights0 = reinterpret_cast<const uint8_t*>(a.W);
      const int row_tile = tile % t.row_tiles, last_blocks = n_kb - (t.units - 1) * kMmBlocks;
      const int last_scales = (t.p.n_groups - (t.units - 1) * S::kGroups) * kQ4Tile * kEntry;
      Place at{u, row_tile, tile / t.row_tiles * (N8 * 8), weights0 + ((size_t)row_tile * n_kb + u * kMmBlocks) * kQ4TileBytes,
               t.p.table + ((size_t)row_tile * t.p.n_groups + u * S::kGroups) * kQ4Tile * kEntry};
      const auto copy_x = [&](int slot, uint8_t* dst) {
        const int blocks = at.u == t.units - 1 ? last_blocks : kMmBlocks;
#pragma unroll
        for (int b = 0; b < kMmBlocks; ++b)
          if (b < blocks) tma_load_2d(dst + b * N8 * 1024, &map_x, at.u * (kMmBlocks * kQ4Block) + b * kQ4Block, at.token, &full[slot]);
      };
      const auto copy_w = [&](int slot, uint8_t* dst) {
        const bool last = at.u == t.units - 1;
        const int blocks = last ? last_blocks : kMmBlocks, bytes = last ? last_scales : S::kS;
        mbar_expect_tx(&full[slot], blocks * (kQ4TileBytes + N8 * 1024) + bytes);
        bulk_load(dst + S::kX, at.weights, blocks * kQ4TileBytes, &full[slot]);
        bulk_load(dst + S::kX + S::kW, at.table, bytes, &full[slot]);
        at.weights += blocks * kQ4TileBytes;
        at.table += bytes;
      };
      const auto next = [&] {
        if (++at.u < t.units) return;
        at.u = 0;
        if (++at.row_tile == t.row_tiles) at.row_tile = 0, at.token += N8 * 8, at.weights = weights0, at.table = t.p.table;
      };
      // the first stages' weights and scales, which no earlier kernel of a step writes; then, behind that kernel, their rows of x
      const int ahead = min(left, kStages);
      const Place begin = at;
      for (int i = 0; i < ahead; ++i, next()) copy_w(i, ring + i * S::kBytes);
      const Place then = at;
      pdl_wait();
      at = begin;
      for (int i = 0; i < ahead; ++i, next()) copy_x(i, ring + i * S::kBytes);
      at = then;
      uint32_t par = 0;
      int slot = 0;
      uint8_t* dst = ring;
      for (int i = ahead; i < left; ++i, next()) {
        if (!mbar_wait(&empty[slot], par, abort)) {
          s_abort = 1;
          break;
        }
        copy_w(slot, dst);
        copy_x(slot, dst);
        dst += S::kBytes;
        if (++slot == kStages) slot = 0, par ^= 1, dst = ring;
      }
      if (*abort)  // copies may still be in flight: let them land before the shared memory goes to another CTA
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
  } else {
    // ---- products --------------------------------------------------------------------------------------------------------------------
    const int quarter = warp / kMmSplit, block = warp % kMmSplit, g = lane >> 2;
    float acc[2][N8][4];
    const auto clear = [&] {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < N8; ++n) acc[h][n][0] = acc[h][n][1] = acc[h][n][2] = acc[h][n][3] = 0.f;
    };
    clear();
    bool ok = true, waited = false;
    // (the integer pipe is what this loop is bound by: running pointers, no remainders)
    const uint8_t* stage = ring;
    const uint8_t* const ring_end = ring + kStages * S::kBytes;
    uint64_t* bar = full;
    uint32_t par = 0;
    const uint32_t x_lane = block * N8 * 1024 + (lane & 7) * 128;  // (the warp's first block; the other lies kMmSplit blocks further)
    const int w_lane = S::kX + block * kQ4TileBytes + quarter * 1024 + lane * 16, s_lane = S::kX + S::kW + (quarter * 32 + g) * kEntry;
    const uint32_t x_piece[2] = {(uint32_t)(((lane >> 3) ^ (lane & 7)) << 4), (uint32_t)(((4 + (lane >> 3)) ^ (lane & 7)) << 4)};
    const int last_blocks = n_kb - (t.units - 1) * kMmBlocks;
    for (int i = 0; i < left;) {
      const int seg = min(left - i, t.units - u);  // stages of this tile
      const int u_first = u;
      for (int e = i + seg; i < e; ++i, ++u) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar, par, abort));
        if (!ok) break;
        const int blocks = u + 1 < t.units ? kMmBlocks : last_blocks;
        const uint32_t sx = smem_u32(stage) + x_lane;
        const uint8_t* sw = stage + w_lane;
        const uint8_t* ss = stage + s_lane;
#pragma unroll
        for (int q = 0; q < kMmBlocks / kMmSplit; ++q) {
          if (block + q * kMmSplit >= blocks) break;
          uint4 w4[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) w4[h] = *reinterpret_cast<const uint4*>(sw + q * kMmSplit * kQ4TileBytes + h * 512);
          uint32_t b[N8][2][4];  // rows 8 n .. of x: inputs 32 h .. 32 h + 31 of the block
#pragma unroll
          for (int n = 0; n < N8; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) ldmatrix4(sx + (q * kMmSplit * N8 + n) * 1024 + x_piece[h], b[n][h]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w[4] = {w4[h].x, w4[h].y, w4[h].z, w4[h].w};
            float sum[N8][4], s0 = 0.f, s1 = 0.f;
            uint32_t z0 = kQ4Middle, z1 = kQ4Middle;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              constexpr int kWords = G == 32 ? 2 : 4;  // of a group in this block
              if (j % kWords == 0) {
                const int at = block + q * kMmSplit;
                // (inputs that end inside a block: its second group is not there, and x is 0)
                const int group = G == 32 ? min(at * 2 + j / 2, t.p.n_groups - u * S::kGroups - 1) : G == 64 ? at : at / 2;
                const uint8_t* e = ss + (group * kQ4Tile + h * 16) * kEntry;
                if constexpr (ZERO) {
                  const uint32_t e0 = *reinterpret_cast<const uint32_t*>(e), e1 = *reinterpret_cast<const uint32_t*>(e + 8 * 4);
                  s0 = __uint_as_float(e0 << 16), s1 = __uint_as_float(e1 << 16);
                  z0 = __byte_perm(e0, e0, 0x3232), z1 = __byte_perm(e1, e1, 0x3232);
                } else {
                  s0 = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(e) << 16);
                  s1 = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(e + 8 * 2) << 16);
                }
              }
              uint32_t r[4];
              q4_expand(w[j], z0, z1, r);
#pragma unroll
              for (int n = 0; n < N8; ++n) {
                if (j % kWords == 0)
                  mma_first(sum[n], r, b[n][j >> 1][(j & 1) * 2], b[n][j >> 1][(j & 1) * 2 + 1]);
                else
                  mma_more(sum[n], r, b[n][j >> 1][(j & 1) * 2], b[n][j >> 1][(j & 1) * 2 + 1]);
              }
              if (j % kWords == kWords - 1) {
#pragma unroll
                for (int n = 0; n < N8; ++n) {
                  acc[h][n][0] = fmaf(s0, sum[n][0], acc[h][n][0]), acc[h][n][1] = fmaf(s0, sum[n][1], acc[h][n][1]);
                  acc[h][n][2] = fmaf(s1, sum[n][2], acc[h][n][2]), acc[h][n][3] = fmaf(s1, sum[n][3], acc[h][n][3]);
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar + kStages);
        stage += S::kBytes;
        ++bar;
        if (stage == ring_end) stage = ring, bar = full, par ^= 1;
      }
      ok = mm_all(ok);  // (also: the sums before have been read)
      if (!ok) break;
      // ---- the segment is done: the two warps' sums, then output, or a share of a tile that another CTA finishes -----------------
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < N8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sums[(block * N8 * 8 + n * 8 + (lane & 3) * 2 + (e & 1)) * kMmPitch + quarter * 32 + h * 16 + (e >> 1) * 8 + g] = acc[h][n][e];
      clear();
      if (!waited) {
        pdl_wait();  // (scratch and outputs belong to earlier kernels until here)
        waited = true;
      }
      mm_all(true);
      const long long tile_begin = (long long)tile * t.units;
      const int row0 = tile % t.row_tiles * kQ4Tile, token0 = tile / t.row_tiles * (N8 * 8), n_tok = a.T - token0;
      // a thread: one output of every kApart-th row of x
      constexpr int kApart = kMmWarps / 4, kMine = (N8 * 8 + kApart - 1) / kApart;
      const int c = tid & 127, tok0 = tid >> 7;
      float v[kMine];
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        v[k] = 0.f;
        if (tok0 + kApart * k < N8 * 8) {
          const float* s = sums + (tok0 + kApart * k) * kMmPitch + c;
#pragma unroll
          for (int q = 0; q < kMmSplit; ++q) v[k] += s[q * N8 * 8 * kMmPitch];
        }
      }
      if (u_first != 0) {
        float* mine = t.w.parts + (size_t)blockIdx.x * (kQ4Tile * kQ4Tile) + tok0 * kQ4Tile + c;
#pragma unroll
        for (int k = 0; k < kMine; ++k)
          if (tok0 + kApart * k < N8 * 8) __stcg(mine + kApart * k * kQ4Tile, v[k]);
        mm_all(true);
        if (tid == 0) {
          __threadfence();
          atomicAdd(&t.w.counters[q4_cta_of(tile_begin, all, gridDim.x)], 1);
        }
      } else {
        const int o = row0 + c;
        const bool there = o < a.out;
        if constexpr (N8 == 1) {
          if (a.u != nullptr && there) {  // (two values a thread: quicker here than a kernel of its own in front of this one)
#pragma unroll
            for (int k = 0; k < kMine; ++k)
              if (tok0 + kApart * k < n_tok) v[k] += q4_adapter(a, t.p.packed_b, token0 + tok0 + kApart * k, o);
          }
        } else if (t.w.delta != nullptr) {
          float add[kMine];
#pragma unroll
          for (int k = 0; k < kMine; ++k) add[k] = there && tok0 + kApart * k < n_tok ? __ldcg(t.w.delta + (size_t)(token0 + tok0 + kApart * k) * a.out + o) : 0.f;
#pragma unroll
          for (int k = 0; k < kMine; ++k) v[k] += add[k];
        }
        if (u != t.units) {  // others have a part: each of them writes it before anything else
          const int last = q4_cta_of(tile_begin + t.units - 1, all, gridDim.x);
          if (tid == 0) {
            ok = false;
            for (uint32_t k = 0; k < kSpinLimit && !ok; ++k) {
              int have;
              asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(have) : "l"(&t.w.counters[blockIdx.x]) : "memory");
              ok = have >= last - (int)blockIdx.x;
              if (!ok) __nanosleep(64);
              if ((k & 255) == 255 && *abort) break;
            }
            t.w.counters[blockIdx.x] = 0;
          }
          ok = mm_all(ok);
          if (!ok) break;
#pragma unroll 4
          for (int part = blockIdx.x + 1; part <= last; ++part) {
            const float* from = t.w.parts + (size_t)part * (kQ4Tile * kQ4Tile) + tok0 * kQ4Tile + c;
#pragma unroll
            for (int k = 0; k < kMine; ++k)
              if (tok0 + kApart * k < N8 * 8) v[k] += __ldcg(from + kApart * k * kQ4Tile);
          }
        }
        const bool silu = (a.flags & MLORA_SILU_MUL) != 0;
        const int act = a.flags & (MLORA_ACT_RELU2 | MLORA_ACT_GELU), col = silu ? o / 16 * 8 + (o & 7) : o;
        if (silu) {
#pragma unroll
          for (int k = 0; k < kMine; ++k) v[k] = silu_mul(v[k], __shfl_xor_sync(0xffffffffu, v[k], 8));  // (8 gate outputs, then their 8 up outputs)
        } else if (act) {
#pragma unroll
          for (int k = 0; k < kMine; ++k) v[k] = q4_act(v[k], act);
        }
        if (there && (!silu || !(c & 8))) {
#pragma unroll
          for (int k = 0; k < kMine; ++k)
            if (tok0 + kApart * k < n_tok) store_out(a, token0 + tok0 + kApart * k, col, v[k]);
        }
      }
      if (u == t.units) u = 0, ++tile;
    }
    if (!ok) s_abort = 1;
  }
  __syncthreads();
  if (tid == 0 && s_abort) atomicOr(t.w.status, 2);
}

template <int N8, bool ZERO, int G>
int launch_mm_as(const MmArgs& t, int grid, cudaStream_t st) {
  CUtensorMap mx;
  const int rc = make_map(&mx, t.p.a.x, t.p.a.T, t.p.a.in, t.p.a.ldx, N8 * 8, kQ4Block);
  if (rc) return rc;
  constexpr int smem = MmStage<N8, ZERO, G>::kSmem;
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!((done.load(std::memory_order_acquire) >> (dev & 63)) & 1ull)) {
    const cudaError_t e = cudaFuncSetAttribute(q4_mm_kernel<N8, ZERO, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(MLORA_ECUDA, "q4_linear: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done.fetch_or(1ull << (dev & 63), std::memory_order_release);
  }
  const cudaError_t e = launch_pdl_if(pdl_enabled_gemm(), q4_mm_kernel<N8, ZERO, G>, dim3((unsigned)grid), dim3(kMmThreads), smem, st, mx, t);
  if (e != cudaSuccess) return fail(MLORA_ECUDA, "q4_mm_kernel: %s", cudaGetErrorString(e));
  count_launch();
  MLORA_CHECK_LAUNCH("q4_mm_kernel");
  return MLORA_OK;
}
template <int N8>
int launch_mm_for(const MmArgs& t, int grid, cudaStream_t st) {
  const bool zero = (t.p.a.flags & MLORA_Q4_ZEROS) != 0;
  switch (t.p.group) {
    case 32: return zero ? launch_mm_as<N8, true, 32>(t, grid, st) : launch_mm_as<N8, false, 32>(t, grid, st);
    case 64: return zero ? launch_mm_as<N8, true, 64>(t, grid, st) : launch_mm_as<N8, false, 64>(t, grid, st);
    default: return zero ? launch_mm_as<N8, true, 128>(t, grid, st) : launch_mm_as<N8, false, 128>(t, grid, st);
  }
}

}  // namespace

int launch_q4_mm(const Q4Args& p, const Q4Work& w, cudaStream_t st) {
  const int n8 = p.a.T <= 8 ? 1 : 2;
  MmArgs t{p, w, (p.a.out + kQ4Tile - 1) / kQ4Tile, (p.a.T + n8 * 8 - 1) / (n8 * 8), (p.n_kb + kMmBlocks - 1) / kMmBlocks};
  const long long all = (long long)t.row_tiles * t.token_tiles * t.units;
  if (all > 2147483647ll) return fail(MLORA_ESIZE, "q4_linear: too many tiles");
  const int grid = q4_ctas(t.row_tiles * (long long)t.token_tiles, t.units, 2);
  return n8 == 1 ? launch_mm_for<1>(t, grid, st) : launch_mm_for<2>(t, grid, st);
}

}  // namespace mlora
