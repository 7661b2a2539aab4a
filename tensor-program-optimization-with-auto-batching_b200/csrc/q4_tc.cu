// Projections with 4-bit weights on the 5th-generation tensor cores, for more than 16 rows (see q4.cuh for the layout).
//
// Tiles of 128 outputs x BN rows of x, in units of 128 inputs.  Eight warps take packed weights from rings of bulk copies, turn them into
// bf16 integers q - z and write them to TMEM (tcgen05.st.16x128b has the lanes where the packed order has them): weights go DRAM -> shared
// memory -> registers -> TMEM and are never written to shared memory as bf16, whose 32 KB per 8 KB of weights would be more than its
// bandwidth.  The MMA takes them from there as its A operand -- 16 cycles per m128n32k16, against 40 from shared memory -- and the rows of
// x (TMA, 128-byte swizzle) as B.  A group's sums have an accumulator of their own, which 4, 8 or 16 warps scale in fp32 registers
// while the next ones are filled: nothing but the output is rounded.
//
// Persistent, one CTA per SM; the units of all tiles are dealt out in equal ranges.  A tile that several CTAs share is finished by the one
// that begins it: the others leave their sums in scratch -- the first thing each of them does -- and it adds them up in the order of the
// inputs.  Adapters are expanded by a kernel of their own in front of this one, into fp32 scratch that is added to the sums: a thread here
// has one output and many rows, whose adapters' rows it would have to wait for one after the other.
//
// What bounds it: the warps that hand units on.  Their instructions come one after the other, some ten cycles each among the 19 or 27
// warps of an SM: with one unit per barrier, counters instead of remainders and one barrier for weights and rows of x a unit takes 950
// cycles at 32 rows, against 350 in which HBM delivers it and 128 in which it is multiplied.  Groups of 32 or 64 have an accumulator to
// hand on for each of them.  Measured (CUDA graph): 32 x 4096 x 22016 25.6 us, 128 rows 36.3, 512 x 4096 x 11008 58.7 (787 TFLOP/s);
// 32 x 4096 x 22016 in groups of 32 44.4.
#include "q4.cuh"
#include "tc_ptx.cuh"

#include <atomic>

namespace mlora {
namespace {

// Warps: weight warpgroups, then those that sum and write (32 columns each), then MMA issue, copies of x,
// copies of weights.
constexpr int q4_weight_groups(int bn) { return bn == 32 ? 3 : 2; }
constexpr int q4_out_warps(int bn) { return bn / 8; }
constexpr int q4_threads(int bn) { return 32 * (4 * q4_weight_groups(bn) + q4_out_warps(bn) + 3); }
constexpr int q4_ring(int bn) { return bn == 32 ? 9 : bn == 64 ? 8 : 6; }  // packed units in shared memory: as many for every weight warpgroup
constexpr int q4_bufs(int bn) { return bn == 128 ? 4 : 6; }  // units of weights in TMEM, and of x in shared memory (from L2, 1 us away)
// Units whose scales lie in shared memory.  A slot is filled again without asking: copies are at most q4_bufs units ahead of the MMAs,
// which are at most as many accumulators (q4_sums, one or more a unit) ahead of the warps that read scales.
constexpr int q4_sums(int bn) { return bn == 32 ? 4 : 2; }
constexpr int q4_scale_slots(int bn) { return q4_bufs(bn) + q4_sums(bn) + 1; }
constexpr int q4_scale_bytes(bool zero, int g) { return 128 / g * kQ4Tile * (zero ? 4 : 2); }  // of a unit's groups
constexpr int q4_slot_bytes(bool zero, int g) { return 2 * kQ4TileBytes + (zero ? q4_scale_bytes(zero, g) : 0); }
constexpr int q4_smem(int bn, bool zero, int g) {
  return 1024 + q4_bufs(bn) * bn * 256 + q4_ring(bn) * q4_slot_bytes(zero, g) + q4_scale_slots(bn) * q4_scale_bytes(zero, g);
}

struct TcArgs {
  Q4Args p;
  int32_t* status;
  int32_t* counters;  // [CTA that the tile begins in]: shares that have arrived, zero between calls
  float* parts;       // [CTA][BN][128]: sums of a CTA's share of a tile that another CTA begins
  const float* delta; // [rows][out]: the adapters' share, or NULL
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
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// (the registers go through the wait, so that nothing that reads them is scheduled before it)
template <int N>
__device__ __forceinline__ void tmem_wait_ld_all(float* v) {
#pragma unroll
  for (int i = 0; i < N; i += 16) tmem_wait_ld16(v + i);
}
template <int N>
__device__ __forceinline__ void out_sync() {
  __syncwarp();
  asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
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
  constexpr int kDbufs = q4_sums(BN), kSlots = q4_scale_slots(BN);
  constexpr int kGroups = q4_weight_groups(BN), kWarpsOut = q4_out_warps(BN);
  constexpr int kOut = 4 * kGroups, kMma = kOut + kWarpsOut;  // first warps of these roles
  constexpr int kCols = BN * 4 / kWarpsOut;               // columns of a thread that sums
  constexpr int kSums = 128 / G;                          // groups of a unit
  constexpr int kEntry = ZERO ? 4 : 2;
  constexpr int kWslots = q4_ring(BN), kBufs = q4_bufs(BN), kSlotBytes = q4_slot_bytes(ZERO, G), kScaleBytes = q4_scale_bytes(ZERO, G);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sx = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sw = sx + kBufs * BN * 256;                  // [slot][kSlotBytes]
  uint8_t* ss = sw + kWslots * kSlotBytes;                // [slot][kScaleBytes]
  __shared__ uint64_t w_full[kWslots], w_empty[kWslots], full[kBufs], empty[kBufs], d_full[kDbufs], d_empty[kDbufs];
  __shared__ uint32_t tmem_slot;
  __shared__ int s_abort;

  pdl_launch_dependents();
  const LinearArgs& a = t.p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < kWslots; ++i) mbar_init(&w_full[i], 1), mbar_init(&w_empty[i], 4);
    for (int i = 0; i < kBufs; ++i) mbar_init(&full[i], 4 + 1), mbar_init(&empty[i], 1);  // (four weight warps, and the copies of x)
    for (int i = 0; i < kDbufs; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_empty[i], kWarpsOut);
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

  if (warp < kOut) {
    // ---- weights -> TMEM: the warpgroups take the units in turn, a warp its 32 outputs -----------------------------------------
    const int wg = warp >> 2, quarter = warp & 3, n_units = (int)(u_end - u_begin);
    int told = -1;  // unit whose stores are on their way to TMEM: told to the MMA warp while the next one is being expanded
    const auto tell = [&] {
      if (told < 0) return;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[told]);
      __syncwarp();
    };
    static_assert(kWslots % kGroups == 0 && kBufs % kGroups == 0, "every warpgroup has slots and buffers of its own");
    int slot = wg, buf = wg;
    uint32_t w_par = 0, a_par = 1;
    for (int seq = wg; seq < n_units; seq += kGroups) {
      if (!__all_sync(0xffffffffu, mbar_wait(&w_full[slot], w_par, abort))) {
        s_abort = 1;
        told = -1;
        break;
      }
      const uint8_t* sp = sw + slot * kSlotBytes + quarter * 1024 + lane * 16;
      const uint32_t* zp = reinterpret_cast<const uint32_t*>(sw + slot * kSlotBytes + 2 * kQ4TileBytes) + quarter * 32 + (lane >> 2);
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
          if (!__all_sync(0xffffffffu, mbar_wait(&empty[buf], a_par, abort))) {
            s_abort = 1;
            told = -1;
            break;
          }
          tc_fence_after();
          told = buf;
        }
        if (h == 3) {  // (everything of the slot has been read)
          __syncwarp();
          if (lane == 0) mbar_arrive(&w_empty[slot]);
          __syncwarp();
        }
        tmem_st_16x128b_x8(tmem_a + buf * 64 + (h >> 1) * 32 + ((uint32_t)(quarter * 32 + (h & 1) * 16) << 16), r);
      }
      if (told < 0) break;
      if ((slot += kGroups) >= kWslots) slot = wg, w_par ^= 1;
      if ((buf += kGroups) >= kBufs) buf = wg, a_par ^= 1;
    }
    tell();
  } else if (warp < kMma) {
    // ---- sums and outputs: one thread per output ---------------------------------------------------------------------------------
    const int row = (warp - kOut) % 4 * 32 + lane, col0 = (warp - kOut) / 4 * kCols;  // (kOut is a multiple of 4: row / 32 = warp % 4)
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    float acc[kCols];
#pragma unroll
    for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
    pdl_wait();  // (scratch and outputs belong to earlier kernels until here)
    Cursor c(t, u_begin, u_end);
    long long unit = u_begin;
    int s_slot = 0;
    uint32_t d = 0, d_par = 0;
    const uint32_t d_full0 = smem_u32(d_full);
    bool ok = true;
    while (c.left > 0 && ok) {
      const int u0 = c.u, token0 = c.token_tile * BN + col0, n_units = min(c.left, t.units - u0);
      const long long seg_begin = unit, tile_begin = unit - u0, seg_end = unit + n_units;
      for (int k = 0; k < n_units && ok; ++k) {
        const int n_g = min(kSums, t.p.n_groups - (u0 + k) * kSums);
        const uint8_t* scales = ss + s_slot * kScaleBytes + row * kEntry;
        if (++s_slot == kSlots) s_slot = 0;
#pragma unroll 1
        for (int g = 0; g < n_g; ++g, scales += kQ4Tile * kEntry) {
          // (a unit's scales arrive at the barrier of its rows of x, which the MMAs have waited for)
          ok = __all_sync(0xffffffffu, mbar_wait_a(d_full0 + 8 * d, d_par, abort));
          if (!ok) break;
          tc_fence_after();
          const uint32_t from = tmem_d + d * BN + col0 + lanes;
          const float s = __uint_as_float((ZERO ? *reinterpret_cast<const uint32_t*>(scales) : (uint32_t)*reinterpret_cast<const uint16_t*>(scales)) << 16);
          constexpr int kStep = BN == 128 ? 16 : 32;  // (27 warps have registers for 16 columns on their way)
#pragma unroll
          for (int c0 = 0; c0 < kCols; c0 += kStep) {
            float v[kStep];
            if constexpr (kStep == 32) tmem_ld32_issue(from + c0, v); else tmem_ld16_issue(from + c0, v);
            tmem_wait_ld_all<kStep>(v);
            if (c0 + kStep == kCols) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&d_empty[d]);
              if (++d == kDbufs) d = 0, d_par ^= 1;
            }
#pragma unroll
            for (int i = 0; i < kStep; ++i) acc[c0 + i] = fmaf(s, v[i], acc[c0 + i]);
          }
        }
      }
      ok = out_all<32 * kWarpsOut>(ok);
      if (!ok) break;
      const bool begins = seg_begin == tile_begin, whole = begins && seg_end == tile_begin + t.units;
      int first = blockIdx.x, last = blockIdx.x;  // CTAs whose ranges hold the tile's first and last unit
      if (!whole) {
        first = q4_cta_of(tile_begin, all, gridDim.x), last = q4_cta_of(tile_begin + t.units - 1, all, gridDim.x);
      }
      if (!begins) {
        float* mine = t.parts + (size_t)blockIdx.x * (BN * kQ4Tile) + col0 * kQ4Tile + row;
#pragma unroll
        for (int i = 0; i < kCols; ++i) __stcg(mine + i * kQ4Tile, acc[i]);
        out_sync<32 * kWarpsOut>();
        if (warp == kOut && lane == 0) {
          __threadfence();
          atomicAdd(&t.counters[first], 1);
        }
        __syncwarp();
      } else {
        if (!whole) {  // wait for the others' shares (each CTA writes its own before anything else)
          if (lane == 0) {
            ok = false;
            for (uint32_t i = 0; i < kSpinLimit && !ok; ++i) {
              int have;
              asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(have) : "l"(&t.counters[first]) : "memory");
              ok = have >= last - first;
              if (!ok) __nanosleep(64);
              if ((i & 255) == 255 && *abort) break;
            }
          }
          ok = out_all<32 * kWarpsOut>(__shfl_sync(0xffffffffu, (int)ok, 0) != 0);
          if (!ok) break;
          if (warp == kOut && lane == 0) t.counters[first] = 0;  // (all of them have seen it)
        }
        const int o = c.row_tile * kQ4Tile + row, n_tok = min(kCols, a.T - token0), act = a.flags & (MLORA_ACT_RELU2 | MLORA_ACT_GELU);
        const bool silu = (a.flags & MLORA_SILU_MUL) != 0, mine = o < a.out && (!silu || !(lane & 8));
        const int col = silu ? o / 16 * 8 + (o & 7) : o;
#pragma unroll 1
        for (int k = first + 1; k <= last; ++k) {
          const float* from = t.parts + (size_t)k * (BN * kQ4Tile) + col0 * kQ4Tile + row;
#pragma unroll
          for (int c0 = 0; c0 < kCols; c0 += 16) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __ldcg(from + (c0 + i) * kQ4Tile);
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[c0 + i] += v[i];
          }
        }
        // 16 columns at a time, with one copy of the code for them all: unrolled over the columns it would come from memory instruction
        // by instruction, a tile at a time
#pragma unroll 1
        for (int c0 = 0; c0 < n_tok; c0 += 16) {
          float v[16], add[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = acc[i];
#pragma unroll
          for (int i = 0; i + 16 < kCols; ++i) acc[i] = acc[i + 16];
          if (t.delta != nullptr) {
#pragma unroll
            for (int i = 0; i < 16; ++i) add[i] = o < a.out && c0 + i < n_tok ? __ldcg(t.delta + (size_t)(token0 + c0 + i) * a.out + o) : 0.f;
          }
          if (t.delta != nullptr) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] += add[i];
          }
          if (silu) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = silu_mul(v[i], __shfl_xor_sync(0xffffffffu, v[i], 8));  // (8 gate outputs, then their 8 up outputs)
          } else if (act) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = q4_act(v[i], act);
          }
          if (mine) {
            const size_t at = (size_t)(token0 + c0) * a.ldy + col;
            if (a.flags & MLORA_OUT_F32) {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (c0 + i < n_tok) reinterpret_cast<float*>(a.y)[at + (size_t)i * a.ldy] = v[i];
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (c0 + i < n_tok) reinterpret_cast<bf16*>(a.y)[at + (size_t)i * a.ldy] = __float2bfloat16_rn(v[i]);
            }
          }
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
      if (elect_one()) {  // (one thread: its instructions come one after the other, and all of them bound the rate)
        const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty), d_full0 = smem_u32(d_full), d_empty0 = smem_u32(d_empty);
        const uint64_t desc = make_smem_desc(smem_u32(sx));
        const uint32_t desc_hi = (uint32_t)(desc >> 32), desc_lo = (uint32_t)desc;
        const int n_units = (int)(u_end - u_begin), last_steps = (a.in - (t.units - 1) * 128) / 16;  // (a group that is not there has no accumulator)
        int u = (int)(u_begin % t.units);
        uint32_t buf = 0, par = 0, d = 0, d_par = 1;
        bool ok = true;
        for (int i = 0; i < n_units; ++i) {
          ok = mbar_wait_a(full0 + 8 * buf, par, abort);
          if (!ok) break;
          const uint32_t b_lo = desc_lo + buf * (BN * 256 >> 4), a_tmem = tmem_a + buf * 64;
          const bool last = u == t.units - 1;
          u = last ? 0 : u + 1;
          const int groups = last ? (last_steps + G / 16 - 1) / (G / 16) : kSums;
#pragma unroll
          for (int s = 0; s < kSums; ++s) {
            if (s < groups && ok) {
              ok = mbar_wait_a(d_empty0 + 8 * d, d_par, abort);
              tc_fence_after();
              const uint32_t d_tmem = tmem_d + d * BN;
#pragma unroll
              for (int k = s * (G / 16); k < (s + 1) * (G / 16); ++k)
                if (G != 128 || !last || k < last_steps)
                  umma_bf16_ta(d_tmem, a_tmem + k * 8, (uint64_t)desc_hi << 32 | (b_lo + 2 * (k & 3) + (k >> 2) * (BN * 128 >> 4)), idesc, k % (G / 16) != 0);
              umma_commit_a(d_full0 + 8 * d);
              if (++d == kDbufs) d = 0, d_par ^= 1;
            }
          }
          if (!ok) break;
          umma_commit_a(empty0 + 8 * buf);
          if (++buf == kBufs) buf = 0, par ^= 1;
        }
        if (!ok) s_abort = 1;
      }
      __syncwarp();
    } else if (warp == kMma + 1) {
      // ---- rows of x and scales -----------------------------------------------------------------------------------------------------------------
      if (lane == 0) {
        pdl_wait();
        // (as in the MMA warp one thread's instructions bound the rate: counters instead of remainders, and scales lie one unit after the
        // other, whole tiles and all)
        const int n_units = (int)(u_end - u_begin);
        int u = (int)(u_begin % t.units), row_tile = (int)(u_begin / t.units) % t.row_tiles, token = (int)(u_begin / t.units / t.row_tiles) * BN;
        const int last_blocks = n_kb - 2 * (t.units - 1), last_bytes = (t.p.n_groups - (t.units - 1) * kSums) * kQ4Tile * kEntry;
        const uint8_t* table = t.p.table + ((size_t)row_tile * t.p.n_groups + u * kSums) * kQ4Tile * kEntry;
        int slot = 0, s_slot = 0;
        uint32_t par = 1;
        uint8_t *dst = sx, *s_dst = ss;
        for (int i = 0; i < n_units; ++i) {
          if (!mbar_wait(&empty[slot], par, abort)) {
            s_abort = 1;
            break;
          }
          const bool last = u == t.units - 1;
          const int bytes = last ? last_bytes : kScaleBytes;
          mbar_expect_tx(&full[slot], (last && last_blocks == 1 ? BN * 128 : BN * 256) + bytes);
          tma_load_2d(dst, &map_x, u * 128, token, &full[slot]);
          if (!last || last_blocks == 2) tma_load_2d(dst + BN * 128, &map_x, u * 128 + 64, token, &full[slot]);
          bulk_load(s_dst, table, bytes, &full[slot]);
          table += bytes;
          ++u;
          if (last) {
            u = 0;
            if (++row_tile == t.row_tiles) row_tile = 0, token += BN, table = t.p.table;
          }
          dst += BN * 256;
          if (++slot == kBufs) slot = 0, par ^= 1, dst = sx;
          s_dst += kScaleBytes;
          if (++s_slot == kSlots) s_slot = 0, s_dst = ss;
        }
        const int seq = n_units;
        // commits arrive at these barriers until the last unit's: nobody leaves before
        for (int k = max(seq - kBufs, 0); k < seq && !*abort; ++k)
          if (!mbar_wait(&empty[k % kBufs], (k / kBufs) & 1, abort)) s_abort = 1;
        if (*abort)  // copies may still be in flight: let them land before the shared memory goes to another CTA
          for (int i = 0; i < 64; ++i) __nanosleep(1000);
      }
    } else if (lane == 0) {
      // ---- packed weights: a unit's 8 KB lie one after the other, and so do its groups' scales (no earlier kernel of a step writes
      // either, so the copies need not wait for it) --------------------------------------------------------------------------------
      const int n_units = (int)(u_end - u_begin);
      int u = (int)(u_begin % t.units), row_tile = (int)(u_begin / t.units) % t.row_tiles, slot = 0;
      const int last_bytes = (n_kb - 2 * (t.units - 1)) * kQ4TileBytes, last_scales = (t.p.n_groups - (t.units - 1) * kSums) * kQ4Tile * kEntry;
      const uint8_t* weights = reinterpret_cast<const uint8_t*>(a.W) + ((size_t)row_tile * n_kb + 2 * u) * kQ4TileBytes;
      const uint8_t* table = t.p.table + ((size_t)row_tile * t.p.n_groups + u * kSums) * kQ4Tile * kEntry;
      uint32_t par = 1;
      uint8_t* dst = sw;
      for (int i = 0; i < n_units; ++i) {
        if (!mbar_wait(&w_empty[slot], par, abort)) {
          s_abort = 1;
          break;
        }
        const bool last = u == t.units - 1;
        const int bytes = last ? last_bytes : 2 * kQ4TileBytes, scales = !ZERO ? 0 : last ? last_scales : kScaleBytes;
        mbar_expect_tx(&w_full[slot], bytes + scales);
        bulk_load(dst, weights, bytes, &w_full[slot]);
        if (ZERO) bulk_load(dst + 2 * kQ4TileBytes, table, scales, &w_full[slot]);
        weights += bytes;
        table += scales;
        ++u;
        if (last) {
          u = 0;
          if (++row_tile == t.row_tiles) row_tile = 0, weights = reinterpret_cast<const uint8_t*>(a.W), table = t.p.table;
        }
        dst += kSlotBytes;
        if (++slot == kWslots) slot = 0, par ^= 1, dst = sw;
      }
      if (*abort)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && s_abort) atomicOr(t.status, 2);
  if (warp == kMma) tmem_dealloc(tmem_slot, 512);
}

int rows_per_tile(int T) { return T <= 32 ? 32 : T <= 64 ? 64 : 128; }

template <int BN, bool ZERO, int G>
int launch_tc_as(const TcArgs& t, int grid, cudaStream_t st) {
  CUtensorMap mx;
  const int rc = make_map(&mx, t.p.a.x, t.p.a.T, t.p.a.in, t.p.a.ldx, BN, kQ4Block);
  if (rc) return rc;
  constexpr int smem = q4_smem(BN, ZERO, G);
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

int launch_q4_tc(const Q4Args& p, const Q4Work& w, cudaStream_t st) {
  TcArgs t{};
  t.p = p, t.status = w.status, t.counters = w.counters, t.parts = w.parts, t.delta = w.delta;
  const int bn = rows_per_tile(p.a.T);
  t.row_tiles = (p.a.out + kQ4Tile - 1) / kQ4Tile;
  t.token_tiles = (p.a.T + bn - 1) / bn;
  t.units = (p.n_kb + 1) / 2;
  const long long all = (long long)t.row_tiles * t.token_tiles * t.units;
  if (all > 2147483647ll) return fail(MLORA_ESIZE, "q4_linear: too many tiles");
  const int grid = q4_ctas(t.row_tiles * (long long)t.token_tiles, t.units, 1);
  return bn == 32 ? launch_tc_for<32>(t, grid, st) : bn == 64 ? launch_tc_for<64>(t, grid, st) : launch_tc_for<128>(t, grid, st);
}

}  // namespace mlora
