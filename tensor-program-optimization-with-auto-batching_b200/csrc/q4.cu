// 4-bit weights: quantising, packing, and the projection kernel of the smallest batches (see q4.cuh for the layout).
//
// Up to 16 rows: y = x W^T is bound by the weights' out in / 2 bytes.  A CTA owns 16 U outputs; its eight warps take the blocks of 64
// inputs in turn, each with a ring of asynchronous copies of its own (weights, the rows of x, scales), multiply with mma.m16n8k16 --
// weights as the 16-row operand, up to 8 or 16 rows of x as the 8-column one: at these sizes the legacy tensor path is a tenth busy, and
// unlike a tcgen05 tile it needs neither 128 outputs per CTA nor a trip of the weights through TMEM -- and are added up at the end.
#include "q4.cuh"
#include "tc_ptx.cuh"

#include <atomic>

namespace mlora {
namespace {

// ---- load time --------------------------------------------------------------------------------------------------------------------
__global__ void q4_quantize_kernel(const bf16* __restrict__ W, int out, int in, int G, uint8_t* __restrict__ q, bf16* __restrict__ scale,
                                   uint8_t* __restrict__ zero) {
  const long long w = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);  // a warp per output and group
  const int lane = threadIdx.x & 31, groups = in / G;
  if (w >= (long long)out * groups) return;
  const size_t at = (size_t)(w / groups) * in + (size_t)(w % groups) * G;
  float lo = 0.f, hi = 0.f;
  for (int i = lane; i < G; i += 32) {
    const float v = __bfloat162float(W[at + i]);
    lo = fminf(lo, v), hi = fmaxf(hi, v);
  }
  lo = -warp_max(-lo), hi = warp_max(hi);
  // with zero points the 16 values span [lo, hi], else -7 .. 7 spans the larger side
  const bf16 sb = __float2bfloat16_rn(zero ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f);
  const float s = __bfloat162float(sb), inv = s > 0.f ? 1.f / s : 0.f;
  const int z = zero ? min(max(__float2int_rn(-lo * inv), 0), 15) : 8;
  for (int i = lane; i < G; i += 32) q[at + i] = (uint8_t)min(max(__float2int_rn(__bfloat162float(W[at + i]) * inv) + z, 0), 15);
  if (lane == 0) {
    scale[w] = sb;
    if (zero) zero[w] = (uint8_t)z;
  }
}

__global__ void q4_pack_kernel(const uint8_t* __restrict__ q, int out, int in, uint32_t* __restrict__ packed, long long words) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= words) return;
  const int j = i & 3, lane = (i >> 2) & 31, part = (i >> 7) & 7, n_kb = (in + kQ4Block - 1) / kQ4Block;
  const long long tile = i >> 10;
  const int kb = (int)(tile % n_kb);
  const long long o0 = tile / n_kb * kQ4Tile + part * 16 + (lane >> 2);
  const int k0 = kb * kQ4Block + j * 16 + (lane & 3) * 2;
  uint32_t w = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const long long o = o0 + (r & 1) * 8;
      const int k = k0 + (r >> 1) * 8 + e;
      if (o < out && k < in) w |= (uint32_t)(q[(size_t)o * in + k] & 15) << (4 * r + 16 * e);
    }
  packed[i] = w;
}

__global__ void q4_table_kernel(const bf16* __restrict__ scale, const uint8_t* __restrict__ zero, int out, int groups, uint8_t* __restrict__ table,
                                long long n) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const long long o = i / (kQ4Tile * (long long)groups) * kQ4Tile + i % kQ4Tile;
  const int g = (int)(i / kQ4Tile % groups);
  const bool in_range = o < out;
  const bf16 s = in_range ? scale[(size_t)o * groups + g] : __float2bfloat16_rn(0.f);
  if (!zero) {
    reinterpret_cast<bf16*>(table)[i] = s;
    return;
  }
  const bf16 z = __float2bfloat16_rn(128.f + (in_range ? (float)(zero[(size_t)o * groups + g] & 15) : 0.f));
  reinterpret_cast<__nv_bfloat162*>(table)[i] = __nv_bfloat162(s, z);
}

// ---- up to 16 rows ----------------------------------------------------------------------------------------------------------------
constexpr int kQrWarps = 8, kQrThreads = kQrWarps * 32;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {  // the rest of the 16 becomes zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// U: parts of 16 outputs of a CTA; N8: rows of x in eights; ZERO: zero points; SUB: groups of 32 (two in a block)
template <int U, int N8, bool ZERO, bool SUB>
struct Q4Ring {
  static constexpr int kScaleBytes = ZERO ? 4 : 2, kSubs = SUB ? 2 : 1;
  static constexpr int kX = U * 512, kS = kX + N8 * 1024, kStage = kS + kSubs * U * 16 * kScaleBytes;
  static constexpr int kStages = U * N8 >= 4 ? 6 : 8;
  static constexpr int kBytes = kQrWarps * kStages * kStage;
  static_assert(kBytes >= kQrWarps * U * 16 * N8 * 8 * 4, "the warps' sums lie in the ring");
};

template <int U, int N8, bool ZERO, bool SUB>
__global__ void __launch_bounds__(kQrThreads) q4_rows_kernel(Q4Args p) {
  using R = Q4Ring<U, N8, ZERO, SUB>;
  constexpr int kStages = R::kStages;
  extern __shared__ __align__(128) uint8_t ring[];
  pdl_launch_dependents();
  const LinearArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = blockIdx.x / (8 / U), part0 = blockIdx.x % (8 / U) * U;
  const uint8_t* weights = reinterpret_cast<const uint8_t*>(a.W) + (size_t)tile * p.n_kb * kQ4TileBytes + part0 * 512 + lane * 16;
  const uint8_t* scales = p.table + ((size_t)tile * p.n_groups * kQ4Tile + part0 * 16) * R::kScaleBytes;
  const uint32_t base = smem_u32(ring) + warp * kStages * R::kStage;
  pdl_wait();  // (before the first asynchronous copy of x)
  auto fetch = [&](int i) {
    const int kb = warp + i * kQrWarps;
    if (kb < p.n_kb) {
      const uint32_t st = base + (i % kStages) * R::kStage;
#pragma unroll
      for (int u = 0; u < U; ++u) cp16(st + u * 512 + lane * 16, weights + (size_t)kb * kQ4TileBytes + u * 512, 16);
#pragma unroll
      for (int c = 0; c < 2 * N8; ++c) {  // rows of 128 bytes, 16-byte pieces XORed with the row
        const int t = c * 4 + (lane >> 3), ch = lane & 7, k = kb * kQ4Block + ch * 8;
        const bool in_range = t < a.T && k < a.in;
        cp16(st + R::kX + t * 128 + ((ch ^ (t & 7)) << 4), in_range ? a.x + (size_t)t * a.ldx + k : a.x, in_range ? 16 : 0);
      }
      constexpr int per = U * R::kScaleBytes;  // 16-byte pieces of a group's scales: U * 16 of them
      if (lane < R::kSubs * per) {
        const int g = min(SUB ? 2 * kb + lane / per : kb * kQ4Block / p.group, p.n_groups - 1);
        cp16(st + R::kS + lane * 16, scales + (size_t)g * (kQ4Tile * R::kScaleBytes) + lane % per * 16, 16);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  float acc[U][N8][4];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int n = 0; n < N8; ++n) acc[u][n][0] = acc[u][n][1] = acc[u][n][2] = acc[u][n][3] = 0.f;
  const int g = lane >> 2;
  for (int i = 0; warp + i * kQrWarps < p.n_kb; ++i) {
    fetch(i + kStages - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const uint32_t st = base + (i % kStages) * R::kStage;
    const uint8_t* sp = ring + (st - smem_u32(ring));
    uint32_t b[N8][2][4];  // rows 8 n .. of x: inputs 32 h .. 32 h + 31
#pragma unroll
    for (int n = 0; n < N8; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) ldmatrix4(st + R::kX + n * 1024 + (lane & 7) * 128 + (((h * 4 + (lane >> 3)) ^ (lane & 7)) << 4), b[n][h]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint4 w4 = *reinterpret_cast<const uint4*>(sp + u * 512 + lane * 16);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
      float sum[N8][4];
      float s0 = 0.f, s1 = 0.f;
      uint32_t z0 = kQ4Middle, z1 = kQ4Middle;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j == 0 || (SUB && j == 2)) {  // a group begins
          const uint8_t* e = sp + R::kS + ((SUB ? j / 2 : 0) * U * 16 + u * 16 + g) * R::kScaleBytes;
          if constexpr (ZERO) {
            const uint32_t e0 = *reinterpret_cast<const uint32_t*>(e), e1 = *reinterpret_cast<const uint32_t*>(e + 8 * 4);
            s0 = __uint_as_float(e0 << 16), s1 = __uint_as_float(e1 << 16);
            z0 = __byte_perm(e0, e0, 0x3232), z1 = __byte_perm(e1, e1, 0x3232);
          } else {
            s0 = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(e) << 16);
            s1 = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(e + 8 * 2) << 16);
          }
#pragma unroll
          for (int n = 0; n < N8; ++n) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
        }
        uint32_t r[4];
        q4_expand(w[j], z0, z1, r);
#pragma unroll
        for (int n = 0; n < N8; ++n) mma_bf16(sum[n], r, b[n][j >> 1][(j & 1) * 2], b[n][j >> 1][(j & 1) * 2 + 1]);
        if (j == 3 || (SUB && j == 1)) {
#pragma unroll
          for (int n = 0; n < N8; ++n) {
            acc[u][n][0] = fmaf(s0, sum[n][0], acc[u][n][0]), acc[u][n][1] = fmaf(s0, sum[n][1], acc[u][n][1]);
            acc[u][n][2] = fmaf(s1, sum[n][2], acc[u][n][2]), acc[u][n][3] = fmaf(s1, sum[n][3], acc[u][n][3]);
          }
        }
      }
    }
    __syncwarp();  // (the next copy overwrites what was read here)
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // ---- the warps' sums: [warp][row of x][16 U outputs] -----------------------------------------------------------------------------
  constexpr int kO = U * 16, kN = N8 * 8;
  float* part = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int n = 0; n < N8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        part[(warp * kN + n * 8 + (lane & 3) * 2 + (e & 1)) * kO + u * 16 + g + (e >> 1) * 8] = acc[u][n][e];
  __syncthreads();
  const int o0 = tile * kQ4Tile + part0 * 16;
  const auto total = [&](int t, int c) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kQrWarps; ++w) s += part[(w * kN + t) * kO + c];
    return o0 + c < a.out ? s + q4_adapter(a, p.packed_b, t, o0 + c) : 0.f;
  };
  if (a.flags & MLORA_SILU_MUL) {
    for (int i = tid; i < a.T * (kO / 2); i += kQrThreads) {
      const int t = i / (kO / 2), c = i % (kO / 2), at = (c >> 3) * 16 + (c & 7);  // (8 gate outputs, then their 8 up outputs)
      if (o0 + at < a.out) store_out(a, t, o0 / 2 + c, silu_mul(total(t, at), total(t, at + 8)));
    }
  } else {
    const int act = a.flags & (MLORA_ACT_RELU2 | MLORA_ACT_GELU);
    for (int i = tid; i < a.T * kO; i += kQrThreads) {
      const int t = i / kO, c = i % kO;
      if (o0 + c < a.out) store_out(a, t, o0 + c, act_one(total(t, c), act));
    }
  }
}

template <int U, int N8, bool ZERO, bool SUB>
int launch_rows_as(const Q4Args& p, cudaStream_t st) {
  using R = Q4Ring<U, N8, ZERO, SUB>;
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!((done.load(std::memory_order_acquire) >> (dev & 63)) & 1ull)) {
    const cudaError_t e = cudaFuncSetAttribute(q4_rows_kernel<U, N8, ZERO, SUB>, cudaFuncAttributeMaxDynamicSharedMemorySize, R::kBytes);
    if (e != cudaSuccess) return fail(MLORA_ECUDA, "q4_linear: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done.fetch_or(1ull << (dev & 63), std::memory_order_release);
  }
  const unsigned grid = (unsigned)((p.a.out + 16 * U - 1) / (16 * U));
  const cudaError_t e = launch_pdl_if(pdl_enabled_gemm(), q4_rows_kernel<U, N8, ZERO, SUB>, dim3(grid), dim3(kQrThreads), R::kBytes, st, p);
  if (e != cudaSuccess) return fail(MLORA_ECUDA, "q4_rows_kernel: %s", cudaGetErrorString(e));
  count_launch();
  MLORA_CHECK_LAUNCH("q4_rows_kernel");
  return MLORA_OK;
}
template <int U, int N8>
int launch_rows_for(const Q4Args& p, bool zero, cudaStream_t st) {
  if (p.group == 32) return zero ? launch_rows_as<U, N8, true, true>(p, st) : launch_rows_as<U, N8, false, true>(p, st);
  return zero ? launch_rows_as<U, N8, true, false>(p, st) : launch_rows_as<U, N8, false, false>(p, st);
}

}  // namespace

int launch_q4_rows(const Q4Args& p, cudaStream_t st) {
  const bool zero = (p.a.flags & MLORA_Q4_ZEROS) != 0;
  // More outputs per CTA read the rows of x fewer times, as long as there are a few CTAs for every SM.
  const int parts = (p.a.out + 15) / 16;
  if (p.a.T <= 8) return parts >= 4 * 4 * 148 ? launch_rows_for<4, 1>(p, zero, st) : parts >= 2 * 4 * 148 ? launch_rows_for<2, 1>(p, zero, st) : launch_rows_for<1, 1>(p, zero, st);
  return parts >= 4 * 2 * 148 ? launch_rows_for<4, 2>(p, zero, st) : parts >= 2 * 2 * 148 ? launch_rows_for<2, 2>(p, zero, st) : launch_rows_for<1, 2>(p, zero, st);
}

}  // namespace mlora

using namespace mlora;

namespace {
bool q4_sizes(int out, int in, int group) {
  return out > 0 && in > 0 && (group == 32 || group == 64 || group == 128) && in % group == 0 && in <= (1 << 24) && out <= (1 << 28);
}
}  // namespace

extern "C" size_t mlora_q4_bytes(int32_t out, int32_t in, int32_t group, int32_t zeros) {
  if (!q4_sizes(out, in, group)) return 0;
  return (size_t)q4_weight_bytes(out, in) + (size_t)((out + kQ4Tile - 1) / kQ4Tile) * kQ4Tile * (in / group) * (zeros ? 4 : 2);
}

extern "C" int mlora_q4_quantize(const void* d_W, int32_t out, int32_t in, int32_t group, void* d_q, void* d_scale, void* d_zero, void* stream) {
  MLORA_REQUIRE(q4_sizes(out, in, group), "q4_quantize: groups of 32, 64 or 128 that divide the inputs (got %d of %d)", group, in);
  MLORA_REQUIRE(d_W && d_q && d_scale, "q4_quantize: null pointer");
  const long long warps = (long long)out * (in / group);
  MLORA_REQUIRE((warps + 7) / 8 <= 2147483647ll, "q4_quantize: too many groups");
  q4_quantize_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, (cudaStream_t)stream>>>((const bf16*)d_W, out, in, group, (uint8_t*)d_q, (bf16*)d_scale,
                                                                                  (uint8_t*)d_zero);
  count_launch();
  MLORA_CHECK_LAUNCH("q4_quantize_kernel");
  return MLORA_OK;
}

extern "C" int mlora_q4_pack(const void* d_q, const void* d_scale, const void* d_zero, int32_t out, int32_t in, int32_t group, void* d_Wq, void* stream) {
  MLORA_REQUIRE(q4_sizes(out, in, group), "q4_pack: groups of 32, 64 or 128 that divide the inputs (got %d of %d)", group, in);
  MLORA_REQUIRE(d_q && d_scale && d_Wq && aligned16(d_Wq), "q4_pack: null pointer or unaligned weights");
  const long long words = q4_weight_bytes(out, in) / 4, n = (long long)((out + kQ4Tile - 1) / kQ4Tile) * kQ4Tile * (in / group);
  MLORA_REQUIRE((words + 255) / 256 <= 2147483647ll && (n + 255) / 256 <= 2147483647ll, "q4_pack: too many weights");
  q4_pack_kernel<<<(unsigned)((words + 255) / 256), 256, 0, (cudaStream_t)stream>>>((const uint8_t*)d_q, out, in, (uint32_t*)d_Wq, words);
  count_launch();
  MLORA_CHECK_LAUNCH("q4_pack_kernel");
  q4_table_kernel<<<(unsigned)((n + 255) / 256), 256, 0, (cudaStream_t)stream>>>((const bf16*)d_scale, (const uint8_t*)d_zero, out, in / group,
                                                                                 (uint8_t*)d_Wq + words * 4, n);
  count_launch();
  MLORA_CHECK_LAUNCH("q4_table_kernel");
  return MLORA_OK;
}

extern "C" size_t mlora_q4_linear_workspace(int32_t T, int32_t in, int32_t out) {
  return T <= 0 || in <= 0 || out <= 0 || T <= kQ4RowsMost ? 0 : q4_tc_workspace(T, in, out);
}

extern "C" int mlora_q4_linear(const void* d_x, int64_t ldx, const void* d_Wq, int32_t group, void* d_y, int64_t ldy, int32_t T, int32_t in,
                               int32_t out, const float* d_u, const void* d_B_all, const float* d_scales, const int32_t* d_slots,
                               int32_t n_adapters, int32_t r_max, int32_t n_mod, const int32_t* h_mod_offsets, int32_t flags, void* d_work,
                               size_t work_bytes, void* stream) {
  MLORA_REQUIRE(T >= 0 && q4_sizes(out, in, group), "q4_linear: groups of 32, 64 or 128 that divide the inputs (got %d of %d, %d rows)", group, in, T);
  const bool silu = (flags & MLORA_SILU_MUL) != 0, lora = d_u != nullptr;
  MLORA_REQUIRE(ldx >= in && ldy >= (silu ? out / 2 : out) && (!silu || out % 16 == 0), "q4_linear: row pitches too small, or gate|up rows not in sixteens");
  MLORA_REQUIRE(!(flags & (MLORA_ACT_RELU2 | MLORA_ACT_GELU)) || (!silu && !lora), "q4_linear: relu^2 and gelu go with plain projections");
  MLORA_REQUIRE(!lora || (d_B_all && d_scales && d_slots && n_adapters > 0 && r_max > 0 && r_max % 8 == 0 && n_mod >= 1 && n_mod <= 8 && (n_mod == 1 || silu || h_mod_offsets)),
                "q4_linear: incomplete adapters (rank pitch %d, %d modules)", r_max, n_mod);
  MLORA_REQUIRE(!lora || !(flags & MLORA_B_SPLIT), "q4_linear: the rank-compact adapter layout is not read here");
  MLORA_REQUIRE(!lora || !silu || n_mod == 2, "q4_linear: gate|up adapters are two modules");
  if (T == 0) return MLORA_OK;
  MLORA_REQUIRE(d_x && d_Wq && d_y, "q4_linear: null pointer");
  MLORA_REQUIRE(aligned16(d_x) && ldx % 8 == 0 && aligned16(d_Wq) && (!lora || (aligned16(d_u) && aligned16(d_B_all))), "q4_linear: 16-byte alignment");
  Q4Args p{};
  LinearArgs& a = p.a;
  a.x = (const bf16*)d_x, a.ldx = ldx, a.W = (const bf16*)d_Wq, a.y = d_y, a.ldy = ldy, a.T = T, a.in = in, a.out = out, a.flags = flags;
  a.r_max = 8, a.n_mod = 1;
  if (lora) {
    a.u = d_u, a.B_all = (const bf16*)d_B_all, a.scales = d_scales, a.slots = d_slots, a.n_adapters = n_adapters;
    a.r_max = silu ? 2 * r_max : r_max;  // (interleaved gate / up rows: one operand over both modules' ranks)
    a.n_mod = silu ? 1 : n_mod;
    if ((flags & MLORA_B_PACKED) && !(a.r_max == 16 || a.r_max == 32 || a.r_max % 64 == 0))
      return fail(MLORA_EINVAL, "q4_linear: tiled adapters have rank pitches of 16, 32 or 64s (got %d)", a.r_max);
    for (int m = 0; m <= a.n_mod; ++m) a.mod_off[m] = a.n_mod > 1 ? h_mod_offsets[m] : m * out;
  }
  p.group = group, p.n_groups = in / group, p.n_kb = (in + kQ4Block - 1) / kQ4Block, p.packed_b = (flags & MLORA_B_PACKED) != 0;
  p.table = (const uint8_t*)d_Wq + q4_weight_bytes(out, in);
  if (T <= kQ4RowsMost) return launch_q4_rows(p, (cudaStream_t)stream);
  return launch_q4_tc(p, d_work, work_bytes, (cudaStream_t)stream);
}
