// 4-bit weights: quantising, packing, and the entry point of their projections (see q4.cuh for the layout).
#include "q4.cuh"

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
  const int z = zero ? min(max(__float2int_rn(isinf(inv) ? -lo / s : -lo * inv), 0), 15) : 8;
  for (int i = lane; i < G; i += 32) {
    const float v = __bfloat162float(W[at + i]);
    q[at + i] = (uint8_t)min(max(__float2int_rn(isinf(inv) ? v / s : v * inv) + z, 0), 15);  // (scales below 2^-128 have no reciprocal)
  }
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

// delta[t, o] = scale[slot] sum_j u[t, j] B[slot][o][j]: a thread per output, eight rows at a time; rows that follow each other with the
// same adapter read its row once (up to 64 ranks wide).
constexpr int kExThreads = 128, kExRows = 8, kExMaxU = 512;

__global__ void __launch_bounds__(kExThreads) q4_expand_kernel(Q4Args p, float* __restrict__ delta) {
  __shared__ __align__(16) float su[kExRows][kExMaxU];
  __shared__ int s_slot[kExRows];
  pdl_launch_dependents();
  pdl_wait();
  const LinearArgs& a = p.a;
  const int o = blockIdx.x * kExThreads + threadIdx.x, t0 = blockIdx.y * kExRows, rows = min(kExRows, a.T - t0), width = a.r_max * a.n_mod;
  if (threadIdx.x < kExRows) s_slot[threadIdx.x] = (int)threadIdx.x < rows ? a.slots[t0 + threadIdx.x] : -1;
  const bool fits = width <= kExMaxU;
  for (int i = threadIdx.x; fits && i < rows * width; i += kExThreads) su[i / width][i % width] = a.u[(size_t)t0 * width + i];
  __syncthreads();
  if (o >= a.out) return;
  const int module = module_of(a, o) * a.r_max, n8 = a.r_max / 8;
  uint4 b[8];
  int have = -1, sw;
  float alpha = 0.f;
#pragma unroll 1
  for (int r = 0; r < rows; ++r) {
    const int s = s_slot[r];
    float sum = 0.f;
    if (s >= 0 && s < a.n_adapters) {
      const float* u = fits ? &su[r][module] : a.u + (size_t)(t0 + r) * width + module;
      if (s != have) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n8) b[j] = ld_cached(q4_b_row(a, p.packed_b, s, o, j, sw));
        alpha = a.scales[s];
        have = s;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n8) sum += dot8(b[j], u + 8 * j);
      for (int j = 8; j < n8; ++j) sum += dot8(ld_cached(q4_b_row(a, p.packed_b, s, o, j, sw)), u + 8 * j);
      sum *= alpha;
    }
    delta[(size_t)(t0 + r) * a.out + o] = sum;
  }
}

}  // namespace

int launch_q4_expand(const Q4Args& p, float* delta, cudaStream_t st) {
  const dim3 grid((unsigned)((p.a.out + kExThreads - 1) / kExThreads), (unsigned)((p.a.T + kExRows - 1) / kExRows));
  q4_expand_kernel<<<grid, kExThreads, 0, st>>>(p, delta);
  count_launch();
  MLORA_CHECK_LAUNCH("q4_expand_kernel");
  return MLORA_OK;
}

static int q4_most_ctas(int per_sm) {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = 148;
  }
  n *= per_sm;
  return n < kQ4MaxCtas ? n : kQ4MaxCtas;
}

// `per_sm` per SM at most.  Where nearly all of them can have equal shares of one tile each (a 4096-wide output: four CTAs a tile, 128 of
// 148), they do: one sum to leave or to collect per CTA instead of two.
int q4_ctas(long long tiles, int units, int per_sm) {
  const int n = q4_most_ctas(per_sm);
  if (tiles <= n) {
    const int per = n / (int)tiles < units ? n / (int)tiles : units;
    if (tiles * per >= n * 85 / 100 || per == units) return (int)tiles * per;
  }
  return (int)(tiles * units < n ? tiles * units : n);
}

// Counters and shares lie at places that no call's sizes move; behind them the adapters' share of a slice of rows.
size_t q4_workspace(int T, int out) {
  return kQ4Header + kQ4MaxCtas * 4 + (size_t)q4_most_ctas(2) * 128 * kQ4Tile * 4 + (size_t)(T < kQ4Slice ? T : kQ4Slice) * out * 4;
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
  return T <= 0 || in <= 0 || out <= 0 ? 0 : q4_workspace(T, out);
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
  const size_t need = q4_workspace(T, out);
  if (!d_work || work_bytes < need) return fail(MLORA_ESIZE, "q4_linear: scratch of %zu bytes needed, %zu given", need, work_bytes);
  MLORA_REQUIRE(aligned16(d_work), "q4_linear: the scratch must be 16-byte aligned");
  Q4Work w{(int32_t*)d_work, (int32_t*)((uint8_t*)d_work + kQ4Header), (float*)((uint8_t*)d_work + kQ4Header + kQ4MaxCtas * 4), nullptr};
  float* delta = (float*)((uint8_t*)d_work + q4_workspace(0, 0));
  const cudaStream_t st = (cudaStream_t)stream;
  const int slice = lora ? kQ4Slice : T;
  for (int t0 = 0; t0 < T; t0 += slice) {
    Q4Args s = p;
    s.a.T = T - t0 < slice ? T - t0 : slice;
    s.a.x += (size_t)t0 * ldx;
    s.a.y = (uint8_t*)d_y + (size_t)t0 * ldy * (flags & MLORA_OUT_F32 ? 4 : 2);
    if (lora) {
      s.a.u += (size_t)t0 * a.r_max * a.n_mod;
      s.a.slots += t0;
      if (s.a.T > kQ4InlineRows) {  // (fewer rows: where the sums are written)
        w.delta = delta;
        const int rc = launch_q4_expand(s, delta, st);
        if (rc) return rc;
      } else {
        w.delta = nullptr;
      }
    }
    const int rc = s.a.T <= kQ4SmallRows ? launch_q4_mm(s, w, st) : launch_q4_tc(s, w, st);
    if (rc) return rc;
  }
  return MLORA_OK;
}
