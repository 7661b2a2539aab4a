// 4-bit weights with group scales: the packed layout, and what its kernels share.
//
//   W[o, k] = (q[o, k] - z[o, k / G]) s[o, k / G],  q and z in 0..15 (z = 8 where there are none), s bf16, G = 32, 64 or 128
//
// q in tiles of 128 outputs x 64 inputs, [out / 128][in / 64][8 parts of 16 outputs][32 lanes][4 words]: word j of a lane holds what that
// lane has of the 16 x 16 A operand of mma.m16n8k16 for the inputs 16 j .. 16 j + 15 -- register i (outputs lane / 4 and + 8, inputs
// 2 (lane % 4) and + 8) has its two weights in bits 4 i and 16 + 4 i, so that one shift and one mask give a register --, which is also
// what a lane of tcgen05.st.16x128b stores.  Behind them the scales, [out / 128][in / G][128]: bf16 s, or with zero points the pair
// (bf16 s, bf16 128 + z).  Outputs and inputs beyond the matrix are zeros.
//
// A nibble under the exponent of 128 is the bf16 number 128 + q, and 128 + q - (128 + z) is exact: the products are taken with the
// integers q - z, a group's sum in fp32 is multiplied by s, and no weight is ever rounded.
#pragma once
#include "linear.cuh"

namespace mlora {

constexpr int kQ4Tile = 128, kQ4Block = 64, kQ4TileBytes = kQ4Tile * kQ4Block / 2;  // outputs, inputs and bytes of a tile

struct Q4Args {
  LinearArgs a;            // x, y, sizes, adapters, flags; W: the packed weights
  const uint8_t* table;    // scales
  int group, n_groups, n_kb, packed_b;
};

__host__ __device__ inline long long q4_weight_bytes(int out, int in) {
  return (long long)((out + kQ4Tile - 1) / kQ4Tile) * ((in + kQ4Block - 1) / kQ4Block) * kQ4TileBytes;
}

__device__ __forceinline__ uint32_t q4_sub(uint32_t v, uint32_t z) {  // two bf16
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(z));
  return r;
}
// The four registers of a word; z0, z1: twice 128 + z of the lane's two outputs.
__device__ __forceinline__ void q4_expand(uint32_t w, uint32_t z0, uint32_t z1, uint32_t (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(v) : "r"(w >> (4 * i)));  // (w & a) | b
    r[i] = q4_sub(v, i & 1 ? z1 : z0);
  }
}
constexpr uint32_t kQ4Middle = 0x43084308u;  // 128 + 8, twice

// sum_j u[j] B[slot][o][j] of one output and row, B row-major or in the tiles of mlora_pack_lora_b
__device__ __forceinline__ const uint4* q4_b_row(const LinearArgs& a, int packed, int slot, int o, int j8, int& swizzle) {
  if (!packed) {
    swizzle = 0;
    return reinterpret_cast<const uint4*>(a.B_all + ((size_t)slot * a.out + o) * a.r_max) + j8;
  }
  const int sub = a.r_max < 64 ? a.r_max : 64, n_sub = a.r_max / sub, chunks = sub / 8, r = o & 127, row_tiles = (a.out + 127) / 128;
  swizzle = chunks == 8 ? (r & 7) : chunks == 4 ? ((r >> 1) & 3) : ((r >> 2) & 1);
  return reinterpret_cast<const uint4*>(a.B_all) + (((size_t)slot * row_tiles + (o >> 7)) * n_sub + j8 / chunks) * (128 * chunks) +
         (size_t)r * chunks + ((j8 % chunks) ^ swizzle);
}
__device__ __forceinline__ float dot8(const uint4& v, const float* u) {
  float b[8], s = 0.f;
  unpack8(v, b);
  const float4 u0 = *reinterpret_cast<const float4*>(u), u1 = *reinterpret_cast<const float4*>(u + 4);
  s = fmaf(b[0], u0.x, s), s = fmaf(b[1], u0.y, s), s = fmaf(b[2], u0.z, s), s = fmaf(b[3], u0.w, s);
  s = fmaf(b[4], u1.x, s), s = fmaf(b[5], u1.y, s), s = fmaf(b[6], u1.z, s), s = fmaf(b[7], u1.w, s);
  return s;
}
__device__ __forceinline__ float q4_adapter(const LinearArgs& a, int packed, int t, int o) {
  if (a.u == nullptr) return 0.f;
  const int s = a.slots[t];
  if (s < 0 || s >= a.n_adapters) return 0.f;
  const float* u = a.u + (size_t)t * (a.r_max * a.n_mod) + module_of(a, o) * a.r_max;
  float sum = 0.f;
  for (int j = 0; j < a.r_max / 8; ++j) {
    int sw;
    sum += dot8(ld_cached(q4_b_row(a, packed, s, o, j, sw)), u + 8 * j);
  }
  return a.scales[s] * sum;
}

// Scratch of a projection: the status word (and the caller's bytes), a counter and a share of 128 x 128 sums per CTA, and the adapters'
// share of a slice of rows.
constexpr int kQ4MaxCtas = 512, kQ4Header = 256, kQ4Slice = 512;
struct Q4Work {
  int32_t* status;
  int32_t* counters;   // [CTA that a tile begins in]: shares of the tile that have arrived, zero between calls
  float* parts;        // [CTA][128 x 128]: sums of a CTA's share of a tile that another CTA begins
  const float* delta;  // [rows][out]: the adapters' share, or NULL
};
size_t q4_workspace(int T, int out);
int q4_ctas(long long tiles, int units, int per_sm);  // CTAs of a persistent launch over tiles of so many units
int launch_q4_expand(const Q4Args& p, float* delta, cudaStream_t st);
int launch_q4_mm(const Q4Args& p, const Q4Work& w, cudaStream_t st);
int launch_q4_tc(const Q4Args& p, const Q4Work& w, cudaStream_t st);
constexpr int kQ4InlineRows = 8;  // rows whose adapters launch_q4_mm expands itself
constexpr int kQ4SmallRows = 16;  // rows that launch_q4_mm is for

__device__ __noinline__ static float q4_act(float v, int act) { return act_one(v, act); }  // (one copy of erf, not one per value)

// Which CTAs of `ctas` share the units [begin, begin + n) of `all`, dealt out in equal ranges.
__device__ __forceinline__ int q4_cta_of(long long unit, long long all, int ctas) {
  int k = (int)(unit * ctas / all);
  while (all * (k + 1) / ctas <= unit) ++k;
  while (all * k / ctas > unit) --k;
  return k;
}

}  // namespace mlora
