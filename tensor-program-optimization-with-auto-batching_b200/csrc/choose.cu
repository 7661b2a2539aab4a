// The next token of every row under the rules of its request: penalties for tokens that its text already has, biases, and a mask of
// what its grammar allows (llama_exec_graph.py:134-137 picks the largest logit on the host; the rules have no reference counterpart).
//
// A cluster of up to eight CTAs shares a row.  A CTA takes pieces of 4096 tokens of the vocabulary: it asks for the piece's logits
// first (eight a thread, in registers), then walks the row's text and counts in shared memory which of the piece's tokens occur how
// often -- a table of counts in global memory would be another 4 bytes per token and row to read, the text is a few KB that the
// row's CTAs find in L2 --, spreads the row's biases the same way, and only then touches the logits.  The best of a CTA is one
// 64-bit key (value, then lowest index), so the order in which keys meet does not matter; the cluster's first CTA collects them
// through distributed shared memory: one launch, no scratch.  Values are rounded step by step as the formula is written (no
// contraction), so that the choice at a near tie is that of plain 32-bit arithmetic.
#include "common.cuh"
#include "tc_ptx.cuh"

namespace mlora {
namespace {

constexpr int kChThreads = 512;
constexpr int kChVec = 2;                                 // float4 of logits a thread keeps
constexpr int kChPiece = kChThreads * kChVec * 4;         // tokens of a piece
constexpr int kChCluster = 8;

struct ChooseArgs {
  const float* logits;
  int64_t ld;
  int V;
  const int32_t* row_src;
  int n;
  const float *repetition, *frequency, *presence;
  const int32_t *prompt, *prompt_len;
  int64_t ld_prompt;
  const int32_t *answer, *answer_len;
  int64_t ld_answer;
  const int32_t *bias_set, *bias_start, *bias_token;
  const float* bias_value;
  int n_sets, n_bias;
  const int32_t *mask_of, *masks;
  int n_masks;
  int64_t ld_mask;
  float* out;
  int64_t ld_out;
  int32_t* tok;
};

// Larger value first, then the lower index; 0 is what no token gives.
__device__ __forceinline__ unsigned long long choice_key(float v, int i) {
  if (!(v > -INFINITY)) return 0;  // (not a number, or not allowed)
  const uint32_t b = __float_as_uint(v + 0.f);  // (-0 is 0)
  const uint32_t u = b & 0x80000000u ? ~b : b | 0x80000000u;
  return ((unsigned long long)u << 32) | (uint32_t)(0x7fffffff - i);
}

__device__ __forceinline__ unsigned long long warp_best(unsigned long long best) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
    best = k > best ? k : best;
  }
  return best;
}

// A text, whose first 4 * kChThreads tokens stay in registers (most texts, all of it): a row's pieces all look through it.
struct Text {
  const int32_t* at;
  int n, first[4];
  __device__ __forceinline__ void begin(const int32_t* text, int len) {
    at = text;
    n = len;
#pragma unroll
    for (int u = 0; u < 4; ++u) first[u] = threadIdx.x + u * kChThreads < n ? at[threadIdx.x + u * kChThreads] : -1;
  }
  // f(place) for the tokens that lie in the piece [v0, v0 + kChPiece)
  template <typename F>
  __device__ __forceinline__ void walk(int v0, F f) const {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned p = (unsigned)first[u] - (unsigned)v0;
      if (first[u] >= 0 && p < (unsigned)kChPiece) f((int)p);
    }
    for (int i = threadIdx.x + 4 * kChThreads; i < n; i += 4 * kChThreads) {
      int w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = i + u * kChThreads < n ? at[i + u * kChThreads] : -1;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned p = (unsigned)w[u] - (unsigned)v0;
        if (w[u] >= 0 && p < (unsigned)kChPiece) f((int)p);
      }
    }
  }
};

__global__ void __launch_bounds__(kChThreads) choose_tokens_kernel(ChooseArgs a) {
  __shared__ __align__(16) uint32_t s_count[kChPiece];  // low 31 bits: times in the answer; top bit: in the prompt
  __shared__ __align__(16) float s_bias[kChPiece];
  __shared__ unsigned long long s_warp[kChThreads / 32];
  __shared__ int s_best[2];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t width;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(width));
  const uint32_t rank = cluster_rank();
  const int t = blockIdx.x / width;
  const int src = a.row_src ? a.row_src[t] : t;
  const bool ruled = src >= 0 && src < a.n;  // (a row of padding: no rules)
  const float* logits = a.logits + (size_t)t * a.ld;
  float* out = a.out ? a.out + (size_t)t * a.ld_out : nullptr;
  const bool vec = a.V % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;

  const float rep = ruled && a.repetition ? a.repetition[src] : 1.f;
  const float freq = ruled && a.frequency ? a.frequency[src] : 0.f;
  const float pres = ruled && a.presence ? a.presence[src] : 0.f;
  const bool counts = ruled && (rep != 1.f || freq != 0.f || pres != 0.f);
  const int n_prompt = counts && a.prompt ? (int)min((int64_t)max(a.prompt_len[src], 0), a.ld_prompt) : 0;
  const int n_answer = counts && a.answer ? (int)min((int64_t)max(a.answer_len[src], 0), a.ld_answer) : 0;
  const int set = ruled && a.bias_set ? a.bias_set[src] : -1;
  int b0 = 0, b1 = 0;
  if (set >= 0 && set < a.n_sets) {
    b0 = max(a.bias_start[set], 0);
    b1 = min(a.bias_start[set + 1], a.n_bias);
  }
  const bool biased = b0 < b1;
  const int mk = ruled && a.mask_of ? a.mask_of[src] : -1;
  const int32_t* mask = mk >= 0 && mk < a.n_masks ? a.masks + (size_t)mk * a.ld_mask : nullptr;

  Text prompt, answer;
  prompt.begin(n_prompt ? a.prompt + (size_t)src * a.ld_prompt : nullptr, n_prompt);
  answer.begin(n_answer ? a.answer + (size_t)src * a.ld_answer : nullptr, n_answer);
  if (counts || biased) {  // (a thread clears what it has read of a piece, so this is done once)
#pragma unroll
    for (int j = 0; j < kChVec; ++j) {
      reinterpret_cast<uint4*>(s_count)[j * kChThreads + tid] = make_uint4(0u, 0u, 0u, 0u);
      reinterpret_cast<float4*>(s_bias)[j * kChThreads + tid] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
  }
  unsigned long long best = 0;
  float next[kChVec][4];
  uint32_t next_word[kChVec];
  const auto load = [&](int64_t v0) {  // a piece's logits and mask, asked for while the piece before is at work
#pragma unroll
    for (int j = 0; j < kChVec; ++j) {
      const int64_t at = v0 + (j * kChThreads + tid) * 4;
      next_word[j] = 0xfu;
      if (mask && at < a.V) next_word[j] = (uint32_t)mask[at >> 5] >> (at & 31);
      if (vec && at < a.V) {
        const float4 q = *reinterpret_cast<const float4*>(logits + at);  // (not the read-only path: `out` may be `logits`)
        next[j][0] = q.x, next[j][1] = q.y, next[j][2] = q.z, next[j][3] = q.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) next[j][e] = at < a.V - e ? logits[at + e] : 0.f;
      }
    }
  };
  const int64_t step = (int64_t)width * kChPiece;
  load((int64_t)rank * kChPiece);
  for (int64_t piece = (int64_t)rank * kChPiece; piece < a.V; piece += step) {
    const int v0 = (int)piece;
    float l[kChVec][4];
    uint32_t word[kChVec];
#pragma unroll
    for (int j = 0; j < kChVec; ++j) {
      word[j] = next_word[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) l[j][e] = next[j][e];
    }
    load(piece + step);
    if (counts || biased) {
      prompt.walk(v0, [&](int p) { atomicOr(&s_count[p], 0x80000000u); });
      answer.walk(v0, [&](int p) { atomicAdd(&s_count[p], 1u); });
      for (int i = b0 + tid; i < b1; i += kChThreads) {  // ascending tokens: equal ones are neighbours, the first one adds them up
        const int w = a.bias_token[i];
        const unsigned at = (unsigned)w - (unsigned)v0;
        if (w < 0 || at >= (unsigned)kChPiece || (i > b0 && a.bias_token[i - 1] == w)) continue;
        float sum = a.bias_value[i];
        for (int k = i + 1; k < b1 && a.bias_token[k] == w; ++k) sum += a.bias_value[k];
        s_bias[at] = sum;
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kChVec; ++j) {
      const int q4 = j * kChThreads + tid, at = v0 + q4 * 4;
      if (counts) {
        const uint4 c4 = reinterpret_cast<const uint4*>(s_count)[q4];
        const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
        if (c4.x | c4.y | c4.z | c4.w) {
          reinterpret_cast<uint4*>(s_count)[q4] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (!c[e]) continue;
            float v = l[j][e];
            v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
            const uint32_t times = c[e] & 0x7fffffffu;
            v = __fsub_rn(v, __fmul_rn(freq, (float)times));
            if (times) v = __fsub_rn(v, pres);
            l[j][e] = v;
          }
        }
      }
      if (biased) {
        const float4 b = reinterpret_cast<const float4*>(s_bias)[q4];
        reinterpret_cast<float4*>(s_bias)[q4] = make_float4(0.f, 0.f, 0.f, 0.f);
        l[j][0] = __fadd_rn(l[j][0], b.x), l[j][1] = __fadd_rn(l[j][1], b.y);
        l[j][2] = __fadd_rn(l[j][2], b.z), l[j][3] = __fadd_rn(l[j][3], b.w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!(word[j] >> e & 1u)) l[j][e] = -INFINITY;
        if (at < a.V - e) {
          const unsigned long long k = choice_key(l[j][e], at + e);
          best = k > best ? k : best;
        }
      }
      if (out && at < a.V) {
        if (vec) {
          *reinterpret_cast<float4*>(out + at) = make_float4(l[j][0], l[j][1], l[j][2], l[j][3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (at < a.V - e) out[at + e] = l[j][e];
        }
      }
    }
    if (counts || biased) __syncthreads();  // (before the next piece counts in the cleared tables)
  }
  best = warp_best(best);
  if (lane == 0) s_warp[warp] = best;
  __syncthreads();
  if (warp == 0) {
    best = warp_best(lane < kChThreads / 32 ? s_warp[lane] : 0);
    if (lane == 0) s_best[0] = (int)(uint32_t)best, s_best[1] = (int)(uint32_t)(best >> 32);
  }
  if (width > 1) {
    cluster_sync();
    if (rank == 0 && warp == 0) {
      best = 0;
      if (lane < (int)width)
        best = (unsigned long long)(uint32_t)ld_cluster(&s_best[1], lane) << 32 | (uint32_t)ld_cluster(&s_best[0], lane);
      best = warp_best(best);
    }
    cluster_sync();  // nobody leaves while its best is being read
  }
  if (rank == 0 && tid == 0) a.tok[t] = best ? 0x7fffffff - (int)(uint32_t)best : -1;
}

}  // namespace
}  // namespace mlora

using namespace mlora;

extern "C" int mlora_choose_tokens(const float* d_logits, int64_t ld, int32_t T, int32_t V, const int32_t* d_row_src, int32_t n,
                                   const float* d_repetition, const float* d_frequency, const float* d_presence, const int32_t* d_prompt,
                                   const int32_t* d_prompt_len, int64_t ld_prompt, const int32_t* d_answer, const int32_t* d_answer_len,
                                   int64_t ld_answer, const int32_t* d_bias_set, const int32_t* d_bias_start, const int32_t* d_bias_token,
                                   const float* d_bias_value, int32_t n_sets, int32_t n_bias, const int32_t* d_mask_of, const int32_t* d_masks,
                                   int32_t n_masks, int64_t ld_mask, float* d_logits_out, int64_t ld_out, int32_t* d_tok, void* stream) {
  MLORA_REQUIRE(T >= 0 && V > 0 && V < 2147483647 - kChCluster * kChPiece && ld >= V && n >= 0, "choose_tokens: bad sizes T=%d V=%d ld=%lld n=%d",
                T, V, (long long)ld, n);
  MLORA_REQUIRE(d_logits && d_tok, "choose_tokens: null pointer");
  MLORA_REQUIRE(!d_prompt || (d_prompt_len && ld_prompt > 0 && ld_prompt < (1ll << 30)), "choose_tokens: prompts need their lengths");
  MLORA_REQUIRE(!d_answer || (d_answer_len && ld_answer > 0 && ld_answer < (1ll << 30)), "choose_tokens: answers need their lengths");
  MLORA_REQUIRE(!d_bias_set || (n_sets > 0 && n_bias >= 0 && d_bias_start && (n_bias == 0 || (d_bias_token && d_bias_value))),
                "choose_tokens: incomplete bias sets");
  MLORA_REQUIRE(!d_mask_of || (n_masks > 0 && d_masks && ld_mask >= (V + 31ll) / 32), "choose_tokens: incomplete masks");
  MLORA_REQUIRE(!d_logits_out || ld_out >= V, "choose_tokens: the kept logits' rows are too short");
  if (T == 0) return MLORA_OK;
  ChooseArgs a{d_logits, ld, V, d_row_src, n, d_repetition, d_frequency, d_presence, d_prompt, d_prompt_len, ld_prompt, d_answer,
               d_answer_len, ld_answer, d_bias_set, d_bias_start, d_bias_token, d_bias_value, n_sets, n_bias, d_mask_of, d_masks, n_masks,
               ld_mask, d_logits_out, ld_out, d_tok};
  const int pieces = (V + kChPiece - 1) / kChPiece;
  int width = 1;
  while (width < kChCluster && width < pieces) width *= 2;
  MLORA_REQUIRE((long long)T * width <= 2147483647ll, "choose_tokens: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(T * width));
  cfg.blockDim = dim3(kChThreads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)width;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, choose_tokens_kernel, a);
  if (e != cudaSuccess) return fail(MLORA_ECUDA, "choose_tokens_kernel: %s", cudaGetErrorString(e));
  count_launch();
  MLORA_CHECK_LAUNCH("choose_tokens_kernel");
  return MLORA_OK;
}
