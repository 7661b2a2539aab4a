// The next token of every row under the rules of its request: penalties for tokens that its text already has, biases, and a mask of
// what its grammar allows (llama_exec_graph.py:134-137 picks the largest logit on the host; the rules have no reference counterpart).
//
// A cluster of up to eight CTAs shares a row.  A CTA takes pieces of 4096 tokens of the vocabulary: it asks for the piece's logits (eight
// a thread, in registers; three CTAs on an SM have 48 KB on their way), then it looks through the row's text and counts in shared memory
// which of the piece's tokens occur how often -- a table of counts in global memory would be another 4 bytes per token and row to read,
// the text is a few KB that stays in registers --, marks the tokens that have a bias (which stay in registers too) and only then
// touches the logits.  The best of a thread is kept as it goes, a later one only if it is larger, so the lowest index
// wins; between threads a 64-bit key of value and index decides, in any order, and the cluster's first CTA collects the CTAs' keys
// through distributed shared memory: one launch, no scratch.  Values are rounded step by step as the formula is written (no
// contraction), so that the choice at a near tie is that of plain 32-bit arithmetic.
// Measured (CUDA graph): one row of 32000 4.6 us, 32 rows 7.5, 256 rows of 128000 with the logits kept 92 us (a copy 42): what the rules
// cost there is looking through the texts once per piece, and its barrier.  Two tables in turn save the other barrier of a piece (104 us
// without); the next piece's logits on their way cost a CTA per SM and lose (99).
#include <atomic>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace mlora {
namespace {

constexpr int kChThreads = 512;
constexpr int kChVec = 2;                                 // float4 of logits a thread keeps
constexpr int kChPiece = kChThreads * kChVec * 4;         // tokens of a piece
constexpr int kChSmem = 2 * kChPiece * 8;  // counts and biases of two pieces
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

__global__ void __launch_bounds__(kChThreads, 3) choose_tokens_kernel(ChooseArgs a) {
  // of every second piece: its counts are made while other threads are still at the piece before
  extern __shared__ __align__(16) uint32_t s_tables[];
  uint32_t* s_counts = s_tables;                                           // low 30 bits: times in the answer; then: has a bias, is in the prompt
  float* s_biases = reinterpret_cast<float*>(s_tables + 2 * kChPiece);     // of the tokens that have one
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
    for (int j = 0; j < 2 * kChVec; ++j) {
      if (j >= kChVec && (int64_t)(rank + width) * kChPiece >= a.V) break;  // (one piece only)
      reinterpret_cast<uint4*>(s_counts)[j * kChThreads + tid] = make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
  }
  // the row's biases, one per thread, in ascending order of tokens: of equal ones the first has the sum
  const auto bias_at = [&](int i, int& w, float& sum) {
    w = i < b1 ? a.bias_token[i] : -1;
    if (w < 0 || (i > b0 && a.bias_token[i - 1] == w)) {
      w = -1;
      return;
    }
    sum = a.bias_value[i];
    for (int k = i + 1; k < b1 && a.bias_token[k] == w; ++k) sum += a.bias_value[k];
  };
  uint32_t* s_count = s_counts;
  float* s_bias = s_biases;
  const auto set_bias = [&](int w, float value, int v0) {
    const unsigned at = (unsigned)w - (unsigned)v0;
    if (w >= 0 && at < (unsigned)kChPiece) {
      atomicOr(&s_count[at], 0x40000000u);
      s_bias[at] = value;
    }
  };
  int bias_w = -1;
  float bias_v = 0.f;
  if (biased) bias_at(b0 + tid, bias_w, bias_v);
  float best_v = -INFINITY;  // (not a number, or not allowed: never above it)
  int best_i = 0;
  for (int64_t piece = (int64_t)rank * kChPiece; piece < a.V; piece += (int64_t)width * kChPiece) {
    const int v0 = (int)piece;
    float l[kChVec][4];
    uint32_t word[kChVec];
#pragma unroll
    for (int j = 0; j < kChVec; ++j) {
      const int at = v0 + (j * kChThreads + tid) * 4;
      word[j] = 0xfu;
      if (mask && at < a.V) word[j] = (uint32_t)mask[at >> 5] >> (at & 31);
      if (vec && at < a.V) {
        const float4 q = *reinterpret_cast<const float4*>(logits + at);  // (not the read-only path: `out` may be `logits`)
        l[j][0] = q.x, l[j][1] = q.y, l[j][2] = q.z, l[j][3] = q.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) l[j][e] = at < a.V - e ? logits[at + e] : -INFINITY;
      }
    }
    if (counts || biased) {
      prompt.walk(v0, [&](int p) { atomicOr(&s_count[p], 0x80000000u); });
      answer.walk(v0, [&](int p) { atomicAdd(&s_count[p], 1u); });
      set_bias(bias_w, bias_v, v0);
      for (int i = b0 + kChThreads + tid; i < b1; i += kChThreads) {
        int w;
        float value = 0.f;
        bias_at(i, w, value);
        set_bias(w, value, v0);
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kChVec; ++j) {
      const int q4 = j * kChThreads + tid, at = v0 + q4 * 4;
      if (counts || biased) {
        const uint4 c4 = reinterpret_cast<const uint4*>(s_count)[q4];
        if (c4.x | c4.y | c4.z | c4.w) {
          const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
          reinterpret_cast<uint4*>(s_count)[q4] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (!c[e]) continue;
            float v = l[j][e];
            const uint32_t times = c[e] & 0x3fffffffu;
            if (times || c[e] >> 31) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
            if (times) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)times)), pres);
            if (c[e] & 0x40000000u) v = __fadd_rn(v, s_bias[q4 * 4 + e]);
            l[j][e] = v;
          }
        }
      }
      if ((word[j] & 0xfu) != 0xfu) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!(word[j] >> e & 1u)) l[j][e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (l[j][e] > best_v) best_v = l[j][e], best_i = at + e;
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
    // (the other tables: nobody counts in these again before everybody has met behind the counts of the next piece)
    s_count = s_count == s_counts ? s_counts + kChPiece : s_counts;
    s_bias = s_bias == s_biases ? s_biases + kChPiece : s_biases;
  }
  unsigned long long best = warp_best(choice_key(best_v, best_i));
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
  // CTAs per row: some six per SM (256 rows x 128000 under all rules, in us: one 99, two 104, four 92, eight 101; 32 rows x 32000: one
  // 19.1, eight 7.5)
  int width = 1;
  while (width < kChCluster && width < pieces && (long long)T * width < 6 * 148) width *= 2;
  MLORA_REQUIRE((long long)T * width <= 2147483647ll, "choose_tokens: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(T * width));
  cfg.blockDim = dim3(kChThreads);
  cfg.dynamicSmemBytes = kChSmem;
  cfg.stream = (cudaStream_t)stream;
  static std::atomic<unsigned long long> allowed{0};  // by device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!((allowed.load(std::memory_order_acquire) >> (dev & 63)) & 1ull)) {
    const cudaError_t e = cudaFuncSetAttribute(choose_tokens_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kChSmem);
    if (e != cudaSuccess) return fail(MLORA_ECUDA, "choose_tokens: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    allowed.fetch_or(1ull << (dev & 63), std::memory_order_release);
  }
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
