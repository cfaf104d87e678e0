// Edits of the logits before the pick: penalties for the tokens that a row has already, biases and
// grammar masks, then the first maximum and its log-softmax.
#include <algorithm>

#include "kernels.cuh"
#include "ptx.cuh"

namespace wv {
namespace {

// A row's vocabulary is cut into slices, one a CTA; the CTAs of a row form a cluster (8 at most, and
// a larger vocabulary goes round). A thread keeps SH_J of the slice's logits in registers: they are
// read once, edited, written where they are wanted, and reduced to (maximum, its first index, sum of
// exponentials) in one pass, which meets the other CTAs' through distributed shared memory.
// What a row's tokens say of a slice stands in a word of shared memory a token: how often it is among
// the history and the row's path in the low half, 1 + the last entry of its bias in the high half.
// Counts and entries are whole numbers, so the order of the atomics does not matter. The logits are on
// their way while the words are made.
constexpr int SH_THREADS = 512;
constexpr int SH_J = 16;                     // logits a thread holds
constexpr int SH_SLICE = SH_THREADS * SH_J;  // logits a CTA holds at a time
constexpr int SH_CTAS = 8;

struct ShapePart {
  float top, sum;  // the largest value, the sum of exp(value - top)
  int at;          // where it is first
};

// Two parts as one: ties go to the lower index; a NaN sum stays.
__device__ __forceinline__ void shape_join(ShapePart &a, float top, float sum, int at) {
  const float m = fmaxf(a.top, top), base = m == -INFINITY ? 0.0f : m;
  a.sum = a.sum * __expf(a.top - base) + sum * __expf(top - base);
  if (top > a.top || (top == a.top && at < a.at)) a.at = at;
  a.top = m;
}

template <typename T>
__global__ void __launch_bounds__(SH_THREADS, 2) shape_kernel(const ShapeArgs a, int slice) {
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  __shared__ alignas(16) uint32_t note[SH_SLICE];
  __shared__ ShapePart warps[SH_THREADS / 32], part;
  const int r = int(blockIdx.y), tid = int(threadIdx.x), lane = tid & 31, w = tid >> 5;
  const int ctas = int(gridDim.x), rank = int(blockIdx.x);
  const int s = a.row_seq ? a.row_seq[r] : r;
  if (s < 0 || s >= a.n) {  // padding
    if (rank == 0 && tid == 0) {
      if (a.picks) a.picks[r] = -1;
      if (a.logprobs) a.logprobs[r] = -INFINITY;
    }
    return;
  }
  const T *in = static_cast<const T *>(a.logits) + r * a.ld;
  T *out = a.out ? static_cast<T *>(a.out) + r * a.ld_out : nullptr;
  const bool pen = a.penalties != nullptr;
  const float rep = pen ? a.penalties[3 * s] : 1.0f, pres = pen ? a.penalties[3 * s + 1] : 0.0f,
              freq = pen ? a.penalties[3 * s + 2] : 0.0f;
  const int hist = pen && a.history ? min(max(a.hist_len[s], 0), a.max_hist) : 0;
  const int path = pen && a.path ? a.path_words * 32 : 0;
  const int bias = a.bias_ids ? min(max(a.bias_len[s], 0), a.max_bias) : 0;
  const int g = a.grammar ? a.grammar_of[r] : -1;
  const uint32_t *allow = g >= 0 && g < a.n_grammar ? a.grammar + (long long)g * a.grammar_ld : nullptr;
  const int first_row = path ? a.row_start[s] : 0;
  const bool notes = hist + path + bias > 0;
  ShapePart all = {-INFINITY, 0.0f, 0x7fffffff};
  for (int lo = rank * slice; lo < a.vocab; lo += ctas * slice) {
    const int cnt = min(slice, a.vocab - lo);
    float x[SH_J];
    uint32_t bits[SH_J];
#pragma unroll
    for (int j = 0; j < SH_J; ++j) {
      const int i = tid + SH_THREADS * j;
      x[j] = i < cnt ? float(in[lo + i]) : -INFINITY;
      // Slices begin at multiples of 32: a warp's 32 tokens share a word.
      bits[j] = allow && i < cnt ? allow[(lo + i) >> 5] : ~0u;
    }
    if (notes) {
      for (int i = tid; i < SH_SLICE / 4; i += SH_THREADS)
        reinterpret_cast<uint4 *>(note)[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
      if (bias > 0) {
        for (int i = tid; i < bias; i += SH_THREADS) {
          const unsigned id = unsigned(a.bias_ids[(long long)s * a.max_bias + i] - lo);
          if (id < unsigned(cnt)) atomicMax(&note[id], uint32_t(i + 1) << 16);
        }
        __syncthreads();  // the counts are added to the entries
      }
      for (int i = tid; i < hist; i += SH_THREADS) {
        const unsigned id = unsigned(a.history[(long long)s * a.max_hist + i] - lo);
        if (id < unsigned(cnt)) atomicAdd(&note[id], 1u);
      }
      for (int i = tid; i < path; i += SH_THREADS) {
        const int at = first_row + i;
        if (at < 0 || at >= a.rows ||
            !((a.path[(long long)r * a.path_words + (i >> 5)] >> (i & 31)) & 1u))
          continue;
        const unsigned id = unsigned(a.tokens[at] - lo);
        if (id < unsigned(cnt)) atomicAdd(&note[id], 1u);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < SH_J; ++j) {
        const int i = tid + SH_THREADS * j;
        const uint32_t e = i < cnt ? note[i] : 0u;
        if (e) {
          const uint32_t c = e & 0xffffu;
          float v = x[j];
          if (c) {
            v = v > 0.0f ? v / rep : v * rep;
            v = __fsub_rn(v, __fadd_rn(__fmul_rn(freq, float(c)), pres));
          }
          if (e >> 16) v += a.bias_vals[(long long)s * a.max_bias + (e >> 16) - 1];
          x[j] = v;
        }
      }
      if (lo + ctas * slice < a.vocab) __syncthreads();  // the words are made anew
    }
    ShapePart mine = {-INFINITY, 0.0f, 0x7fffffff};
#pragma unroll
    for (int j = 0; j < SH_J; ++j) {
      const int i = tid + SH_THREADS * j;
      if (!((bits[j] >> ((lo + i) & 31)) & 1u)) x[j] = -INFINITY;
      if (out && i < cnt) out[lo + i] = T(x[j]);
      if (x[j] > mine.top) {
        mine.top = x[j];
        mine.at = lo + i;
      }
    }
    const float base = mine.top == -INFINITY ? 0.0f : mine.top;
#pragma unroll
    for (int j = 0; j < SH_J; ++j) mine.sum += __expf(x[j] - base);
    shape_join(all, mine.top, mine.sum, mine.at);
  }
  if (!a.picks && !a.logprobs) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    shape_join(all, __shfl_xor_sync(0xffffffffu, all.top, o), __shfl_xor_sync(0xffffffffu, all.sum, o),
               __shfl_xor_sync(0xffffffffu, all.at, o));
  if (lane == 0) warps[w] = all;
  __syncthreads();
  if (w == 0) {
    all = lane < SH_THREADS / 32 ? warps[lane] : ShapePart{-INFINITY, 0.0f, 0x7fffffff};
#pragma unroll
    for (int o = SH_THREADS / 64; o > 0; o >>= 1)
      shape_join(all, __shfl_xor_sync(0xffffffffu, all.top, o),
                 __shfl_xor_sync(0xffffffffu, all.sum, o), __shfl_xor_sync(0xffffffffu, all.at, o));
    if (lane == 0) part = all;
  }
  if (ctas > 1) cluster_sync();
  if (rank == 0 && tid == 0) {
    for (int p = 1; p < ctas; ++p) {
      uint32_t v[3];
#pragma unroll
      for (int k = 0; k < 3; ++k)
        asm volatile("ld.shared::cluster.u32 %0, [%1];"
                     : "=r"(v[k])
                     : "r"(mapa_shared(&part, p) + 4 * k)
                     : "memory");
      shape_join(all, __uint_as_float(v[0]), __uint_as_float(v[1]), int(v[2]));
    }
    const bool dead = all.top == -INFINITY;
    if (a.picks) a.picks[r] = dead ? -1 : all.at;
    if (a.logprobs) a.logprobs[r] = !dead ? -logf(all.sum) : isnan(all.sum) ? all.sum : -INFINITY;
  }
  if (ctas > 1) cluster_sync();  // the parts stay until they are read
}

template <typename T>
cudaError_t launch(const ShapeArgs &a, cudaStream_t s) {
  const int ctas = std::min(SH_CTAS, (a.vocab + SH_SLICE - 1) / SH_SLICE);
  const int rounds = (a.vocab + ctas * SH_SLICE - 1) / (ctas * SH_SLICE);
  const int slice = ((a.vocab + ctas * rounds - 1) / (ctas * rounds) + 31) / 32 * 32;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, a.rows);
  cfg.blockDim = dim3(SH_THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, shape_kernel<T>, a, slice);
}

}  // namespace

cudaError_t launch_shape(const ShapeArgs &a, int f16, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  return f16 ? launch<__half>(a, s) : launch<float>(a, s);
}

}  // namespace wv
