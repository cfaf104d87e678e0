// Edits of the logits before the pick: penalties for the tokens that a row has already, biases and
// grammar masks, then the first maximum and its log-softmax.
#include "kernels.cuh"
#include "ptx.cuh"

namespace wv {
namespace {

constexpr int SH_THREADS = 256;
constexpr int SH_J = 32;                     // logits a thread holds
constexpr int SH_SLICE = SH_THREADS * SH_J;  // logits a CTA holds at a time

// (value, index) pairs: the larger value, ties to the lower index.
__device__ __forceinline__ void first_of(float &v, int &i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) {
    v = ov;
    i = oi;
  }
}

// One CTA a row, its vocabulary a slice at a time. Per slice a word of shared memory a token: the
// token's count among the history and the drafted tokens of the row's path in the low half, 1 + the
// last entry of its bias in the high half; counts and entries are whole numbers, so the order of the
// atomics does not matter. Then one read of the logits: edits in registers, the running maximum and
// sum of exponentials, and the edited row written where it is wanted.
template <typename T>
__global__ void __launch_bounds__(SH_THREADS) shape_kernel(const ShapeArgs a) {
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  __shared__ uint32_t note[SH_SLICE];
  __shared__ float wm[SH_THREADS / 32], ws[SH_THREADS / 32], wv_[SH_THREADS / 32];
  __shared__ int wi[SH_THREADS / 32];
  const int r = int(blockIdx.x), tid = int(threadIdx.x), lane = tid & 31, w = tid >> 5;
  const int s = a.row_seq ? a.row_seq[r] : r;
  if (s < 0 || s >= a.n) {  // padding
    if (tid == 0) {
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
  float m = -INFINITY, sum = 0.0f, bv = -INFINITY;
  int bi = 0x7fffffff;
  for (int lo = 0; lo < a.vocab; lo += SH_SLICE) {
    const int cnt = min(SH_SLICE, a.vocab - lo);
    for (int i = tid; i < SH_SLICE; i += SH_THREADS) note[i] = 0u;
    __syncthreads();
    for (int i = tid; i < bias; i += SH_THREADS) {
      const unsigned id = unsigned(a.bias_ids[(long long)s * a.max_bias + i] - lo);
      if (id < unsigned(cnt)) atomicMax(&note[id], uint32_t(i + 1) << 16);
    }
    __syncthreads();
    for (int i = tid; i < hist; i += SH_THREADS) {
      const unsigned id = unsigned(a.history[(long long)s * a.max_hist + i] - lo);
      if (id < unsigned(cnt)) atomicAdd(&note[id], 1u);
    }
    for (int i = tid; i < path; i += SH_THREADS) {
      const int at = first_row + i;
      if (at < 0 || at >= a.rows || !((a.path[(long long)r * a.path_words + (i >> 5)] >> (i & 31)) & 1u))
        continue;
      const unsigned id = unsigned(a.tokens[at] - lo);
      if (id < unsigned(cnt)) atomicAdd(&note[id], 1u);
    }
    __syncthreads();
    float x[SH_J], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < SH_J; ++j) {
      const int i = tid + SH_THREADS * j;
      if (i >= cnt) {
        x[j] = -INFINITY;
        continue;
      }
      float v = float(in[lo + i]);
      const uint32_t e = note[i], c = e & 0xffffu;
      if (c) {
        v = v > 0.0f ? v / rep : v * rep;
        v = __fsub_rn(v, __fadd_rn(__fmul_rn(freq, float(c)), pres));
      }
      if (e >> 16) v += a.bias_vals[(long long)s * a.max_bias + (e >> 16) - 1];
      if (allow && !((allow[(lo + i) >> 5] >> ((lo + i) & 31)) & 1u)) v = -INFINITY;
      if (out) out[lo + i] = T(v);
      if (v > bv) {
        bv = v;
        bi = lo + i;
      }
      top = fmaxf(top, v);
      x[j] = v;
    }
    const float m1 = fmaxf(m, top);
    if (m1 != -INFINITY) {
      sum *= __expf(m - m1);
      m = m1;
    }
#pragma unroll
    for (int j = 0; j < SH_J; ++j)
      if (x[j] != -INFINITY) sum += __expf(x[j] - m);
    __syncthreads();  // the notes are cleared for the next slice
  }
  float all = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    first_of(bv, bi, __shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
  }
  if (lane == 0) {
    wm[w] = all;
    wv_[w] = bv;
    wi[w] = bi;
  }
  __syncthreads();
  for (int k = 0; k < SH_THREADS / 32; ++k) all = fmaxf(all, wm[k]);
  sum *= m == -INFINITY ? 0.0f : __expf(m - all);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) ws[w] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.0f;
    for (int k = 0; k < SH_THREADS / 32; ++k) {
      sum += ws[k];
      first_of(bv, bi, wv_[k], wi[k]);
    }
    const bool dead = bv == -INFINITY;
    if (a.picks) a.picks[r] = dead ? -1 : bi;
    if (a.logprobs) a.logprobs[r] = !dead ? bv - all - logf(sum) : isnan(sum) ? sum : -INFINITY;
  }
}

}  // namespace

cudaError_t launch_shape(const ShapeArgs &a, int f16, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  if (f16) return launch_pdl(shape_kernel<__half>, dim3(a.rows), dim3(SH_THREADS), 0, s, a);
  return launch_pdl(shape_kernel<float>, dim3(a.rows), dim3(SH_THREADS), 0, s, a);
}

}  // namespace wv
