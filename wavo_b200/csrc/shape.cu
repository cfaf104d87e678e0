// Edits of the logits before the pick: penalties for the tokens that a row has already, biases and
// grammar masks, then the first maximum and its log-softmax.
#include <algorithm>

#include "kernels.cuh"
#include "ptx.cuh"

namespace wv {
namespace {

// A row's vocabulary is cut into ranges, one a CTA; the CTAs of a row form a cluster (8 at most). A
// range passes through registers, four tokens a load and the next ones on their way: read once,
// masked, written where it is wanted, and reduced to (maximum, its first index, sum of
// exponentials), which meets the other CTAs' through distributed shared memory. The tokens that a
// row's history, path or biases name are few, and their edits (a division among them) many times
// the work of the others'. A bit a token takes them out of that pass; in the order of their ids
// they have a place each in a list, with a word: how often the token is in the history and the path
// in the low half, 1 + the last entry of its bias in the high half (whole numbers, so the order of
// the atomics does not matter). A thread edits one of them. 249 rows of 51866 f32 logits with
// grammars, 448 tokens of history and 200 biases (105 MB read and written): 29 us, 3.6 TB/s; 56 % of
// the issue slots are taken and 249 rows leave 47 of the 148 SMs with one row where the others
// have two. 32 rows 10 us, the call's host side.
constexpr int SH_THREADS = 512;
constexpr int SH_WARPS = SH_THREADS / 32;
constexpr int SH_G = 2;                         // groups of four tokens a thread holds
constexpr int SH_STEP = SH_THREADS * SH_G * 4;  // tokens a CTA holds at a time
constexpr int SH_NAMED = 4096;                  // named tokens that the list holds
constexpr int SH_SLICE = 65536;                 // tokens a range goes through at a time
constexpr int SH_CTAS = 8;                      // of a cluster
constexpr float SH_LOG2E = 1.4426950408889634f;

struct ShapePart {
  float top, sum;  // the largest value, the sum of exp(value - top)
  int at;          // where it is first
};

// Two parts as one: ties go to the lower index; a NaN sum stays.
__device__ __forceinline__ void shape_join(ShapePart &a, float top, float sum, int at) {
  const float m = fmaxf(a.top, top), base = m == -INFINITY ? 0.0f : m;
  a.sum = a.sum * ex2((a.top - base) * SH_LOG2E) + sum * ex2((top - base) * SH_LOG2E);
  if (top > a.top || (top == a.top && at < a.at)) a.at = at;
  a.top = m;
}

template <int LANES>
__device__ __forceinline__ void shape_join_lanes(ShapePart &a) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1)
    shape_join(a, __shfl_xor_sync(0xffffffffu, a.top, o), __shfl_xor_sync(0xffffffffu, a.sum, o),
               __shfl_xor_sync(0xffffffffu, a.at, o));
}

__device__ __forceinline__ void load4(const float *p, float (&x)[4]) {
  *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(p);
}
__device__ __forceinline__ void load4(const __half *p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2 *>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ void store4(float *p, const float (&x)[4]) {
  *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(__half *p, const float (&x)[4]) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
}

struct ShapeShared {
  uint32_t named[SH_SLICE / 32];    // a bit a place: a named token
  uint16_t before[SH_SLICE / 32];   // the bits of the words before each
  int list[SH_NAMED];               // the named tokens in order
  uint32_t note[SH_NAMED];
  int scan[SH_WARPS];
  ShapePart warps[SH_WARPS], part;
};

template <typename T>
__global__ void __launch_bounds__(SH_THREADS, 2)
    shape_kernel(const ShapeArgs a, int range, int slice) {
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  __shared__ ShapeShared sh;
  const int tid = int(threadIdx.x), lane = tid & 31, w = tid >> 5;
  const int r = int(blockIdx.y), ctas = int(gridDim.x), rank = int(blockIdx.x);
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
  // Places are token + shift, so that a place that four divides is an aligned address.
  const int shift = int(reinterpret_cast<uintptr_t>(in) / sizeof(T)) & 3;
  const bool vec_out =
      ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & (4 * sizeof(T) - 1)) == 0;
  const int places = a.vocab + shift, last = (a.vocab - 1) >> 5;
  const auto fetch = [&](int v, int hi, float (&x)[4]) {  // places v .. v + 3, -inf outside the row
    const int i = v - shift;
    if (v < hi && i >= 0 && i + 3 < a.vocab) {
      load4(in + i, x);
    } else {
#pragma unroll
      for (int y = 0; y < 4; ++y)
        x[y] = v < hi && i + y >= 0 && i + y < a.vocab ? float(in[i + y]) : -INFINITY;
    }
  };
  const int begin = rank * range, end = min(begin + range, places);
  float next[SH_G][4];
#pragma unroll
  for (int j = 0; j < SH_G; ++j)
    fetch(begin + 4 * (tid + SH_THREADS * j), min(begin + slice, end), next[j]);
  const bool pen = a.penalties != nullptr;
  const int hist = pen && a.history ? min(max(a.hist_len[s], 0), a.max_hist) : 0;
  const int path = pen && a.path ? a.path_words * 32 : 0;
  const int bias = a.bias_ids ? min(max(a.bias_len[s], 0), a.max_bias) : 0;
  const int set = a.grammar ? a.grammar_of[r] : -1;
  const uint32_t *allow =
      set >= 0 && set < a.n_grammar ? a.grammar + (long long)set * a.grammar_ld : nullptr;
  const int first_row = path ? a.row_start[s] : 0;
  const int *history = a.history + (long long)s * a.max_hist;
  const int *bias_ids = a.bias_ids + (long long)s * a.max_bias;
  const bool any_named = hist + path + bias > 0;
  // Drafted token i of the request if it is on the row's path, else -1.
  const auto path_token = [&](int i) {
    const int at = first_row + i;
    return at >= 0 && at < a.rows &&
                   ((a.path[(long long)r * a.path_words + (i >> 5)] >> (i & 31)) & 1u)
               ? a.tokens[at]
               : -1;
  };
  ShapePart all = {-INFINITY, 0.0f, 0x7fffffff};
  for (int lo = begin; lo < end; lo += slice) {
    const int hi = min(lo + slice, end), words = (hi - lo + 31) / 32;
    int listed = 0;
    if (any_named) {
      const unsigned cnt = unsigned(hi - lo);
      const auto place = [&](int id) {  // the token's place in the slice, or past it
        return id >= 0 && id < a.vocab ? unsigned(id + shift - lo) : ~0u;
      };
      // A thread's first entries stay in registers.
      const int h0 = tid < hist ? history[tid] : -1, b0 = tid < bias ? bias_ids[tid] : -1;
      const int p0 = tid < path ? path_token(tid) : -1;
      for (int i = tid; i < words; i += SH_THREADS) sh.named[i] = 0u;
      __syncthreads();
      const auto each = [&](const auto &use) {
        use(place(h0), -1);
        for (int i = tid + SH_THREADS; i < hist; i += SH_THREADS) use(place(history[i]), -1);
        use(place(p0), -1);
        for (int i = tid + SH_THREADS; i < path; i += SH_THREADS) use(place(path_token(i)), -1);
      };
      const auto each_bias = [&](const auto &use) {
        use(place(b0), tid);
        for (int i = tid + SH_THREADS; i < bias; i += SH_THREADS) use(place(bias_ids[i]), i);
      };
      const auto name = [&](unsigned to, int) {
        if (to < cnt) atomicOr(&sh.named[to >> 5], 1u << (to & 31));
      };
      each(name);
      each_bias(name);
      __syncthreads();
      // Where each word's tokens begin in the list: four words a thread.
      int mine[4], sum = 0;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        mine[y] = sum;
        if (4 * tid + y < words) sum += __popc(sh.named[4 * tid + y]);
      }
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      if (lane == 31) sh.scan[w] = upto;
      __syncthreads();
      int at = upto - sum;
      for (int k = 0; k < SH_WARPS; ++k) {
        if (k < w) at += sh.scan[k];
        listed += sh.scan[k];
      }
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (4 * tid + y < words) sh.before[4 * tid + y] = uint16_t(at + mine[y]);
      for (int i = tid; i < listed; i += SH_THREADS) sh.note[i] = 0u;
      __syncthreads();
      const auto rank_of = [&](unsigned to) {
        return int(sh.before[to >> 5]) + __popc(sh.named[to >> 5] & ((1u << (to & 31)) - 1u));
      };
      each_bias([&](unsigned to, int entry) {
        if (to < cnt) {
          const int k = rank_of(to);
          sh.list[k] = int(to);
          atomicMax(&sh.note[k], uint32_t(entry + 1) << 16);
        }
      });
      if (bias > 0) __syncthreads();  // the counts are added to the entries
      each([&](unsigned to, int) {
        if (to < cnt) {
          const int k = rank_of(to);
          sh.list[k] = int(to);
          atomicAdd(&sh.note[k], 1u);
        }
      });
      __syncthreads();
      const float rep = pen ? a.penalties[3 * s] : 1.0f, pres = pen ? a.penalties[3 * s + 1] : 0.0f;
      const float freq = pen ? a.penalties[3 * s + 2] : 0.0f;
      for (int k = tid; k < listed; k += SH_THREADS) {
        const int i = sh.list[k] + lo - shift;
        const uint32_t e = sh.note[k], c = e & 0xffffu;
        float z = float(in[i]);
        if (c) {
          z = z > 0.0f ? z / rep : z * rep;
          z = __fsub_rn(z, __fadd_rn(__fmul_rn(freq, float(c)), pres));
        }
        if (e >> 16) z += a.bias_vals[(long long)s * a.max_bias + (e >> 16) - 1];
        if (allow && !((allow[i >> 5] >> (i & 31)) & 1u)) z = -INFINITY;
        sh.note[k] = __float_as_uint(z);
      }
      if (out == in) __syncthreads();  // the pass writes over what was read here
    }
#pragma unroll 1
    for (int v0 = lo + 4 * tid; v0 - 4 * tid < hi; v0 += SH_STEP) {
      float x[SH_G][4];
#pragma unroll
      for (int j = 0; j < SH_G; ++j) {
#pragma unroll
        for (int y = 0; y < 4; ++y) x[j][y] = next[j][y];
        // The next step's, or the next slice's first.
        const int v = v0 + SH_STEP + 4 * SH_THREADS * j;
        const bool on = v0 - 4 * tid + SH_STEP < hi;
        fetch(on ? v : hi + 4 * (tid + SH_THREADS * j), on ? hi : min(hi + slice, end), next[j]);
      }
      float top = all.top;
#pragma unroll
      for (int j = 0; j < SH_G; ++j) {
        const int v = v0 + 4 * SH_THREADS * j, i = v - shift;
        if (v < hi) {
          const bool whole = i >= 0 && i + 3 < a.vocab;
          // What the pass keeps of the four: allowed and not named (those come after).
          uint32_t drop = 0u;
          if (allow) {
            const int i0 = max(i, 0), q = i0 >> 5;
            drop = ~(__funnelshift_r(allow[q], allow[min(q + 1, last)], i0 & 31) << (i0 - i));
          }
          if (listed) drop |= sh.named[(v - lo) >> 5] >> ((v - lo) & 31);
#pragma unroll
          for (int y = 0; y < 4; ++y) x[j][y] = drop & (1u << y) ? -INFINITY : x[j][y];
          if (out) {
            if (vec_out && whole) {
              store4(out + i, x[j]);
            } else {
#pragma unroll
              for (int y = 0; y < 4; ++y)
                if (i + y >= 0 && i + y < a.vocab) out[i + y] = T(x[j][y]);
            }
          }
          if (fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])) > top) {
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (x[j][y] > top) {
                top = x[j][y];
                all.at = i + y;
              }
          }
        }
      }
      // The difference first: a rounded product of the maximum would be common to all terms and stay
      // in the sum, and past the largest value it is no number.
      const float base = top == -INFINITY ? 0.0f : top;
      if (top > all.top) {
        all.sum *= ex2((all.top - base) * SH_LOG2E);
        all.top = top;
      }
#pragma unroll
      for (int j = 0; j < SH_G; ++j)
#pragma unroll
        for (int y = 0; y < 4; ++y) all.sum += ex2((x[j][y] - base) * SH_LOG2E);
    }
    if (listed) {
      __syncthreads();  // the pass has written its values there
      // The named tokens join the maximum here: the pass takes the first of equal values by going
      // upwards, and these are below and above what it has seen.
      for (int k = tid; k < listed; k += SH_THREADS) {
        const int i = sh.list[k] + lo - shift;
        const float z = __uint_as_float(sh.note[k]);
        if (out) out[i] = T(z);
        shape_join(all, z, z == -INFINITY ? 0.0f : isnan(z) ? z : 1.0f, i);
      }
    }
    if (any_named && hi < end) __syncthreads();  // the list is made anew
  }
  if (!a.picks && !a.logprobs) return;
  shape_join_lanes<32>(all);
  if (lane == 0) sh.warps[w] = all;
  __syncthreads();
  if (w == 0) {
    all = sh.warps[lane % SH_WARPS];
    shape_join_lanes<SH_WARPS>(all);
    if (lane == 0) sh.part = all;
  }
  if (ctas > 1) cluster_sync();
  if (rank == 0 && tid == 0) {
    for (int p = 1; p < ctas; ++p) {
      uint32_t v[3];
#pragma unroll
      for (int x = 0; x < 3; ++x)
        asm volatile("ld.shared::cluster.u32 %0, [%1];"
                     : "=r"(v[x])
                     : "r"(mapa_shared(&sh.part, p) + 4 * x)
                     : "memory");
      shape_join(all, __uint_as_float(v[0]), __uint_as_float(v[1]), int(v[2]));
    }
    const bool dead = all.top == -INFINITY;  // nothing left
    if (a.picks) a.picks[r] = dead ? -1 : all.at;
    if (a.logprobs) a.logprobs[r] = !dead ? -logf(all.sum) : isnan(all.sum) ? all.sum : -INFINITY;
  }
  if (ctas > 1) cluster_sync();  // the parts stay until they are read
}

template <typename T>
cudaError_t launch(const ShapeArgs &a, int sms, cudaStream_t s) {
  // As many CTAs a row (a power of two) as the SMs hold at once, two each; ranges of 2048 tokens at
  // least. Every CTA names the row's tokens anew and waits for its cluster, so more cost more: 249
  // rows of 51866 with 1, 2, 4, 8 CTAs 30, 37, 51, 80 us, 90 rows 25, 19, 25, 32, 32 rows 17, 14,
  // 12, 11.
  int ctas = 1;
  while (ctas < SH_CTAS && a.rows * 2ll * ctas <= 2ll * sms && a.vocab / (2 * ctas) >= 2048) ctas *= 2;
  const int places = a.vocab + 3;
  const int range = ((places + ctas - 1) / ctas + 31) / 32 * 32;
  // The list holds every named token of a slice.
  const long long named = (long long)(a.penalties && a.history ? a.max_hist : 0) +
                          (a.penalties && a.path ? 32 * a.path_words : 0) +
                          (a.bias_ids ? a.max_bias : 0);
  const int slice = std::min(range, named <= SH_NAMED ? SH_SLICE : SH_NAMED);
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
  return cudaLaunchKernelEx(&cfg, shape_kernel<T>, a, range, slice);
}

}  // namespace

cudaError_t launch_shape(const ShapeArgs &a, int f16, int sms, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  return f16 ? launch<__half>(a, sms, s) : launch<float>(a, sms, s);
}

}  // namespace wv
