// Attention of drafted tokens over a paged KV cache (the pool of paged.cu).
//
// Row i of a request sees its len cached positions and, with a mask, those of the rows drafted with
// it whose bits its mask words hold (row j's K and V are at position len + j). o = softmax(q.k /
// sqrt(hd)) v over what it sees, zeros where it sees nothing.
#include "kernels.cuh"
#include "ptx.cuh"

namespace wv {
namespace {

constexpr int TS_THREADS = 128;

// One CTA a (row, head, request): 128 keys a step, a key a thread for the scores, then an
// element a thread for the values; the running maximum and sum as usual.
template <typename T>
__global__ void __launch_bounds__(TS_THREADS) attend_tree_kernel(const AttendTreeArgs a) {
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  __shared__ float qs[128], ps[TS_THREADS], red[TS_THREADS / 32];
  __shared__ long long at[TS_THREADS];
  const int i = int(blockIdx.x), h = int(blockIdx.y), s = int(blockIdx.z);
  const int tid = int(threadIdx.x), lane = tid & 31, w = tid >> 5;
  const int lo = a.row_start ? a.row_start[s] : s;
  const int t = min(a.row_start ? a.row_start[s + 1] - lo : 1, a.max_rows);
  const int row = lo + i;
  if (i >= t || row < 0 || row >= a.rows) return;
  const T *q = static_cast<const T *>(a.q) + row * a.q_stride + h * a.hd;
  if (tid < a.hd) qs[tid] = float(q[tid]);
  const long long tile = (long long)a.bs * a.hd;
  const int kvh = h / (a.heads / a.kv_heads);
  const int *table = a.table + (long long)s * a.width;
  const int len = max(a.lens[s], 0);
  const int keys = int(min((long long)len + (a.mask ? t : 0), (long long)a.width * a.bs));
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  __syncthreads();
  for (int j0 = 0; j0 < keys; j0 += TS_THREADS) {
    const int j = j0 + tid;
    float x = -INFINITY;
    if (j < keys) {
      const int d = j - len;
      const bool seen = d < 0 || (d < 32 * a.words &&
                                  ((a.mask[(long long)row * a.words + (d >> 5)] >> (d & 31)) & 1u));
      const int b = table[j / a.bs];
      if (seen && b >= 0 && b < a.blocks) {
        const long long o = ((long long)b * 2 * a.kv_heads + kvh) * tile + (long long)(j % a.bs) * a.hd;
        at[tid] = o + a.kv_heads * tile;
        x = 0.0f;
        for (int e = 0; e < a.hd; ++e) x = fmaf(qs[e], __half2float(a.pool[o + e]), x);
        x *= a.scale;
      }
    }
    float mx = x;
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) red[w] = mx;
    __syncthreads();
    for (int k = 0; k < TS_THREADS / 32; ++k) mx = fmaxf(mx, red[k]);
    const float m1 = fmaxf(m, mx);
    if (m1 != -INFINITY) {
      const float c = __expf(m - m1);
      ps[tid] = x == -INFINITY ? 0.0f : __expf(x - m1);
      l *= c;
      acc *= c;
      m = m1;
    } else {
      ps[tid] = 0.0f;
    }
    __syncthreads();
    for (int k = 0; k < min(TS_THREADS, keys - j0); ++k)
      if (ps[k] != 0.0f) {
        l += ps[k];
        if (tid < a.hd) acc = fmaf(ps[k], __half2float(a.pool[at[k] + tid]), acc);
      }
    __syncthreads();
  }
  if (tid < a.hd)
    (static_cast<T *>(a.o) + row * a.o_stride + h * a.hd)[tid] = T(l != 0.0f ? acc / l : 0.0f);
}

}  // namespace

cudaError_t launch_attend_tree(const AttendTreeArgs &a, int f16, int n, cudaStream_t s) {
  if (n <= 0 || a.max_rows <= 0) return cudaSuccess;
  const dim3 grid(a.max_rows, a.heads, n);
  if (f16) return launch_pdl(attend_tree_kernel<__half>, grid, dim3(TS_THREADS), 0, s, a);
  return launch_pdl(attend_tree_kernel<float>, grid, dim3(TS_THREADS), 0, s, a);
}

}  // namespace wv
