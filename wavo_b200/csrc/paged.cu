// Paged KV caches: the plan of a step (block tables and slot maps from request lengths) and the
// write of its K and V rows.
//
// A cache ("pool") is f16 [blocks][K, V][kv_heads][bs][hd]: the bs positions of one head's K (or V)
// in a block are one contiguous tile of bs x hd, which the attention loads as rows of a matrix. A
// slot is block * bs + offset.
#include <algorithm>

#include "kernels.cuh"
#include "ptx.cuh"

namespace wv {
namespace {

// ---- block tables and slot maps -----------------------------------------------------------
//
// want = ceil((len + add) / bs), need = max(0, want - owned); requests take their blocks in order
// while they fit: granted iff need = 0 or the running sum of needs (itself included) <= free. The
// sum only grows, so the granted requests' blocks are one run of the ring of free blocks from its
// head; what finished requests give back goes behind its tail, which no request of this call reads.
// A refused request's entries for the blocks that it lacks may name blocks of others (zeros from the
// start, or what it gave back once): they become -1, so that neither the attention nor the commit of
// the same step reaches those blocks through its rows.
//
// One launch and no hand-over between CTAs: a CTA takes `per` consecutive requests, sums what the
// others before it need (and what all do) from the 12 bytes of each, and scans its own. A few
// microseconds of latency, not bytes, bound it: at 2048 requests every CTA reads 24 KB out of L2.
// 32 requests of 16 rows take 6.7 us on the device from cold caches, 2048 requests of up to 96 rows
// 16 us; a call from Python costs the host 8 to 10 us.
constexpr int BT_THREADS = 256;

struct BtNeed {
  int add, need, gone, wide, owned, len;
};

__device__ __forceinline__ BtNeed bt_need(const BlockTablesArgs &a, int s) {
  BtNeed r;
  const int add = a.adds[s];
  r.len = max(a.lens[s], 0);
  r.owned = min(max(a.owned[s], 0), a.width);
  r.add = max(add, 0);
  const long long want = ((long long)r.len + r.add + a.bs - 1) >> a.shift;  // bs is a power of two
  r.wide = add >= 0 && want > a.width;
  r.need = add >= 0 && !r.wide ? max(int(want) - r.owned, 0) : 0;
  r.gone = add < 0 ? r.owned : 0;
  return r;
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Inclusive scan over the CTA's threads; `sh` holds a slot per warp.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T *sh) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) sh[w] = v;
  __syncthreads();
  for (int k = 0; k < w; ++k) v += sh[k];
  return v;
}

__global__ void __launch_bounds__(BT_THREADS) block_tables_kernel(const BlockTablesArgs a, int per) {
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  constexpr int W = BT_THREADS / 32;
  __shared__ long long sh_rows[2][W];
  __shared__ int sh_sum[2][W][4];
  __shared__ long long scan_l[W];
  __shared__ int scan_i[W];
  __shared__ long long first[BT_THREADS + 1];  // first row of each request of this CTA
  __shared__ int s_len[BT_THREADS], s_owned[BT_THREADS], s_at[BT_THREADS], s_got[BT_THREADS],
      s_gone[BT_THREADS], s_back[BT_THREADS], s_lack[BT_THREADS];
  __shared__ bool s_ok[BT_THREADS];
  const int tid = int(threadIdx.x), lane = tid & 31, w = tid >> 5;
  const int lo = int(blockIdx.x) * per, hi = min(a.n, lo + per);
  const int head = ((a.state[0] % a.cap) + a.cap) % a.cap;
  const int free = min(max(a.state[1], 0), a.cap);

  // Sums over the requests before this CTA's ([0]) and over all ([1]): rows, needs, blocks given
  // back, requests with a need, requests wider than the table.
  long long rows[2] = {0, 0};
  int sum[2][4] = {};
#pragma unroll 4
  for (int s = tid; s < a.n; s += BT_THREADS) {
    const BtNeed r = bt_need(a, s);
    const int v[4] = {r.need, r.gone, r.need > 0, r.wide};
    rows[1] += r.add;
    if (s < lo) rows[0] += r.add;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sum[1][k] += v[k];
      if (s < lo) sum[0][k] += v[k];
    }
  }
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    rows[g] = warp_sum(rows[g]);
    if (lane == 0) sh_rows[g][w] = rows[g];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sum[g][k] = warp_sum(sum[g][k]);
      if (lane == 0) sh_sum[g][w][k] = sum[g][k];
    }
  }
  __syncthreads();
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    rows[g] = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[g][k] = 0;
    for (int i = 0; i < W; ++i) {
      rows[g] += sh_rows[g][i];
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[g][k] += sh_sum[g][i][k];
    }
  }
  const long long all_rows = min(rows[1], 0x7fffffffll);

  // This CTA's requests, one a thread.
  const int s = lo + tid;
  const bool mine = tid < per && s < hi;
  BtNeed r = {};
  if (mine) r = bt_need(a, s);
  const long long row_end = rows[0] + block_scan<long long>(r.add, scan_l);
  const int upto = sum[0][0] + block_scan<int>(r.need, scan_i);
  const int gone_end = sum[0][1] + block_scan<int>(r.gone, scan_i);
  const int pos_end = sum[0][2] + block_scan<int>(r.need > 0, scan_i);
  const bool back = mine && a.adds[s] < 0;
  const bool ok = mine && !back && !r.wide && (r.need == 0 || upto <= free);
  const int got = ok ? r.need : 0;
  const bool writer = blockIdx.y == 0;
  if (mine) {
    first[tid + 1] = row_end;
    s_len[tid] = r.len;
    s_owned[tid] = r.owned;
    s_at[tid] = int((head + (long long)(upto - r.need)) % a.cap);
    s_got[tid] = got;
    s_ok[tid] = ok;
    s_gone[tid] = r.gone;
    s_lack[tid] = ok || back ? 0 : r.wide ? a.width - r.owned : r.need;
    s_back[tid] = int((head + (long long)free + gone_end - r.gone) % a.cap);
    if (writer) {
      a.row_start[s + 1] = int(min(row_end, 0x7fffffffll));
      a.owned_out[s] = back ? 0 : r.owned + got;
    }
  }
  if (tid == 0) {
    first[0] = rows[0];
    if (writer && blockIdx.x == 0) a.row_start[0] = 0;
  }
  // The ring's new state: all needs met, or the run ends before the first request that is not.
  if (writer) {
    const bool cross = mine && r.need > 0 && upto > free && upto - r.need <= free;
    if (cross || (sum[1][0] <= free && blockIdx.x == 0 && tid == 0)) {
      const int taken = cross ? upto - r.need : sum[1][0];
      a.state_out[0] = int((head + (long long)taken) % a.cap);
      a.state_out[1] = free - taken + sum[1][1];
      a.state_out[2] = int(all_rows);
      a.state_out[3] = sum[1][3] + (cross ? sum[1][2] - (pos_end - 1) : 0);
    }
  }
  __syncthreads();
  const int cnt = hi - lo;
  // New table entries, and the blocks given back, a warp a request.
  if (writer) {
    for (int q = w; q < cnt; q += W) {
      int *t = a.table + (long long)(lo + q) * a.width;
      for (int k = lane; k < s_got[q]; k += 32)
        t[s_owned[q] + k] = a.ring[int((s_at[q] + (long long)k) % a.cap)];
      for (int k = lane; k < s_gone[q]; k += 32)
        a.ring[int((s_back[q] + (long long)k) % a.cap)] = t[k];
      for (int k = lane; k < s_lack[q]; k += 32)
        if (t[s_owned[q] + k] >= 0) t[s_owned[q] + k] = -1;
    }
  }
  // Slots of this CTA's rows; a block taken in this call is read from the ring.
  const long long end = min(first[cnt], (long long)a.rows_cap);
  for (long long i = first[0] + blockIdx.y * BT_THREADS + tid; i < end;
       i += (long long)gridDim.y * BT_THREADS) {
    int q = 0, top = cnt - 1;  // the request whose rows hold i
    while (q < top) {
      const int m = (q + top) / 2;
      if (first[m + 1] > i) top = m;
      else q = m + 1;
    }
    const int pos = s_len[q] + int(i - first[q]);
    const int blk = pos >> a.shift;
    int slot = -1;
    if (s_ok[q]) {
      const int b = blk < s_owned[q]
                        ? a.table[(long long)(lo + q) * a.width + blk]
                        : a.ring[int((s_at[q] + (long long)(blk - s_owned[q])) % a.cap)];
      slot = (b << a.shift) + (pos & (a.bs - 1));
    }
    a.row_seq[i] = lo + q;
    a.slots[i] = slot;
  }
  // Rows past the last request's.
  const long long cta = blockIdx.y * (long long)gridDim.x + blockIdx.x;
  const long long ctas = (long long)gridDim.x * gridDim.y;
  for (long long i = all_rows + cta * BT_THREADS + tid; i < a.rows_cap; i += ctas * BT_THREADS) {
    a.row_seq[i] = -1;
    a.slots[i] = -1;
  }
}

// ---- K and V rows into the cache ----------------------------------------------------------

// Eight elements a thread and row (one 16-byte store); a thread keeps its place in the row, so that
// the head and the element are divided out once. Bound by the memory: 48000 f32 rows of 2560 (737
// MB) take 126 us, 5.9 TB/s, 0.91 of the measured copy.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load8(const T *p) {
  uint4 o;
  if constexpr (sizeof(T) == 2) {
    if constexpr (VEC) return *reinterpret_cast<const uint4 *>(p);
    __half2 h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = __halves2half2(p[2 * k], p[2 * k + 1]);
    o = *reinterpret_cast<uint4 *>(h);
  } else {
    float v[8];
    if constexpr (VEC) {
      *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(p);
      *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(p + 4);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = p[k];
    }
    o = make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]),
                   pack_half2(v[6], v[7]));
  }
  return o;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    pack_slots_kernel(const T *__restrict__ x, long long stride, const int *__restrict__ slots,
                      int rows, __half *__restrict__ pool, int nslots, int bs, int kv_heads,
                      int hd) {
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  const int kvd = kv_heads * hd;
  const int v = int(blockIdx.x * blockDim.x + threadIdx.x) * 8;  // element of the row's [K | V]
  if (v >= 2 * kvd) return;
  const int part = v >= kvd, c = v - part * kvd, h = c / hd, e = c - h * hd;
  const long long tile = (long long)bs * hd;
  const long long in_block = (long long)(part * kv_heads + h) * tile + e;
  for (int r = int(blockIdx.y); r < rows; r += int(gridDim.y)) {
    const int slot = slots[r];
    if (slot < 0 || slot >= nslots) continue;
    const int b = slot / bs, i = slot - b * bs;
    const uint4 o = load8<T, VEC>(x + r * stride + v);
    *reinterpret_cast<uint4 *>(pool + (long long)b * 2 * kv_heads * tile + in_block +
                               (long long)i * hd) = o;
  }
}

// ---- the commit of a drafted path -----------------------------------------------------------

// One CTA a request and layer. The walk: from the root (node 0) to the first child whose token is
// the pick of the node, as long as there is one; a child's path is its parent's and itself, so the
// test is one comparison of mask words. Warp 0 walks (32 candidates a step); every layer's CTA
// walks for itself, which costs less than a second launch. Then the accepted nodes' K and V move to
// consecutive positions. path[k] >= k and rises, so no destination is the source of a later move,
// and a thread that keeps its place in the head and walks k upwards needs no barrier. A chain of
// latencies (row starts, tokens, the walk, table entries, one load and store) bounds it: 128
// requests of up to 64 nodes over 4 layers take 9 to 12 us on the device from cold caches, and took
// 16 to 20 with each move's store before the next move's load.
constexpr int TA_THREADS = 256;
constexpr int TA_MAX = 256;  // nodes of a tree
constexpr int TA_BATCH = 8;

__global__ void __launch_bounds__(TA_THREADS) tree_accept_kernel(const TreeAcceptArgs a) {
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  __shared__ uint32_t mask[TA_MAX * 8];
  __shared__ int tok[TA_MAX], pick[TA_MAX], path[TA_MAX];
  // Element offsets of the accepted nodes off their place, and of the places they go to; -1: not
  // there.
  __shared__ long long from[TA_MAX], to[TA_MAX];
  __shared__ int s_count;
  const int s = int(blockIdx.x), layer = int(blockIdx.y), tid = int(threadIdx.x);
  const int lo = min(max(a.row_start[s], 0), a.rows);
  const int t = min(min(max(a.row_start[s + 1] - lo, 0), a.max_rows), a.rows - lo);
  const int len = max(a.lens[s], 0), words = a.words;
  for (int i = tid; i < t; i += TA_THREADS) {
    tok[i] = a.tokens[lo + i];
    pick[i] = a.picks[lo + i];
  }
  for (int i = tid; i < t * words; i += TA_THREADS) mask[i] = a.mask[(long long)lo * words + i];
  __syncthreads();
  if (tid < 32) {
    int cur = 0, count = 0;
    if (t > 0) {
      if (tid == 0) path[0] = 0;
      count = 1;
      while (true) {
        int next = -1;
        for (int base = cur + 1; base < t && next < 0; base += 32) {
          const int j = base + tid;
          bool fits = j < t && tok[j] == pick[cur];
          for (int k = 0; fits && k < words; ++k) {
            const uint32_t self = (j >> 5) == k ? 1u << (j & 31) : 0u;
            fits = (mask[j * words + k] ^ self) == mask[cur * words + k];
          }
          const unsigned m = __ballot_sync(0xffffffffu, fits);
          if (m) next = base + __ffs(m) - 1;
        }
        if (next < 0) break;
        cur = next;
        if (tid == 0) path[count] = cur;
        ++count;
      }
    }
    if (tid == 0) {
      s_count = count;
      if (layer == 0) {
        a.count[s] = count;
        a.next[s] = count ? pick[cur] : -1;
        a.new_lens[s] = len + count;
      }
    }
  }
  __syncthreads();
  const int count = s_count;
  if (layer == 0)
    for (int i = tid; i < a.max_rows; i += TA_THREADS)
      a.path[(long long)s * a.max_rows + i] = i < count ? path[i] : -1;
  if (!a.pool) return;
  const long long tile = (long long)a.bs * a.hd, block = 2ll * a.kv_heads * tile;
  const int *table = a.table + (long long)s * a.width;
  const auto place = [&](int pos) -> long long {
    const int blk = pos / a.bs;
    if (pos < 0 || blk >= a.width) return -1;
    const int b = table[blk];
    return b < 0 || b >= a.blocks ? -1 : b * block + (long long)(pos - blk * a.bs) * a.hd;
  };
  __half *pool = a.pool + layer * a.layer_stride;
  int k0 = 0;  // the first node off its place
  while (k0 < count && path[k0] == k0) ++k0;
  const int moves = count - k0;
  for (int i = tid; i < moves; i += TA_THREADS) {
    from[i] = place(len + path[k0 + i]);
    to[i] = place(len + k0 + i);
  }
  __syncthreads();
  const int vecs = a.kv_heads * a.hd / 4;  // 16-byte words of a position's K and V
  for (int v = tid; v < vecs; v += TA_THREADS) {
    const int e = v * 8, h = e / a.hd;  // h counts K's heads, then V's
    const long long at = h * tile + (e - h * a.hd);
    // Eight moves' loads before their stores: no destination of these is a later move's source.
    for (int i0 = 0; i0 < moves; i0 += TA_BATCH) {
      uint4 x[TA_BATCH];
#pragma unroll
      for (int i = 0; i < TA_BATCH; ++i)
        if (i0 + i < moves && from[i0 + i] >= 0)
          x[i] = *reinterpret_cast<const uint4 *>(pool + from[i0 + i] + at);
#pragma unroll
      for (int i = 0; i < TA_BATCH; ++i)
        if (i0 + i < moves && from[i0 + i] >= 0 && to[i0 + i] >= 0)
          *reinterpret_cast<uint4 *>(pool + to[i0 + i] + at) = x[i];
    }
  }
}

}  // namespace

cudaError_t launch_block_tables(const BlockTablesArgs &a, int sms, cudaStream_t s) {
  if (a.n <= 0) return cudaSuccess;
  // One request a CTA up to two waves of CTAs, else as many as it takes (256 at most); several
  // CTAs share a request's rows where they come to more than 1024 a CTA.
  const int per = std::min(BT_THREADS, std::max(1, (a.n + 2 * sms - 1) / (2 * sms)));
  const int gx = (a.n + per - 1) / per;
  const long long each = ((long long)a.rows_cap + gx - 1) / gx;
  const int gy = int(std::min<long long>(std::max(1, 4 * sms / gx), (each + 1023) / 1024));
  return launch_pdl(block_tables_kernel, dim3(gx, std::max(gy, 1)), dim3(BT_THREADS), 0, s, a, per);
}

cudaError_t launch_pack_slots(const void *x, int x_f16, long long stride, const int *slots,
                              int rows, __half *pool, int nslots, int bs, int kv_heads, int hd,
                              int sms, cudaStream_t s) {
  if (rows <= 0) return cudaSuccess;
  const int vecs = kv_heads * hd / 4;
  const int parts = (vecs + 255) / 256, threads = ((vecs + parts - 1) / parts + 31) / 32 * 32;
  const dim3 grid(parts, std::min(rows, 65535));
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && stride * (x_f16 ? 2 : 4) % 16 == 0;
  const auto go = [&](auto kernel, auto *p) {
    return launch_pdl(kernel, grid, dim3(threads), 0, s, p, stride, slots, rows, pool, nslots, bs,
                      kv_heads, hd);
  };
  if (x_f16) {
    const auto *p = static_cast<const __half *>(x);
    return vec ? go(pack_slots_kernel<__half, true>, p) : go(pack_slots_kernel<__half, false>, p);
  }
  const auto *p = static_cast<const float *>(x);
  return vec ? go(pack_slots_kernel<float, true>, p) : go(pack_slots_kernel<float, false>, p);
}

cudaError_t launch_tree_accept(const TreeAcceptArgs &a, int n, int layers, cudaStream_t s) {
  if (n <= 0) return cudaSuccess;
  return launch_pdl(tree_accept_kernel, dim3(n, std::max(layers, 1)), dim3(TA_THREADS), 0, s, a);
}

}  // namespace wv
