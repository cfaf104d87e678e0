// Attention of drafted tokens over a paged KV cache (the pool of paged.cu).
//
// Row i of a request sees its len cached positions and, with a mask, those of the rows drafted with
// it whose bits its mask words hold (row j's K and V are at position len + j). o = softmax(q.k /
// sqrt(hd)) v over what it sees, zeros where it sees nothing.
//
// One pass over K and V with a running softmax. An item is one K and V head of one request with all
// the rows that read it (its drafted rows and the heads that share it, NR at most), so that K and V
// are read once for them all. The rows are few and the positions many, so the products are turned:
// 128 positions are the UMMA's M and the rows its N,
//   S^T [128 x NR] = K [128 x hd] . Q^T,   O^T [hd x NR] += V^T [hd x 128] . P^T,
// and a padded row costs N columns in steps of 16 where it would cost 128 lanes. A thread of the
// softmax has one position and all the rows (or half of them): no row is reduced over lanes but where
// its reference value has to rise. That is 8 (base 2) above it, at which a probability is still 256 in
// f16, so it happens at an item's first tile and seldom after; a vote a tile asks.
//
// The items' tiles of 128 positions lie one after another and are cut into equal runs, one a CTA, as
// many CTAs as are resident: ragged lengths, few long requests and many short ones fill the GPU alike,
// and the loads run ahead across the items of a run. A run that ends inside an item leaves its
// part in global memory; whichever CTA finishes an item's last part joins them, in the order
// of the runs.
#include <algorithm>
#include <type_traits>

#include "tree.cuh"

namespace wv {
namespace {

constexpr int TT_KEYS = 128;                  // positions a tile
constexpr uint32_t TT_HALF = TT_KEYS * 128;   // bytes of 128 positions x 64 elements
constexpr float TT_RISE = 8.0f;
constexpr int TT_PIECES = 3;                  // items in flight: loaded, multiplied, written
constexpr int TT_WHOLE = 4;                   // items of up to this many tiles stay in one run

// v[k] of 32 lanes reduced for each k: lane k gets the result of v[k] (31 shuffles for 32 values; the
// halves that a lane gives away it reads from its partner).
template <bool MAX, int N>
__device__ __forceinline__ float lanes_reduce(float (&v)[N]) {
  const int lane = int(threadIdx.x) & 31;
#pragma unroll
  for (int h = 16; h > 0; h >>= 1) {
    const bool up = (lane & h) != 0;
#pragma unroll
    for (int k = 0; k < h; ++k) {
      const float give = up ? v[k] : v[k + h], keep = up ? v[k + h] : v[k];
      const float got = __shfl_xor_sync(0xffffffffu, give, h);
      v[k] = MAX ? fmaxf(keep, got) : keep + got;
    }
  }
  return v[0];
}

// HDP: head size padded to 64 or 128. NR: rows of an item. WIDE: f32 rows, as two f16 parts each.
template <int HDP, int NR, bool WIDE>
struct TreeTile {
  static constexpr int kParts = WIDE ? 2 : 1;
  static constexpr uint32_t kSlot = (HDP / 64) * TT_HALF;           // a tile of K or of V
  static constexpr uint32_t kQ = (HDP / 64) * NR * 128;             // Q, one part
  static constexpr uint32_t kP = (NR + 63) / 64 * TT_HALF;          // P, one part
  // Up to 32 rows of heads of 64, two CTAs share an SM (113 KB of shared memory each); else one.
  static constexpr int kCtas = HDP == 64 && NR <= 32 ? 2 : 1;
  static constexpr int kPBufs = kCtas * kParts * kP >= 2 * TT_HALF ? 1 : 2;
  static constexpr int kQBufs = kParts * kQ > 16384 ? 1 : 2;
  static constexpr int kRing = HDP == 128 ? (kParts * NR >= 128 ? 3 : 4) : kCtas == 2 ? 4 : 8;
  // Softmax warps: a group of four holds the 128 positions; the groups share the rows, 16 at a time.
  static constexpr int kGroups = NR <= 32 ? 1 : 4;
  static constexpr int kRows = NR / kGroups;                        // rows a thread holds at most
  static constexpr int kSoft = 128 * kGroups;
  static constexpr int kThreads = kSoft + 96;                       // and loads, UMMAs, rows
  static constexpr uint32_t kOffQ = kRing * kSlot;
  static constexpr uint32_t kOffP = kOffQ + kQBufs * kParts * kQ;
  static constexpr uint32_t kOffBar = kOffP + kPBufs * kParts * kP;
  static constexpr uint32_t kCols = NR == 16 ? 64 : NR == 32 ? 128 : NR == 64 ? 256 : 512;
};

// A run's share of an item.
struct TreePiece {
  int s, kvh, r0, here;     // request, K and V head, first row, rows
  int lo, rows, len, keys;  // the request's first row, its drafted rows, positions without and with them
  int tile0, tiles;         // tiles of the item
  int slot;                 // where a partial result goes; -1: the item is whole
  int first, parts;         // the run that the item begins in, the runs that it takes
};

template <int NR>
struct TreeRows {
  long long out[NR];        // element offset of the row's output, -1: none
  uint32_t mask[NR][8];
};

template <int NR>
struct TreeShared {
  uint64_t full[8], empty[8], s_full[2], p_full[2], pv_done[2], q_full[2], q_empty[2];
  uint64_t piece_full[TT_PIECES], piece_empty[TT_PIECES], row_full[TT_PIECES], drain;
  TreePiece piece[TT_PIECES];
  TreeRows<NR> rows[TT_PIECES];
  uint32_t tmem, abort, last;
  uint32_t odd[8];              // drafted positions whose V holds an infinity or NaN
  long long scan[20], begin, end;
  int begin_s, begin_n;         // the run's first request and the tiles of it that lie before
  alignas(16) float lim[NR];    // a score above it raises its row's reference
  alignas(16) float base[NR];   // the reference (0 where a row has seen nothing)
  alignas(16) float fac[NR];    // what a rise takes off; at the end 1 / the sum
  float ref[NR];                // the reference, -inf where a row has seen nothing
  float red[4][NR];
};

// What an item's size follows from. A request without positions has one (empty) tile an item, which
// gives its rows their zeros.
struct TreeRequest {
  int lo, rows, len, keys;
  int row_tiles, tiles;  // items a K and V head; tiles an item
};

template <int NR>
__device__ __forceinline__ TreeRequest tree_request(const AttendTreeArgs &a, int s) {
  TreeRequest r;
  r.lo = a.row_start ? a.row_start[s] : s;
  r.rows = min(a.row_start ? a.row_start[s + 1] - r.lo : 1, a.max_rows);
  if (r.lo < 0 || r.rows < 0) r.rows = 0;
  r.len = max(a.lens[s], 0);
  r.keys = int(min((long long)r.len + (a.mask ? r.rows : 0), (long long)a.width * a.bs));
  r.row_tiles = (r.rows * (a.heads / a.kv_heads) + NR - 1) / NR;
  r.tiles = max((r.keys + TT_KEYS - 1) / TT_KEYS, 1);
  return r;
}

template <int HDP, int NR, bool WIDE>
__global__ void __launch_bounds__(TreeTile<HDP, NR, WIDE>::kThreads, TreeTile<HDP, NR, WIDE>::kCtas)
    attend_tree_kernel(const __grid_constant__ CUtensorMap map, const AttendTreeArgs a) {
  using T = TreeTile<HDP, NR, WIDE>;
  using E = typename std::conditional<WIDE, float, __half>::type;
  constexpr int D = T::kRing, SOFT = T::kSoft, R = T::kRows;
  constexpr int W_LOAD = SOFT / 32, W_MMA = W_LOAD + 1, W_ROWS = W_LOAD + 2, WARPS = W_LOAD + 3;
  extern __shared__ uint8_t raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  TreeShared<NR> &sh = *reinterpret_cast<TreeShared<NR> *>(smem + T::kOffBar);
  const int tid = int(threadIdx.x), lane = tid & 31, w = int(warp_id());
  const int group = a.heads / a.kv_heads;
  const Abort ab{&sh.abort, a.err};
  if (tid == 0) {
    for (int i = 0; i < D; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], W_LOAD);
      mbar_init(&sh.pv_done[i], 1);
      mbar_init(&sh.q_full[i], 1);
      mbar_init(&sh.q_empty[i], 1);
    }
    for (int i = 0; i < TT_PIECES; ++i) {
      mbar_init(&sh.piece_full[i], 1);
      mbar_init(&sh.piece_empty[i], 1);
      mbar_init(&sh.row_full[i], 1);
    }
    mbar_init(&sh.drain, 1);
    sh.abort = 0u;
    sh.begin = sh.end = 0;
    fence_mbar_init();
    prefetch_tmap(&map);
  }
  if (tid < 8) sh.odd[tid] = 0u;
  if (w == W_MMA) {
    tmem_alloc(&sh.tmem, T::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  const uint32_t tmem = sh.tmem;

  // ---- this CTA's run: tiles begin .. end of all ---------------------------------------------------
  const int per = (a.n + T::kThreads - 1) / T::kThreads;
  const int s_lo = min(tid * per, a.n), s_hi = min(s_lo + per, a.n);
  long long mine = 0;
  for (int s = s_lo; s < s_hi; ++s) {
    const TreeRequest r = tree_request<NR>(a, s);
    mine += (long long)r.row_tiles * a.kv_heads * r.tiles;
  }
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) sh.scan[w] = upto;
  __syncthreads();
  long long total = 0;
  for (int k = 0; k < WARPS; ++k) {
    if (k < w) upto += sh.scan[k];
    total += sh.scan[k];
  }
  const int runs = int(min((long long)gridDim.x, total));
  if (int(blockIdx.x) < runs) {
    // A boundary inside a short item moves to the item's end.
    for (int side = 0; side < 2; ++side) {
      const long long at = total * (blockIdx.x + side) / runs;
      if (side == 1 && at == total) {
        if (tid == 0) sh.end = total;
      } else if (at >= upto - mine && at < upto) {
        long long left = at - (upto - mine);
        int s = s_lo;
        TreeRequest r = tree_request<NR>(a, s);
        long long all = (long long)r.row_tiles * a.kv_heads * r.tiles;
        while (left >= all) {
          left -= all;
          r = tree_request<NR>(a, ++s);
          all = (long long)r.row_tiles * a.kv_heads * r.tiles;
        }
        const int into = int(left % r.tiles);
        const int move = into && r.tiles <= TT_WHOLE ? r.tiles - into : 0;
        if (side == 0) {
          sh.begin = at + move;
          sh.begin_s = s;
          sh.begin_n = int(left + move);
        } else {
          sh.end = at + move;
        }
      }
    }
  }
  __syncthreads();
  const int n = int(sh.end - sh.begin);  // tiles of this run

  if (w == W_LOAD) {
    // ---- loads: a lane a page of the tile. The ring takes them in the order in which the UMMAs do:
    // K0, K1, V0, K2, V1, ..., V(n-1). This warp also cuts the run into items for the others.
    const int box = min(a.bs, TT_KEYS), boxes = TT_KEYS / box;
    int s = sh.begin_s;
    TreeRequest r = {};
    const int *table = nullptr;
    int item = 0, tile = 0, items = 0;  // item of the request, tile of the item
    const auto enter = [&](int at) {
      s = at;
      r = tree_request<NR>(a, s);
      items = r.row_tiles * a.kv_heads;
      table = a.table + (long long)s * a.width;
    };
    const auto block_of = [&](int t) {
      const int p = t * TT_KEYS + lane * box;
      const int b = lane < boxes && p < r.keys ? table[p / a.bs] : -1;
      return b < 0 || b >= a.blocks ? a.blocks : b;  // past the tensor's end: zeros
    };
    if (n > 0) {
      enter(s);
      item = sh.begin_n / r.tiles;
      tile = sh.begin_n % r.tiles;
    }
    int p = 0, k = 0, z = 0, z_next = 0, zv = 0, yv = 0, hv = 0;
    bool ok = true, fresh = true, ahead = false;
    const auto load = [&](int y, int head, int block) {
      const int slot = p % D;
      ok = p < D || mbar_wait_warp(&sh.empty[slot], (p / D - 1) & 1, ab, kErrTimeoutProducer);
      if (!ok) return;
      if (lane == 0) mbar_arrive_expect_tx(&sh.full[slot], T::kSlot);
      __syncwarp();
      if (lane < boxes) {
        uint8_t *to = smem + slot * T::kSlot + lane * box * 128;
#pragma unroll
        for (int h = 0; h < HDP / 64; ++h)
          tma_load_4d(to + h * TT_HALF, &map, &sh.full[slot], 64 * h, y, head, block);
      }
      ++p;
    };
    for (int g = 0; g <= n && n > 0; ++g) {
      const int z_v = z, y_v = yv, h_v = hv;
      if (g < n) {
        while (tile == r.tiles || item >= items) {  // on to the next item, past requests without rows
          if (tile == r.tiles) tile = 0, ++item;
          if (item >= items) {
            enter(s + 1);
            item = 0;
          }
          fresh = true;
        }
        const int kvh = item / r.row_tiles;
        if (fresh) {
          if (k >= TT_PIECES &&
              !mbar_wait_warp(&sh.piece_empty[k % TT_PIECES], (k / TT_PIECES - 1) & 1, ab,
                              kErrTimeoutProducer))
            break;
          if (lane == 0) {
            TreePiece q;
            q.s = s;
            q.kvh = kvh;
            q.r0 = (item - kvh * r.row_tiles) * NR;
            q.here = min(r.rows * group - q.r0, NR);
            q.lo = r.lo;
            q.rows = r.rows;
            q.len = r.len;
            q.keys = r.keys;
            q.tile0 = tile;
            q.tiles = min(r.tiles - tile, n - g);
            q.slot = -1;
            q.first = q.parts = 0;
            if (q.tiles < r.tiles) {
              // Run c holds tile x where c = ((x + 1) runs - 1) / total, rounded down.
              const long long x0 = sh.begin + g - tile, x1 = x0 + r.tiles - 1;
              q.first = int(((x0 + 1) * runs - 1) / total);
              q.parts = int(((x1 + 1) * runs - 1) / total) - q.first + 1;
              q.slot = 2 * int(blockIdx.x) + (tile == 0 ? 1 : 0);
            }
            sh.piece[k % TT_PIECES] = q;
            mbar_arrive(&sh.piece_full[k % TT_PIECES]);
          }
          ++k;
          fresh = false;
          ahead = false;
        }
        z = ahead ? z_next : block_of(tile);
        ahead = tile + 1 < r.tiles;
        if (ahead) z_next = block_of(tile + 1);
        yv = (tile * TT_KEYS + lane * box) % a.bs;
        hv = kvh;
        zv = z;
        load(yv, hv, zv);
        if (!ok) break;
        ++tile;
      }
      if (g > 0) {
        load(y_v, a.kv_heads + h_v, z_v);
        if (!ok) break;
      }
    }
    // The shared memory stays until the last loads have landed, also where a wait gave up.
    for (int q = max(p - D, 0); q < p; ++q)
      for (int i = 0; i < 2000 && !mbar_try_wait_sleep(&sh.full[q % D], (q / D) & 1, 100000u); ++i) {}
  } else if (w == W_MMA) {
    // ---- UMMAs: S of a tile, then P.V of the one before it ---------------------------------------
    if (lane == 0 && n > 0) {
      const uint64_t dq = sdesc_sw128(smem_u32(smem + T::kOffQ), 16, 1024);
      const uint64_t dk = sdesc_sw128(smem_u32(smem), 16, 1024);
      // With heads of 64 lanes 64.. multiply what lies behind V in shared memory; nobody reads them.
      const uint64_t dv = sdesc_sw128(smem_u32(smem), TT_HALF, 1024);
      const uint64_t dp = sdesc_sw128(smem_u32(smem + T::kOffP), TT_HALF, 1024);
      int p = 0, k = -1, left = 0;
      uint32_t cols = 0, cols_v = 0;
      bool first = false, first_v = false, ok = true;
      for (int g = 0; g <= n; ++g) {
        cols_v = cols;
        first_v = first;
        if (g < n) {
          first = left == 0;
          if (first) {
            ++k;
            if (!mbar_wait(&sh.piece_full[k % TT_PIECES], (k / TT_PIECES) & 1, ab, kErrTimeoutMma))
              break;
            cols = uint32_t(sh.piece[k % TT_PIECES].here + 15) / 16 * 16;
            left = sh.piece[k % TT_PIECES].tiles;
            if (!mbar_wait(&sh.q_full[k % T::kQBufs], (k / T::kQBufs) & 1, ab, kErrTimeoutMma)) break;
          }
          const int slot = p % D;
          if (!mbar_wait(&sh.full[slot], (p / D) & 1, ab, kErrTimeoutMma)) break;
          ++p;
          tc_fence_after();
          const uint32_t id = idesc_f16(TT_KEYS, cols, 0);
          const uint64_t kd = dk + uint64_t(slot * T::kSlot >> 4);
          const uint64_t qd = dq + uint64_t((k % T::kQBufs) * T::kParts * T::kQ >> 4);
#pragma unroll
          for (int part = 0; part < T::kParts; ++part)
#pragma unroll
            for (int kk = 0; kk < HDP / 16; ++kk)
              umma_f16(tmem + (g & 1) * NR, kd + (((kk >> 2) * TT_HALF + (kk & 3) * 32) >> 4),
                       qd + ((part * T::kQ + (kk >> 2) * NR * 128 + (kk & 3) * 32) >> 4), id,
                       part + kk > 0 ? 1u : 0u);
          umma_commit(&sh.s_full[g & 1]);
          umma_commit(&sh.empty[slot]);
          if (--left == 0) umma_commit(&sh.q_empty[k % T::kQBufs]);
        }
        if (g > 0) {
          const int j = g - 1, slot = p % D;
          if (!(ok = mbar_wait(&sh.full[slot], (p / D) & 1, ab, kErrTimeoutMma) &&
                     mbar_wait(&sh.p_full[j & 1], (j >> 1) & 1, ab, kErrTimeoutMma)))
            break;
          ++p;
          tc_fence_after();
          const uint32_t id = idesc_f16(TT_KEYS, cols_v, 1) | (1u << 15);  // V^T: A is MN-major
          const uint64_t vd = dv + uint64_t(slot * T::kSlot >> 4);
          const uint64_t pd = dp + uint64_t((j % T::kPBufs) * T::kParts * T::kP >> 4);
#pragma unroll
          for (int part = 0; part < T::kParts; ++part)
#pragma unroll
            for (int kk = 0; kk < TT_KEYS / 16; ++kk)
              umma_f16(tmem + 2 * NR, vd + uint64_t(kk * 16 * 128 >> 4),
                       pd + uint64_t((part * T::kP + kk * 16 * 128) >> 4), id,
                       !first_v || part + kk > 0 ? 1u : 0u);
          umma_commit(&sh.pv_done[j & 1]);
          umma_commit(&sh.empty[slot]);
        }
      }
      // TMEM and shared memory stay until the last UMMA is done, also where a wait gave up.
      umma_commit(&sh.drain);
      const long long t0 = clock64();
      while (!mbar_try_wait(&sh.drain, 0) && clock64() - t0 < kWaitCycles) {
      }
    }
    __syncwarp();
  } else if (w == W_ROWS) {
    // ---- an item's rows: where they go, what they see, and Q into shared memory ------------------
    const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | (a.q_stride * sizeof(E))) & 15u) == 0;
    for (int k = 0, done = 0; done < n; ++k) {
      const int pc = k % TT_PIECES, qb = k % T::kQBufs;
      if (!mbar_wait_warp(&sh.piece_full[pc], (k / TT_PIECES) & 1, ab, kErrTimeoutConsumer)) break;
      const TreePiece &q = sh.piece[pc];
      TreeRows<NR> &to = sh.rows[pc];
      done += q.tiles;
      for (int r = lane; r < NR; r += 32) {
        const int i = (q.r0 + r) / group, head = q.kvh * group + (q.r0 + r) - i * group;
        const bool live = r < q.here && q.lo + i < a.rows;
        const long long row = q.lo + i;
        to.out[r] = !live ? -1
                    : q.slot < 0 ? row * a.o_stride + (long long)head * a.hd
                                 : ((long long)q.slot * NR + r) * (a.hd + 4);
        for (int x = 0; x < a.words; ++x)
          to.mask[r][x] = live ? a.mask[row * a.words + x] : 0u;
      }
      if (k >= T::kQBufs &&
          !mbar_wait_warp(&sh.q_empty[qb], (k / T::kQBufs - 1) & 1, ab, kErrTimeoutConsumer))
        break;
      uint8_t *base = smem + T::kOffQ + qb * T::kParts * T::kQ;
      // Eight elements a lane and step; rows to the next 16 are zeros.
      const int chunks = (q.here + 15) / 16 * 16 * (HDP / 8);
      const auto source = [&](int e) -> const E * {
        const int r = e / (HDP / 8), c = e % (HDP / 8);
        const int i = (q.r0 + r) / group, head = q.kvh * group + (q.r0 + r) - i * group;
        if (e >= chunks || r >= q.here || q.lo + i >= a.rows || c * 8 >= a.hd) return nullptr;
        return static_cast<const E *>(a.q) + (long long)(q.lo + i) * a.q_stride + head * a.hd + c * 8;
      };
      const auto target = [&](int e) {
        const int r = e / (HDP / 8), c = e % (HDP / 8);
        return base + (c >> 3) * NR * 128 + sw128_offset(r, c & 7);
      };
      if (!WIDE && vec) {
        // As they are, all in flight at once.
        for (int e = lane; e < chunks; e += 32) {
          const E *from = source(e);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(target(e))),
                       "l"(from ? from : static_cast<const E *>(a.q)), "r"(from ? 16 : 0)
                       : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
      } else {
        for (int e0 = lane; e0 < chunks; e0 += 128) {  // four steps in flight
          E v[4][8];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const E *from = source(e0 + 32 * u);
#pragma unroll
            for (int x = 0; x < 8; ++x) v[u][x] = E(0.0f);
            if (from && vec) {
#pragma unroll
              for (int x = 0; x < int(sizeof(E)) / 2; ++x)
                reinterpret_cast<uint4 *>(v[u])[x] = reinterpret_cast<const uint4 *>(from)[x];
            } else if (from) {
#pragma unroll
              for (int x = 0; x < 8; ++x) v[u][x] = from[x];
            }
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (e0 + 32 * u >= chunks) break;
            uint8_t *at = target(e0 + 32 * u);
            if constexpr (WIDE) {
              uint32_t hi[4], low[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) split2(v[u][2 * x], v[u][2 * x + 1], hi[x], low[x]);
              *reinterpret_cast<uint4 *>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
              *reinterpret_cast<uint4 *>(at + T::kQ) = make_uint4(low[0], low[1], low[2], low[3]);
            } else {
              *reinterpret_cast<uint4 *>(at) = *reinterpret_cast<const uint4 *>(v[u]);
            }
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh.row_full[pc]);
        mbar_arrive(&sh.q_full[qb]);
      }
    }
  } else {
    // ---- softmax: a position a thread, the warps of a group the rows from col0 on ------------------
    const auto sync = [] { asm volatile("barrier.cta.sync 1, %0;" ::"n"(SOFT) : "memory"); };
    const auto any = [](bool x) {  // a barrier that says whether any thread holds x
      uint32_t r;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.u32 p, %1, 0;\n\t"
          "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t}\n"
          : "=r"(r)
          : "r"(uint32_t(x)), "n"(SOFT)
          : "memory");
      return r != 0;
    };
    const int key = tid & 127, quarter = w & 3;
    const float scale = a.scale * 1.4426950408889634f;  // exponentials of base 2
    int pv = 0;  // V's place in the ring
    for (int k = 0, g = 0; g < n; ++k) {
      const int pc = k % TT_PIECES;
      // Where a wait gives up, all warps leave together; inside an item they run on (later waits give
      // up soon): the barriers need them all.
      bool ok = mbar_wait_warp(&sh.row_full[pc], (k / TT_PIECES) & 1, ab, kErrTimeoutConsumer);
      if (any(!ok)) break;
      const TreePiece &q = sh.piece[pc];
      const TreeRows<NR> &rows = sh.rows[pc];
      // This group's rows: col0 up to `here`, an even share in steps of 16.
      const int share = ((q.here + 15) / 16 + T::kGroups - 1) / T::kGroups * 16;
      const int col0 = (w >> 2) * share, tiles = q.tiles;
      const int here = min(q.here, col0 + share);
      const uint32_t lanes = tmem + (uint32_t(quarter) * 32u << 16) + col0;
      const int *table = a.table + (long long)q.s * a.width;
      for (int r = tid; r < NR; r += SOFT) {
        sh.ref[r] = -INFINITY;
        sh.base[r] = 0.0f;
        sh.lim[r] = rows.out[r] >= 0 ? -INFINITY : INFINITY;
      }
      float l[R];
#pragma unroll
      for (int r = 0; r < R; ++r) l[r] = 0.0f;
      const auto entry = [&](int pos) { return pos < q.keys ? table[pos / a.bs] : -1; };
      int b = entry(q.tile0 * TT_KEYS + key);
      sync();
      for (int i = 0; i < tiles; ++i, ++g) {
        const int pos = (q.tile0 + i) * TT_KEYS + key, d = pos - q.len;
        const bool there = b >= 0 && b < a.blocks;  // below q.keys and in the pool
        if (i + 1 < tiles) b = entry(pos + TT_KEYS);
        const bool all = __all_sync(0xffffffffu, there && d < 0);  // every row sees the warp's
        // What this position is seen by, a bit a row.
        uint32_t vis[(R + 31) / 32];
        if (!all) {
#pragma unroll
          for (int x = 0; x < (R + 31) / 32; ++x) {
            vis[x] = there ? ~0u : 0u;
            if (there && d >= 0) {
              vis[x] = 0u;
              if (d < 32 * a.words)
#pragma unroll
                for (int r = 0; r < (R < 32 ? R : 32); ++r)
                  if (col0 + 32 * x + r < here)
                    vis[x] |= ((rows.mask[col0 + 32 * x + r][d >> 5] >> (d & 31)) & 1u) << r;
            }
          }
        }
        mbar_wait_warp(&sh.s_full[g & 1], (g >> 1) & 1, ab, kErrTimeoutConsumer);
        tc_fence_after();
        uint32_t u[R / 16][16];
        __syncwarp();
#pragma unroll
        for (int c = 0; c < R / 16; ++c)
          if (col0 + 16 * c < here) tmem_ld16(lanes + (g & 1) * NR + 16 * c, u[c]);
        tmem_wait_ld();
        const auto x_of = [&](int r) -> float {
          return __uint_as_float(u[r / 16][r % 16]);
        };
        bool rise = false;
#pragma unroll
        for (int c = 0; c < R / 16; ++c)
          if (col0 + 16 * c < here) {
            if (!all) {
#pragma unroll
              for (int y = 0; y < 16; ++y)
                if (!((vis[c / 2] >> (16 * (c & 1) + y)) & 1u)) u[c][y] = 0xff800000u;  // -inf
            }
#pragma unroll
            for (int y = 0; y < 16; y += 4) {
              const float4 lim = *reinterpret_cast<const float4 *>(&sh.lim[col0 + 16 * c + y]);
              const int r = 16 * c + y;
              rise |= (x_of(r) > lim.x) | (x_of(r + 1) > lim.y) | (x_of(r + 2) > lim.z) |
                      (x_of(r + 3) > lim.w);
            }
          }
        if (any(rise)) {
          // The tile's maximum of every row, and what is summed so far brought down to it.
#pragma unroll
          for (int c = 0; c < (R + 31) / 32; ++c)
            if (col0 + 32 * c < here) {
              float x[32];
#pragma unroll
              for (int y = 0; y < 32; ++y) {
                const int r = 32 * c + y;
                x[y] = r < R && col0 + r / 16 * 16 < here ? x_of(r % R) : -INFINITY;
              }
              const float top = lanes_reduce<true>(x);
              if (32 * c + lane < R && col0 + 32 * c + lane < here)
                sh.red[quarter][col0 + 32 * c + lane] = top;
            }
          sync();
          for (int r = tid; r < q.here; r += SOFT) {
            const float old = sh.ref[r];
            const float top =
                fmaxf(fmaxf(sh.red[0][r], sh.red[1][r]), fmaxf(sh.red[2][r], sh.red[3][r]));
            const float ref = fmaxf(old, top * scale);
            sh.fac[r] = ref == -INFINITY ? 1.0f : ex2(old - ref);
            sh.ref[r] = ref;
            sh.base[r] = ref == -INFINITY ? 0.0f : ref;
            if (rows.out[r] >= 0) sh.lim[r] = (ref + TT_RISE) / scale;
          }
          sync();
          if (i > 0) {
            const int j = g - 1;
            mbar_wait_warp(&sh.pv_done[j & 1], (j >> 1) & 1, ab, kErrTimeoutConsumer);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < R / 16; ++c)
              if (col0 + 16 * c < here) {
                uint32_t o[16];
                __syncwarp();
                tmem_ld16(lanes + 2 * NR + 16 * c, o);
                tmem_wait_ld();
#pragma unroll
                for (int y = 0; y < 16; ++y) {
                  const float f = sh.fac[col0 + 16 * c + y];
                  o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                  l[16 * c + y] *= f;
                }
                tmem_st16(lanes + 2 * NR + 16 * c, o);
              }
            tmem_wait_st();
          }
        }
        // P is free once the product that read it is done.
        if (g >= T::kPBufs) {
          const int j = g - T::kPBufs;
          mbar_wait_warp(&sh.pv_done[j & 1], (j >> 1) & 1, ab, kErrTimeoutConsumer);
        }
        uint8_t *to = smem + T::kOffP + (g % T::kPBufs) * T::kParts * T::kP;
#pragma unroll
        for (int c = 0; c < R / 16; ++c)
          if (col0 + 16 * c < here) {
            uint32_t hi[8], low[8];
#pragma unroll
            for (int y = 0; y < 16; y += 4) {
              const float4 base = *reinterpret_cast<const float4 *>(&sh.base[col0 + 16 * c + y]);
              const int r = 16 * c + y;
              const float x0 = ex2(fmaf(x_of(r), scale, -base.x));
              const float x1 = ex2(fmaf(x_of(r + 1), scale, -base.y));
              const float x2 = ex2(fmaf(x_of(r + 2), scale, -base.z));
              const float x3 = ex2(fmaf(x_of(r + 3), scale, -base.w));
              l[r] += x0;
              l[r + 1] += x1;
              l[r + 2] += x2;
              l[r + 3] += x3;
              if constexpr (WIDE) {
                split2(x0, x1, hi[y / 2], low[y / 2]);
                split2(x2, x3, hi[y / 2 + 1], low[y / 2 + 1]);
              } else {
                hi[y / 2] = pack_half2(x0, x1);
                hi[y / 2 + 1] = pack_half2(x2, x3);
              }
            }
            const int cc = col0 / 16 + c;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint8_t *at = to + (cc >> 2) * TT_HALF + sw128_offset(key, 2 * (cc & 3) + y);
              *reinterpret_cast<uint4 *>(at) =
                  make_uint4(hi[4 * y], hi[4 * y + 1], hi[4 * y + 2], hi[4 * y + 3]);
              if constexpr (WIDE)
                *reinterpret_cast<uint4 *>(at + T::kP) =
                    make_uint4(low[4 * y], low[4 * y + 1], low[4 * y + 2], low[4 * y + 3]);
            }
          }
        // What a row does not see must not reach it through 0 times infinity: V is zero past the
        // end, and a drafted position's infinities and NaN are zeros here and added at the end to the
        // rows that see them.
        pv = g == n - 1 ? 2 * n - 1 : 2 * g + 2;
        if (!all && w < 4) {
          mbar_wait_warp(&sh.full[pv % D], (pv / D) & 1, ab, kErrTimeoutConsumer);
          uint8_t *v = smem + (pv % D) * T::kSlot;
          if (!there || d >= 0) {
            bool odd = false;
#pragma unroll 2
            for (int c = 0; c < HDP / 8; ++c) {
              uint4 *at = reinterpret_cast<uint4 *>(v + (c >> 3) * TT_HALF + sw128_offset(key, c & 7));
              const uint4 x = *at;
              uint4 y = make_uint4(0u, 0u, 0u, 0u);
              if (there) y = make_uint4(finite2(x.x), finite2(x.y), finite2(x.z), finite2(x.w));
              if (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w) {
                *at = y;
                odd = true;
              }
            }
            if (there && odd && d < 256) atomicOr(&sh.odd[d >> 5], 1u << (d & 31));
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[g & 1]);
      }

      // ---- the item's sums, and its rows out ---------------------------------------------------------
#pragma unroll
      for (int c = 0; c < (R + 31) / 32; ++c) {
        float x[32];
#pragma unroll
        for (int y = 0; y < 32; ++y) x[y] = 32 * c + y < R ? l[(32 * c + y) % R] : 0.0f;
        const float sum = lanes_reduce<false>(x);
        if (32 * c + lane < R && col0 + 32 * c + lane < here)
          sh.red[quarter][col0 + 32 * c + lane] = sum;
      }
      sync();
      for (int r = tid; r < q.here; r += SOFT) {
        const float sum = sh.red[0][r] + sh.red[1][r] + sh.red[2][r] + sh.red[3][r];
        sh.fac[r] = q.slot >= 0 ? 1.0f : sum != 0.0f ? 1.0f / sum : 0.0f;
        if (q.slot >= 0 && rows.out[r] >= 0)
          *reinterpret_cast<float2 *>(a.part + rows.out[r] + a.hd) = make_float2(sh.ref[r], sum);
      }
      ok = mbar_wait_warp(&sh.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, ab, kErrTimeoutConsumer);
      const bool good = !any(!ok || ab.raised());
      tc_fence_after();
      uint32_t odd = 0u;
#pragma unroll
      for (int x = 0; x < 8; ++x) odd |= sh.odd[x];
      const int dim = quarter * 32 + lane;  // the TMEM lane is the element of the head
      if (quarter * 32 < a.hd) {
#pragma unroll 1
        for (int c = 0; c < R / 16; ++c) {
          if (col0 + 16 * c >= here) break;
          uint32_t o[16];
          __syncwarp();
          tmem_ld16(lanes + 2 * NR + 16 * c, o);
          tmem_wait_ld();
          if (odd) {
            for (int d = 0; d < min(q.rows, 256); ++d) {
              if (!((sh.odd[d >> 5] >> (d & 31)) & 1u)) continue;
              const int pos = q.len + d, blk = table[pos / a.bs];
              const __half h = dim < a.hd ? a.pool[(((long long)blk * 2 + 1) * a.kv_heads + q.kvh) * a.bs * a.hd +
                                                   (long long)(pos % a.bs) * a.hd + dim]
                                          : __half(0.0f);
              if ((__half_as_ushort(h) & 0x7c00u) != 0x7c00u) continue;
#pragma unroll
              for (int y = 0; y < 16; ++y)
                if ((rows.mask[col0 + 16 * c + y][d >> 5] >> (d & 31)) & 1u)
                  o[y] = __float_as_uint(__uint_as_float(o[y]) + __half2float(h));
            }
          }
          long long at[16];
#pragma unroll
          for (int y = 0; y < 16; ++y) at[y] = good && dim < a.hd ? rows.out[col0 + 16 * c + y] : -1;
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            const float v = __uint_as_float(o[y]) * sh.fac[col0 + 16 * c + y];
            if (at[y] >= 0) {
              if (q.slot < 0) static_cast<E *>(a.o)[at[y] + dim] = E(v);
              else a.part[at[y] + dim] = v;
            }
          }
        }
      }
      if (q.slot >= 0) {
        // The run that brings the last part of an item joins them all.
        __threadfence();
        sync();
        if (tid == 0) sh.last = atomicAdd(&a.count[q.first], 1) == q.parts - 1;
        sync();
        if (sh.last && good) {
          __threadfence();
          const auto part_of = [&](int x, int r) {
            const long long slot = 2ll * (q.first + x) + (x == 0 ? 1 : 0);
            return a.part + (slot * NR + r) * (a.hd + 4);
          };
          for (int r = tid; r < q.here; r += SOFT) {
            float top = -INFINITY, sum = 0.0f;
            for (int x = 0; x < q.parts; ++x) top = fmaxf(top, __ldcg(part_of(x, r) + a.hd));
            const float base = top == -INFINITY ? 0.0f : top;
            for (int x = 0; x < q.parts; ++x) {
              const float2 ml = __ldcg(reinterpret_cast<const float2 *>(part_of(x, r) + a.hd));
              sum = fmaf(ex2(ml.x - base), ml.y, sum);
            }
            sh.base[r] = base;
            sh.fac[r] = sum != 0.0f ? 1.0f / sum : 0.0f;
          }
          sync();
          const int quads = a.hd / 4;
          for (int e = tid; e < q.here * quads; e += SOFT) {
            const int r = e / quads, c = (e - r * quads) * 4;
            const int row = q.lo + (q.r0 + r) / group, head = q.kvh * group + (q.r0 + r) % group;
            if (row >= a.rows) continue;
            const float base = sh.base[r], inv = sh.fac[r];
            float o[4] = {};
#pragma unroll 4
            for (int x = 0; x < q.parts; ++x) {
              const float *from = part_of(x, r);
              const float f = ex2(__ldcg(from + a.hd) - base);
              const float4 v = __ldcg(reinterpret_cast<const float4 *>(from + c));
              o[0] = fmaf(f, v.x, o[0]);
              o[1] = fmaf(f, v.y, o[1]);
              o[2] = fmaf(f, v.z, o[2]);
              o[3] = fmaf(f, v.w, o[3]);
            }
            E *to = static_cast<E *>(a.o) + row * a.o_stride + (long long)head * a.hd + c;
#pragma unroll
            for (int x = 0; x < 4; ++x) to[x] = E(o[x] * inv);
          }
          if (tid == 0) a.count[q.first] = 0;  // for the next call
        }
      }
      sync();  // the rows and references are read, the item's place is free
      if (odd && tid < 8) sh.odd[tid] = 0u;
      tc_fence_before();
      if (tid == 0) mbar_arrive(&sh.piece_empty[pc]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (w == W_MMA) tmem_dealloc(tmem, T::kCols);
}

template <int HDP, int NR, bool WIDE>
cudaError_t launch_tile(const CUtensorMap &map, const AttendTreeArgs &a, int sms, cudaStream_t s) {
  auto *kernel = attend_tree_kernel<HDP, NR, WIDE>;
  using T = TreeTile<HDP, NR, WIDE>;
  constexpr size_t smem = T::kOffBar + sizeof(TreeShared<NR>) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory");
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !configured[dev]) {
    cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    if (dev < 64) configured[dev] = true;
  }
  // No more runs than there can be tiles.
  const long long items =
      ((long long)a.max_rows * (a.heads / a.kv_heads) + NR - 1) / NR * a.kv_heads * a.n;
  const long long tiles = items * std::max((a.max_len + TT_KEYS - 1) / TT_KEYS, 1);
  const int grid = int(std::min<long long>((long long)sms * T::kCtas, tiles));
  return launch_pdl(kernel, dim3(grid), dim3(T::kThreads), smem, s, map, a);
}

template <int HDP>
cudaError_t launch_rows(const CUtensorMap &map, const AttendTreeArgs &a, int f16, int sms,
                        cudaStream_t s) {
  switch (attend_tree_rows(a.max_rows, a.heads, a.kv_heads, f16)) {
    case 16:
      return f16 ? launch_tile<HDP, 16, false>(map, a, sms, s) : launch_tile<HDP, 16, true>(map, a, sms, s);
    case 32:
      return f16 ? launch_tile<HDP, 32, false>(map, a, sms, s) : launch_tile<HDP, 32, true>(map, a, sms, s);
    case 64:
      return f16 ? launch_tile<HDP, 64, false>(map, a, sms, s) : launch_tile<HDP, 64, true>(map, a, sms, s);
    default:
      return launch_tile<HDP, 128, false>(map, a, sms, s);
  }
}

}  // namespace

bool attend_tree_few(int max_rows, int heads, int kv_heads, int f16) {
  return (long long)max_rows * (heads / kv_heads) <= 64;
}

int attend_tree_rows(int max_rows, int heads, int kv_heads, int f16) {
  const long long rows = (long long)max_rows * (heads / kv_heads);
  return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 || !f16 ? 64 : 128;
}

size_t attend_tree_part_bytes(int max_rows, int heads, int kv_heads, int hd, int f16, int sms) {
  // Two parts a run: of the item that it begins in, and of the one that it ends in.
  return size_t(2) * kTreeRunsPerSm * sms * attend_tree_rows(max_rows, heads, kv_heads, f16) *
         (hd + 4) * sizeof(float);
}

cudaError_t launch_attend_tree(const CUtensorMap &map, const AttendTreeArgs &a, int f16, int sms,
                               cudaStream_t s) {
  if (a.n <= 0 || a.max_rows <= 0) return cudaSuccess;
  return a.hd <= 64 ? launch_rows<64>(map, a, f16, sms, s) : launch_rows<128>(map, a, f16, sms, s);
}

}  // namespace wv
