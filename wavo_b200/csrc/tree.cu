// Attention of drafted tokens over a paged KV cache (the pool of paged.cu).
//
// Row i of a request sees its len cached positions and, with a mask, those of the rows drafted with
// it whose bits its mask words hold (row j's K and V are at position len + j). o = softmax(q.k /
// sqrt(hd)) v over what it sees, zeros where it sees nothing.
//
// This is the form for many rows (tree_few.cu has the one for few). One pass over K and V with a
// running softmax. An item is one K and V head of one request with up to 128 rows that read it (its
// drafted rows and the heads that share it); the rows are the UMMA's M and 128 positions its N,
//   S [128 x 128] = Q [128 x hd] . K^T,   O [128 x hd] += P [128 x 128] . V,
// S and O in tensor memory and P there over the S that it came from. Two threads of a warp have a
// row's scores of a tile, so its maximum takes one shuffle, and warps without rows do nothing. A
// row's reference value rises when a score is 4 (base 2) above the one that set it: at an item's
// first tile and seldom after, so O is seldom rescaled. The largest probability is then 2^11 to 2^15
// where it is rounded to f16 (see kLift).
//
// The items' tiles of 128 positions lie one after another and are cut into equal runs, one a CTA,
// as many CTAs as are resident: ragged lengths, few long requests and many short ones fill the GPU
// alike, and the loads run ahead across the items of a run. A run that ends inside an item leaves
// its part in global memory, and a second kernel joins an item's parts in the order of the runs.
//
// Two requests of up to 131072 positions, 8 K and V heads of 128 and up to 96 rows each (685 MB, 53
// GFLOP): a pass by itself 144 us and 9 for the join, 4.5 TB/s; among other passes, at the clocks that
// the power limit leaves, 166 us in all, 4.1 TB/s. The loads alone, in the same runs, took 137 to
// 157. A tile costs the softmax warps about 2300 cycles (the exponentials 770 of them) and its 64 KB
// an SM's share of the memory 2800; at the lower clocks the two are close.
// Positions as the UMMA's M and the rows as its N (P through shared memory, a vote of all warps a
// tile) took 215 us, the join by the last CTA alone 57 more.
#include <algorithm>
#include <type_traits>

#include "softmax.cuh"
#include "tree.cuh"

namespace wv {
namespace {

constexpr int TT_KEYS = 128;                  // positions a tile
constexpr uint32_t TT_HALF = TT_KEYS * 128;   // bytes of 128 positions x 64 elements
constexpr int TT_ROWS = 128;                  // rows of an item
constexpr int TT_RISE = 4;
constexpr int TT_LIFT = kLift - TT_RISE;      // log2 of the probability of a reference
constexpr int TT_PIECES = 3;                  // items in flight: loaded, multiplied, written
constexpr int TT_WHOLE = 4;                   // items of up to this many tiles stay in one run

// HDP: head size padded to 64 or 128. WIDE: f32 rows, as two f16 parts each.
template <int HDP, bool WIDE>
struct TreeTile {
  static constexpr int kParts = WIDE ? 2 : 1;
  static constexpr uint32_t kSlot = (HDP / 64) * TT_HALF;           // a tile of K or of V
  static constexpr uint32_t kQ = (HDP / 64) * TT_HALF;              // Q, one part
  static constexpr int kQBufs = kParts * kQ > 16384 ? 1 : 2;
  static constexpr int kRing = HDP == 64 ? 8 : WIDE ? 4 : 5;
  static_assert(kRing >= 4, "the softmax's wait for V");
  static constexpr uint32_t kOffQ = kRing * kSlot;
  static constexpr uint32_t kOffBar = kOffQ + kQBufs * kParts * kQ;
  // TMEM: S and P twice, then O; f32's low parts sum apart (they are scaled, and each step of a long
  // sum drops bits of its size), and join at the end.
  static constexpr uint32_t kColO = 256;
};
constexpr int TT_SOFT = 256;                                        // softmax threads
constexpr int TT_THREADS = TT_SOFT + 96;                            // and loads, UMMAs, rows

// A run's share of an item.
struct TreePiece {
  int s, kvh, r0, here;     // request, K and V head, first row, rows
  int lo, rows;             // the request's first row, its drafted rows
  int len, keys;            // its positions without and with them
  int tile0, tiles;         // tiles of the item
  int slot;                 // where a partial result goes; -1: the item is whole
};

struct TreeRows {
  long long out[TT_ROWS];   // element offset of the row's output, -1: none
  uint32_t mask[TT_ROWS][8];
};

struct TreeShared {
  uint64_t full[8], empty[8], s_full[2], p_full[2], pv_done[2], q_full[2], q_empty[2], info_full[8];
  uint64_t piece_full[TT_PIECES], piece_empty[TT_PIECES], row_full[TT_PIECES], drain;
  TreePiece piece[TT_PIECES];
  TreeRows rows[TT_PIECES];
  uint32_t info[8];             // of a tile: bit b: box b is in the pool; bit 31: every row sees it all
  uint32_t tmem, abort;
  uint32_t odd[8];              // drafted positions whose V holds an infinity or NaN
  long long scan[12], begin, end;
  int begin_s, begin_n;         // the run's first request and the tiles of it that lie before
  long long q_at[TT_ROWS];      // element offsets of the rows in q, -1: none
};

// What an item's size follows from. A request without positions has one (empty) tile an item, which
// gives its rows their zeros.
struct TreeRequest {
  int lo, rows, len, keys;
  int row_tiles, tiles;  // items a K and V head; tiles an item
};

__device__ __forceinline__ TreeRequest tree_request(const AttendTreeArgs &a, int s) {
  TreeRequest r;
  r.lo = a.row_start ? a.row_start[s] : s;
  r.rows = min(a.row_start ? a.row_start[s + 1] - r.lo : 1, a.max_rows);
  if (r.lo < 0 || r.rows < 0) r.rows = 0;
  r.len = max(a.lens[s], 0);
  r.keys = int(min((long long)r.len + (a.mask ? r.rows : 0), (long long)a.max_len));
  r.row_tiles = (r.rows * (a.heads / a.kv_heads) + TT_ROWS - 1) / TT_ROWS;
  r.tiles = max((r.keys + TT_KEYS - 1) / TT_KEYS, 1);
  return r;
}

template <int HDP, bool WIDE>
__global__ void __launch_bounds__(TT_THREADS, 1)
    attend_tree_kernel(const __grid_constant__ CUtensorMap map, const AttendTreeArgs a) {
  using T = TreeTile<HDP, WIDE>;
  using E = typename std::conditional<WIDE, float, __half>::type;
  constexpr int D = T::kRing, SOFT = TT_SOFT;
  constexpr int W_LOAD = SOFT / 32, W_MMA = W_LOAD + 1, W_ROWS = W_LOAD + 2, WARPS = W_LOAD + 3;
  extern __shared__ uint8_t raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                              ~uintptr_t(1023));
  TreeShared &sh = *reinterpret_cast<TreeShared *>(smem + T::kOffBar);
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
    for (int i = 0; i < 8; ++i) mbar_init(&sh.info_full[i], 1);
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
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  const uint32_t tmem = sh.tmem;

  // ---- this CTA's run: tiles begin .. end of all ---------------------------------------------------
  const int per = (a.n + TT_THREADS - 1) / TT_THREADS;
  const int s_lo = min(tid * per, a.n), s_hi = min(s_lo + per, a.n);
  long long mine = 0;
  for (int s = s_lo; s < s_hi; ++s) {
    const TreeRequest r = tree_request(a, s);
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
        TreeRequest r = tree_request(a, s);
        long long all = (long long)r.row_tiles * a.kv_heads * r.tiles;
        while (left >= all) {
          left -= all;
          r = tree_request(a, ++s);
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
      r = tree_request(a, s);
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
    TreeJoin join = {};  // the item that this run begins and does not end
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
            q.r0 = (item - kvh * r.row_tiles) * TT_ROWS;
            q.here = min(r.rows * group - q.r0, TT_ROWS);
            q.lo = r.lo;
            q.rows = r.rows;
            q.len = r.len;
            q.keys = r.keys;
            q.tile0 = tile;
            q.tiles = min(r.tiles - tile, n - g);
            q.slot = -1;
            if (q.tiles < r.tiles) {
              q.slot = 2 * int(blockIdx.x) + (tile == 0 ? 1 : 0);
              if (tile == 0) {
                // Run c holds tile x where c = ((x + 1) runs - 1) / total, rounded down.
                const long long x1 = sh.begin + g + r.tiles - 1;
                join = {q.lo, q.r0, q.here, kvh, int(((x1 + 1) * runs - 1) / total) - int(blockIdx.x) + 1};
              }
            }
            sh.piece[k % TT_PIECES] = q;
            mbar_arrive(&sh.piece_full[k % TT_PIECES]);
          }
          ++k;
          fresh = false;
          ahead = false;
        }
        z = ahead ? z_next : block_of(tile);
        const uint32_t in = __ballot_sync(0xffffffffu, z < a.blocks) & ((1u << boxes) - 1u);
        if (lane == 0) {
          // (The softmax is past tile g - 8: the ring holds fewer tiles than that.)
          const bool all = in == (1u << boxes) - 1u && (tile + 1) * TT_KEYS <= min(r.len, r.keys);
          sh.info[g & 7] = in | (all ? 1u << 31 : 0u);
          mbar_arrive(&sh.info_full[g & 7]);
        }
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
    if (lane == 0) a.joins[blockIdx.x] = join;
    // The shared memory stays until the last loads have landed, also where a wait gave up.
    for (int q = max(p - D, 0); q < p; ++q)
      for (int i = 0; i < 2000 && !mbar_try_wait_sleep(&sh.full[q % D], (q / D) & 1, 100000u); ++i) {}
  } else if (w == W_MMA) {
    // ---- UMMAs: S of a tile, then P.V of the one before it ---------------------------------------
    if (lane == 0 && n > 0) {
      const uint64_t dq = sdesc_sw128(smem_u32(smem + T::kOffQ), 16, 1024);
      const uint64_t dk = sdesc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t dv = sdesc_sw128(smem_u32(smem), TT_HALF, 1024);
      constexpr uint32_t id_s = idesc_f16(TT_ROWS, TT_KEYS, 0), id_o = idesc_f16(TT_ROWS, HDP, 1);
      int p = 0, k = -1, left = 0;
      bool first = false, first_v = false, ok = true;
      for (int g = 0; g <= n; ++g) {
        first_v = first;
        if (g < n) {
          first = left == 0;
          if (first) {
            ++k;
            if (!mbar_wait(&sh.piece_full[k % TT_PIECES], (k / TT_PIECES) & 1, ab, kErrTimeoutMma))
              break;
            left = sh.piece[k % TT_PIECES].tiles;
            if (!mbar_wait(&sh.q_full[k % T::kQBufs], (k / T::kQBufs) & 1, ab, kErrTimeoutMma)) break;
          }
          const int slot = p % D;
          if (!mbar_wait(&sh.full[slot], (p / D) & 1, ab, kErrTimeoutMma)) break;
          // S lies over the P of two tiles before.
          if (g >= 2 && !mbar_wait(&sh.pv_done[g & 1], ((g - 2) >> 1) & 1, ab, kErrTimeoutMma)) break;
          ++p;
          tc_fence_after();
          const uint64_t kd = dk + uint64_t(slot * T::kSlot >> 4);
          const uint64_t qd = dq + uint64_t((k % T::kQBufs) * T::kParts * T::kQ >> 4);
          // The low parts first: the sums are small until the high ones come, and so is what a step
          // drops.
#pragma unroll
          for (int part = T::kParts - 1; part >= 0; --part)
#pragma unroll
            for (int kk = 0; kk < HDP / 16; ++kk)
              umma_f16(tmem + (g & 1) * 128,
                       qd + ((part * T::kQ + (kk >> 2) * TT_HALF + (kk & 3) * 32) >> 4),
                       kd + (((kk >> 2) * TT_HALF + (kk & 3) * 32) >> 4), id_s,
                       part < T::kParts - 1 || kk > 0 ? 1u : 0u);
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
          const uint64_t vd = dv + uint64_t(slot * T::kSlot >> 4);
          // P over S: f16 pairs, 8 columns a step of 16 positions, the second part 64 columns on.
#pragma unroll
          for (int part = 0; part < T::kParts; ++part)
#pragma unroll
            for (int kk = 0; kk < TT_KEYS / 16; ++kk)
              umma_f16_ts(tmem + T::kColO + part * HDP, tmem + (j & 1) * 128 + part * 64 + kk * 8,
                          vd + uint64_t(kk * 16 * 128 >> 4), id_o, !first_v || kk > 0 ? 1u : 0u);
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
      TreeRows &to = sh.rows[pc];
      done += q.tiles;
      for (int r = lane; r < TT_ROWS; r += 32) {
        const int i = (q.r0 + r) / group, head = q.kvh * group + (q.r0 + r) - i * group;
        const bool live = r < q.here && q.lo + i < a.rows;
        const long long row = q.lo + i;
        sh.q_at[r] = live ? row * a.q_stride + (long long)head * a.hd : -1;
        to.out[r] = !live ? -1
                    : q.slot < 0 ? row * a.o_stride + (long long)head * a.hd
                                 : ((long long)q.slot * TT_ROWS + r) * (a.hd + 4);
        for (int x = 0; x < a.words; ++x)
          to.mask[r][x] = live ? a.mask[row * a.words + x] : 0u;
      }
      if (k >= T::kQBufs &&
          !mbar_wait_warp(&sh.q_empty[qb], (k / T::kQBufs - 1) & 1, ab, kErrTimeoutConsumer))
        break;
      uint8_t *base = smem + T::kOffQ + qb * T::kParts * T::kQ;
      __syncwarp();
      // Eight elements a lane and step; rows to the next 16 are zeros.
      const int chunks = (q.here + 15) / 16 * 16 * (HDP / 8);
      const auto source = [&](int e) -> const E * {
        const int c = e % (HDP / 8);
        const long long at = e < chunks ? sh.q_at[e / (HDP / 8)] : -1;
        return at < 0 || c * 8 >= a.hd ? nullptr : static_cast<const E *>(a.q) + at + c * 8;
      };
      const auto target = [&](int e) {
        const int r = e / (HDP / 8), c = e % (HDP / 8);
        return base + (c >> 3) * TT_HALF + sw128_offset(r, c & 7);
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
    // ---- softmax: 16 rows a warp, threads t and t + 16 the halves of a row's positions -------------
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
    const int first_row = (w & 3) * 32 + (w >> 2) * 16, row = first_row + (lane & 15), half = lane >> 4;
    const uint32_t lanes = tmem + (uint32_t(first_row) << 16);
    const float scale = a.scale * 1.4426950408889634f;  // exponentials of base 2
    for (int k = 0, g = 0; g < n; ++k) {
      const int pc = k % TT_PIECES;
      // Where a wait gives up, all warps leave together; inside an item they run on (later waits
      // give up soon).
      bool ok = mbar_wait_warp(&sh.row_full[pc], (k / TT_PIECES) & 1, ab, kErrTimeoutConsumer);
      if (any(!ok)) break;
      const TreePiece &q = sh.piece[pc];
      const TreeRows &rows = sh.rows[pc];
      const bool work = first_row < q.here;
      const int tiles = q.tiles;
      float m = -INFINITY, l0 = 0.0f, l1 = 0.0f;
      for (int i = 0; i < tiles; ++i, ++g) {
        mbar_wait_warp(&sh.info_full[g & 7], (g >> 3) & 1, ab, kErrTimeoutConsumer);
        const uint32_t info = sh.info[g & 7];
        const bool all = info >> 31;  // every row sees the whole tile
        const int pos0 = (q.tile0 + i) * TT_KEYS;
        mbar_wait_warp(&sh.s_full[g & 1], (g >> 1) & 1, ab, kErrTimeoutConsumer);
        tc_fence_after();
        if (!all && tid < TT_KEYS) {
          // What a row does not see must not reach it through 0 times infinity: V is zero past the
          // end, and a drafted position's infinities and NaN are zeros here and added at the end to
          // the rows that see them. (After S of this tile, and so after P.V of two tiles before: in a
          // ring of four that V lies in this one's place, and a wait by parity that starts before it
          // has landed is let through at once.)
          const int p = g == n - 1 ? 2 * n - 1 : 2 * g + 2, pos = pos0 + tid, d = pos - q.len;
          mbar_wait_warp(&sh.full[p % D], (p / D) & 1, ab, kErrTimeoutConsumer);
          const bool there = pos < q.keys && ((info >> (tid / min(a.bs, TT_KEYS))) & 1u);
          uint8_t *v = smem + (p % D) * T::kSlot;
          if (!there || d >= 0) {
            bool odd = false;
#pragma unroll 2
            for (int c = 0; c < HDP / 8; ++c) {
              uint4 *at = reinterpret_cast<uint4 *>(v + (c >> 3) * TT_HALF + sw128_offset(tid, c & 7));
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
          fence_proxy_async_smem();
        }
        if (work) {
          float x[64];
          {
            uint32_t u[32], v[32];
            __syncwarp();
            tmem_ld_16x2_x32<64>(lanes + (g & 1) * 128, u);
            tmem_ld_16x2_x32<64>(lanes + (g & 1) * 128 + 32, v);
            tmem_wait_ld();
#pragma unroll
            for (int y = 0; y < 32; ++y) {
              x[y] = __uint_as_float(u[y]);
              x[32 + y] = __uint_as_float(v[y]);
            }
          }
          if (!all) {
            const auto word = [&](int y) { return y < a.words ? rows.mask[row][y] : 0u; };
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              // 32 positions from p on, d of the drafted: a bit each.
              const int at = 64 * half + 32 * c, p = pos0 + at, d = p - q.len;
              uint32_t see = ~0u;
              if (d >= 0) see = __funnelshift_r(word(d >> 5), word((d >> 5) + 1), d & 31);
              else if (d > -32) see = (word(0) << -d) | ((1u << -d) - 1u);
              if (q.keys - p < 32) see = q.keys > p ? see & ((1u << (q.keys - p)) - 1u) : 0u;
              const int box = min(a.bs, TT_KEYS);
#pragma unroll
              for (int y = 0; y < 4; ++y)
                if (!((info >> ((at + 8 * y) / box)) & 1u)) see &= ~(0xffu << (8 * y));
#pragma unroll
              for (int y = 0; y < 32; ++y)
                if (!((see >> y) & 1u)) x[32 * c + y] = -INFINITY;
            }
          }
          float top = -INFINITY;
          {
            float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int y = 0; y < 64; y += 8) {
              float &t = t4[(y / 8) & 3];
              t = max3(t, x[y], x[y + 1]);
              t = max3(t, x[y + 2], x[y + 3]);
              t = max3(t, x[y + 4], x[y + 5]);
              t = max3(t, x[y + 6], x[y + 7]);
            }
            top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
            // The reference it would set, rounded up: what it stands for is at most 2^TT_LIFT.
            top = __fmaf_ru(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)), scale,
                            WIDE ? 0.0f : -float(TT_LIFT));
          }
          const bool rise = top > __fadd_rd(m, float(TT_RISE));  // (-inf + 4 at the first score)
          const float fac = rise ? ex2(m - top) : 1.0f;
          if (__any_sync(0xffffffffu, rise)) {
            l0 *= fac;
            l1 *= fac;
            if (rise) m = top;
            if (i > 0) {
              const int j = g - 1;
              mbar_wait_warp(&sh.pv_done[j & 1], (j >> 1) & 1, ab, kErrTimeoutConsumer);
              tc_fence_after();
#pragma unroll 1
              for (int part = 0; part < T::kParts; ++part)
#pragma unroll 1
                for (int c = 0; c < HDP / 2; c += 16) {
                  const uint32_t at = lanes + T::kColO + part * HDP + c;
                  uint32_t o[16];
                  tmem_ld_16x2_x16<HDP / 2>(at, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * fac);
                  tmem_st_16x2_x16<HDP / 2>(at, o);
                }
            }
          }
          const float base = m == -INFINITY ? 0.0f : -m;
          uint32_t hi[32];
#pragma unroll
          for (int y = 0; y < 64; y += 4) {
            fma2(x[y], x[y + 1], x[y], x[y + 1], scale, scale, base, base);
            fma2(x[y + 2], x[y + 3], x[y + 2], x[y + 3], scale, scale, base, base);
#pragma unroll
            for (int z = y; z < y + 4; ++z) x[z] = ex2(x[z]);
            float s0, s1;
            add2(s0, s1, x[y], x[y + 1], x[y + 2], x[y + 3]);
            add2(l0, l1, l0, l1, s0, s1);
            if constexpr (!WIDE) {
              hi[y / 2] = pack_half2(x[y], x[y + 1]);
              hi[y / 2 + 1] = pack_half2(x[y + 2], x[y + 3]);
            }
          }
          if constexpr (WIDE) {
            uint32_t low[32];
#pragma unroll
            for (int y = 0; y < 32; ++y) split2_up<TT_LIFT>(x[2 * y], x[2 * y + 1], hi[y], low[y]);
            tmem_st_16x2_x32<32>(lanes + (g & 1) * 128 + 64, low);
          }
          tmem_st_16x2_x32<32>(lanes + (g & 1) * 128, hi);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[g & 1]);
      }

      // ---- the item's sums, and its rows out ---------------------------------------------------------
      ok = mbar_wait_warp(&sh.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, ab, kErrTimeoutConsumer);
      const bool good = !any(!ok || ab.raised());
      tc_fence_after();
      uint32_t odd = 0u;
#pragma unroll
      for (int x = 0; x < 8; ++x) odd |= sh.odd[x];
      if (work) {
        float sum = l0 + l1;
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const float fac = q.slot >= 0 ? 1.0f : sum != 0.0f ? 1.0f / sum : 0.0f;
        const long long at = good ? rows.out[row] : -1;
        if (q.slot >= 0 && at >= 0 && half == 0)
          *reinterpret_cast<float2 *>(a.part + at + a.hd) = make_float2(m, sum);
        const bool vec =
            ((reinterpret_cast<uintptr_t>(a.o) | (a.o_stride * sizeof(E))) & 15u) == 0;
#pragma unroll 1
        for (int c = 0; c < HDP / 2; c += 16) {
          const int dim = half * (HDP / 2) + c;
          uint32_t u[16];
          __syncwarp();
          tmem_ld_16x2_x16<HDP / 2>(lanes + T::kColO + c, u);
          tmem_wait_ld();
          float o[16];
#pragma unroll
          for (int y = 0; y < 16; ++y) o[y] = __uint_as_float(u[y]);
          if constexpr (WIDE) {
            tmem_ld_16x2_x16<HDP / 2>(lanes + T::kColO + HDP + c, u);
            tmem_wait_ld();
#pragma unroll
            for (int y = 0; y < 16; ++y)
              o[y] = fmaf(__uint_as_float(u[y]), 1.0f / kLowUp, o[y]) * (1.0f / (1 << TT_LIFT));
          }
          if (odd && at >= 0) {
            const int *table = a.table + (long long)q.s * a.width;
            for (int d = 0; d < min(q.rows, 256); ++d) {
              if (!((sh.odd[d >> 5] & rows.mask[row][d >> 5]) >> (d & 31) & 1u)) continue;
              const int pos = q.len + d, blk = table[pos / a.bs];
              const __half *v = a.pool + (((long long)blk * 2 + 1) * a.kv_heads + q.kvh) * a.bs * a.hd +
                                (long long)(pos % a.bs) * a.hd + dim;
              for (int y = 0; y < 16; ++y)
                if (dim + y < a.hd && (__half_as_ushort(v[y]) & 0x7c00u) == 0x7c00u)
#pragma unroll
                  for (int z = 0; z < 16; ++z)
                    if (z == y) o[z] += __half2float(v[y]);
            }
          }
#pragma unroll
          for (int y = 0; y < 16; y += 8) {
            if (at < 0 || dim + y >= a.hd) break;  // hd is a multiple of 8
            if (q.slot >= 0) {
              float *to = a.part + at + dim + y;
              *reinterpret_cast<float4 *>(to) = make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]);
              *reinterpret_cast<float4 *>(to + 4) = make_float4(o[y + 4], o[y + 5], o[y + 6], o[y + 7]);
            } else {
              E v[8];
#pragma unroll
              for (int z = 0; z < 8; ++z) v[z] = E(o[y + z] * fac);
              E *to = static_cast<E *>(a.o) + at + dim + y;
              if (vec) {
#pragma unroll
                for (int z = 0; z < int(sizeof(E)) / 2; ++z)
                  reinterpret_cast<uint4 *>(to)[z] = reinterpret_cast<const uint4 *>(v)[z];
              } else {
#pragma unroll
                for (int z = 0; z < 8; ++z) to[z] = v[z];
              }
            }
          }
        }
      }
      sync();  // the rows are read, the item's place is free
      if (odd && tid < 8) sh.odd[tid] = 0u;
      tc_fence_before();
      if (tid == 0) mbar_arrive(&sh.piece_empty[pc]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (w == W_MMA) tmem_dealloc(tmem, 512);
}

// The parts of an item joined: CTA (c, y) takes 8 of the rows of the item that run c begins, if
// that run does not end it. Four elements a thread.
constexpr int TT_JOIN = 8;

template <typename E>
__global__ void __launch_bounds__(TT_JOIN * 32) attend_tree_join_kernel(const AttendTreeArgs a) {
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  const int c = int(blockIdx.x), lane = int(threadIdx.x) & 31;
  const TreeJoin q = a.joins[c];
  const int r = int(blockIdx.y) * TT_JOIN + int(threadIdx.x >> 5);
  if (q.parts < 2 || r >= q.here) return;
  const int group = a.heads / a.kv_heads, i = (q.r0 + r) / group;
  const int row = q.lo + i, head = q.kvh * group + (q.r0 + r) - i * group;
  if (row >= a.rows) return;
  const auto part_of = [&](int x) {
    return a.part + ((2ll * (c + x) + (x == 0 ? 1 : 0)) * TT_ROWS + r) * (a.hd + 4);
  };
  // A lane a part for the reference and the sum, then a lane four elements.
  float top = -INFINITY, sum = 0.0f;
  for (int x = lane; x < q.parts; x += 32) {
    const float2 ml = *reinterpret_cast<const float2 *>(part_of(x) + a.hd);
    const float m = fmaxf(top, ml.x), base = m == -INFINITY ? 0.0f : m;
    sum = sum * ex2(top - base) + ml.y * ex2(ml.x - base);
    top = m;
  }
  float all = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
  const float base = all == -INFINITY ? 0.0f : all;
  sum *= ex2(top - base);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (4 * lane >= a.hd) return;
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
  float o[4] = {};
#pragma unroll 8
  for (int x = 0; x < q.parts; ++x) {
    const float f = ex2(part_of(x)[a.hd] - base);
    const float4 v = *reinterpret_cast<const float4 *>(part_of(x) + 4 * lane);
    o[0] = fmaf(f, v.x, o[0]);
    o[1] = fmaf(f, v.y, o[1]);
    o[2] = fmaf(f, v.z, o[2]);
    o[3] = fmaf(f, v.w, o[3]);
  }
  E *to = static_cast<E *>(a.o) + row * a.o_stride + (long long)head * a.hd + 4 * lane;
#pragma unroll
  for (int x = 0; x < 4; ++x) to[x] = E(o[x] * inv);
}

template <int HDP, bool WIDE>
cudaError_t launch_tile(const CUtensorMap &map, const AttendTreeArgs &a, int sms, cudaStream_t s) {
  auto *kernel = attend_tree_kernel<HDP, WIDE>;
  constexpr size_t smem = TreeTile<HDP, WIDE>::kOffBar + sizeof(TreeShared) + 1024;
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
      ((long long)a.max_rows * (a.heads / a.kv_heads) + TT_ROWS - 1) / TT_ROWS * a.kv_heads * a.n;
  const long long tiles = items * std::max((a.max_len + TT_KEYS - 1) / TT_KEYS, 1);
  const int grid = int(std::min<long long>(sms, tiles));
  const cudaError_t e = launch_pdl(kernel, dim3(grid), dim3(TT_THREADS), smem, s, map, a);
  if (e != cudaSuccess || a.max_len <= TT_WHOLE * TT_KEYS) return e;  // no item spans two runs
  return launch_pdl(attend_tree_join_kernel<typename std::conditional<WIDE, float, __half>::type>,
                    dim3(grid, TT_ROWS / TT_JOIN), dim3(TT_JOIN * 32), 0, s, a);
}

}  // namespace

// Measured on both sides, us few : many, f16 and f32, all requests with that many rows of a K and V
// head and no mask. Long: 2 x 16384 positions, 8 K and V heads of 128: 32 rows 51 : 47, 58 : 57; 48
// rows 53 : 49, 78 : 63; 96 rows 70 : 55, 104 : 80; heads of 64: 32 rows 39 : 37, 43 : 43; 48 rows
// 39 : 37, 51 : 47. 32 x 1500, 20 heads of 64: 48 rows 104 : 90, 137 : 131; 96 rows 141 : 106,
// 202 : 164. Trees of 1 to that many rows bring less work to CTAs of 32 rows, and the border lies
// higher: 32 x 1500, 48 rows 86 : 94, 104 : 126; 96 rows 123 : 109, 174 : 167; 32 x 512, 8 heads of 128:
// 64 rows 47 : 47, 63 : 68; 128 rows 74 : 68, 84 : 97; 192 rows 74 : 72, 115 : 113; 20 heads of 64: 96
// rows 68 : 66, 96 : 112. The rule lies between the two: the host does not know the trees.
bool attend_tree_few(int max_rows, int max_len, int heads, int kv_heads) {
  const long long rows = (long long)max_rows * (heads / kv_heads);
  return rows <= 32 || (rows <= 128 && max_len < 1280);
}

size_t attend_tree_part_bytes(int hd, int sms) {
  // Two parts a run: of the item that it begins in, and of the one that it ends in; and its join.
  return size_t(2) * sms * TT_ROWS * (hd + 4) * sizeof(float) + sms * sizeof(TreeJoin);
}

cudaError_t launch_attend_tree(const CUtensorMap &map, const AttendTreeArgs &a, int f16, int sms,
                               cudaStream_t s) {
  if (a.n <= 0 || a.max_rows <= 0) return cudaSuccess;
  if (a.hd <= 64)
    return f16 ? launch_tile<64, false>(map, a, sms, s) : launch_tile<64, true>(map, a, sms, s);
  return f16 ? launch_tile<128, false>(map, a, sms, s) : launch_tile<128, true>(map, a, sms, s);
}

}  // namespace wv
