// attend_tree for few rows: an item is one K and V head of one request with the rows that read it
// (its drafted rows and the heads that share it), 32 at most in a CTA. The steps from a tile's
// arrival to its sums are then short and the tiles of a request few, so what counts is how many of
// them are under way at once: mma.sync with the scores, probabilities and sums in registers, no tensor
// memory, no hand-over between warps, and 2 to 5 CTAs an SM. (The f32 forms spill 8 to 17 words a
// thread for that many.) The form with tcgen05 (tree.cu) takes over where the products would bound
// it; the figures of both are beside the rule there.
//
// One pass over K and V with the softmax's running maximum and sum: a CTA takes an item's rows over
// a range of positions. A producer warp loads 64 positions at a time, page by page, through TMA
// boxes that follow the block table; four warps multiply, 16 rows each: they share a tile's
// positions, and meet in shared memory at the end.
//
// Bound by the loads: 32 x 20 items of 16 rows over 1500 positions (246 MB, f16) take 48 us, 5.2
// TB/s; the same loads without the products took 54 us in CTAs of their own. One f32 row an item
// over 448 positions at most (34 MB) 19 us, of which launch and the first page's way (row starts,
// table, K) are most. Up to 64 f32 rows an item over 448 positions (two products each way) 48 us,
// bound by the latency of 16 warps an SM; 64 rows a CTA, a page read once, took 7 more (three CTAs
// an SM), 16 rows a CTA as long, but 33 for 25 us where 32 rows have 1500 positions. Two stages and
// five CTAs instead of three and four: 62 -> 50 us at the first; Q in shared memory, not registers:
// 50 -> 48. The scaling of f32's probabilities (split2_up) is 0.6 and 1.2 us of the two f32 figures.
#include <algorithm>
#include <type_traits>

#include "tree.cuh"

namespace wv {
namespace {

constexpr int TF_KEYS = 64;                  // positions a tile
constexpr int TF_WARPS = 4;                  // multiplying warps
constexpr int TF_THREADS = TF_WARPS * 32 + 32;
constexpr int TF_ROWS = 32;                  // rows of a CTA at most
constexpr uint32_t TF_HALF = TF_KEYS * 128;  // bytes of 64 positions x 64 elements

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
// c[16 x 8] += a[16 x 16] b[16 x 8], f16 in, f32 sums.
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte offset of 16-byte chunk `chunk` of tile row `row`: halves of 64 elements one after another.
__device__ __forceinline__ uint32_t tile_at(uint32_t row, uint32_t chunk) {
  return (chunk >> 3) * TF_HALF + sw128_offset(row, chunk & 7u);
}

// The multiplying warps alone.
__device__ __forceinline__ void warps_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(TF_WARPS * 32) : "memory");
}

// MAXR: rows that a CTA can have, 16 or 32. WIDE: f32 rows, as two f16 parts each.
template <int HDP, int MAXR, bool WIDE>
struct FewTile {
  static constexpr uint32_t kStage = 2 * (HDP / 64) * TF_HALF;
  static constexpr int kStages = 2;
  static constexpr int kCtas = HDP == 128 ? 2 : MAXR == 16 ? 5 : 4;  // of an SM
  static constexpr size_t kSmem =
      kStages * kStage + (WIDE ? 2 : 1) * (HDP / 64) * MAXR * 128 + 1024;
};

template <int ST>
struct FewShared {
  uint64_t full[ST], empty[ST];
  uint32_t info[ST];  // bit b: box b is in the pool; bit 31: every row sees all of it
  uint32_t abort;
  float m[TF_WARPS][16], l[TF_WARPS][16];
};

// A CTA's share: rows r0 .. of the item of request s and K and V head kvh, positions k0 .. k1.
struct FewItem {
  int s, kvh, r0, rows, lo, len, k0, k1, n_tiles, split;
};

// The multiplying warps' part, WR of them over the rows (16 each), 4 / WR over a tile's positions.
template <int HDP, int ST, int WR, bool WIDE>
__device__ __forceinline__ void few_rows(const AttendTreeArgs &a, const FewItem &f, uint8_t *tiles,
                                         FewShared<ST> &sh, const Abort &ab) {
  using E = typename std::conditional<WIDE, float, __half>::type;
  constexpr int WK = TF_WARPS / WR, KEYS = TF_KEYS / WK, KS = HDP / 16, NT = KEYS / 8;
  constexpr int MT = 16 * WR;
  constexpr uint32_t STAGE = 2 * (HDP / 64) * TF_HALF;
  const int tid = int(threadIdx.x), lane = tid & 31, w = int(warp_id());
  const int group = a.heads / a.kv_heads, len = f.len, k0 = f.k0, k1 = f.k1;
  const int wr = w % WR, wk = w / WR;
  const int g = lane >> 2, c2 = (lane & 3) * 2;
  // This thread's rows r and r + 8 of the warp's, and the first 32 drafted positions that they see.
  int row[2];
  uint32_t seen[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = f.r0 + wr * 16 + g + 8 * u, i = r / group;
    row[u] = r < f.rows && f.lo + i < a.rows ? f.lo + i : -1;
    seen[u] = a.mask && row[u] >= 0 ? a.mask[(long long)row[u] * a.words] : 0u;
  }
  // Q into shared memory behind the tiles, rows of 128 bytes in the tiles' swizzle, f32's low parts
  // after the high ones: registers for it would cost a CTA an SM.
  const uint32_t qs = smem_u32(tiles + ST * STAGE);
  constexpr uint32_t Q_HALF = MT * 128, Q_PART = (HDP / 64) * Q_HALF;
  {
    const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | (a.q_stride * sizeof(E))) & 15u) == 0;
    for (int e = tid; e < MT * (HDP / 8); e += TF_WARPS * 32) {
      const int r = e / (HDP / 8), c = e % (HDP / 8), i = (f.r0 + r) / group;
      E v[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) v[x] = E(0.0f);
      if (f.r0 + r < f.rows && f.lo + i < a.rows && c * 8 < a.hd) {
        const int head = f.kvh * group + (f.r0 + r) - i * group;
        const E *from = static_cast<const E *>(a.q) + (f.lo + i) * a.q_stride + head * a.hd + c * 8;
        if (vec) {
#pragma unroll
          for (int x = 0; x < int(sizeof(E)) / 2; ++x)
            reinterpret_cast<uint4 *>(v)[x] = reinterpret_cast<const uint4 *>(from)[x];
        } else {
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = from[x];
        }
      }
      uint8_t *to = tiles + ST * STAGE + (c >> 3) * Q_HALF + sw128_offset(r, c & 7);
      if constexpr (WIDE) {
        uint32_t hi[4], low[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) split2(v[2 * x], v[2 * x + 1], hi[x], low[x]);
        *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(to + Q_PART) = make_uint4(low[0], low[1], low[2], low[3]);
      } else {
        *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(v);
      }
    }
    warps_sync();
  }
  float acc[2 * KS][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  const float scale = a.scale * 1.4426950408889634f;  // exponentials of base 2
  bool ok = true;
  for (int i = 0; i < f.n_tiles; ++i) {
    const int st = i % ST;
    ok = mbar_wait_warp(&sh.full[st], (i / ST) & 1, ab, kErrTimeoutConsumer);
    if (!ok) break;
    const uint32_t kb = smem_u32(tiles + st * STAGE), vb = kb + (HDP / 64) * TF_HALF;
    const uint32_t bits = sh.info[st];
    const int first = wk * KEYS;  // the warp's first position in the tile
    const int p0 = k0 + i * TF_KEYS + first;
    float sc[NT][4] = {};
    // The low parts first: the sums are small until the high ones come, and so is what a step
    // drops.
#pragma unroll
    for (int part = WIDE ? 1 : 0; part >= 0; --part)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t qf[4];
        ldsm4(qf, qs + part * Q_PART + (ks >> 2) * Q_HALF +
                      sw128_offset(wr * 16 + (lane & 15), (2 * ks + (lane >> 4)) & 7));
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
          uint32_t b[4];
          ldsm4(b, kb + tile_at(first + n * 16 + (lane >> 4) * 8 + (lane & 7),
                                2 * ks + ((lane >> 3) & 1)));
          mma16(sc[2 * n], qf, b[0], b[1]);
          mma16(sc[2 * n + 1], qf, b[2], b[3]);
        }
      }
    bool odd = false;  // a V row that some rows do not see holds an infinity or NaN
    if (!(bits >> 31)) {
      // Positions past the end, outside the pool, or drafted off a row's path.
      const int box = min(a.bs, TF_KEYS);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int j = first + 8 * n + c2 + (x & 1), p = k0 + i * TF_KEYS + j, d = p - len;
          bool see = p < k1 && ((bits >> (j / box)) & 1u);
          if (see && d >= 0) {
            uint32_t word = seen[x >> 1];
            if (d >= 32)
              word = row[x >> 1] >= 0 && d < 32 * a.words
                         ? a.mask[(long long)row[x >> 1] * a.words + (d >> 5)]
                         : 0u;
            see = (word >> (d & 31)) & 1u;
          }
          if (!see) sc[n][x] = -INFINITY;
        }
      // What lies in a page past the end is nobody's: zeros in V (0 times NaN is not 0).
      if (p0 + KEYS > k1) {
        const int from = max(k1 - p0, 0);
        for (int e = lane; e < (KEYS - from) * (HDP / 8); e += 32) {
          const uint32_t at = vb + tile_at(first + from + e / (HDP / 8), e % (HDP / 8));
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0u) : "memory");
        }
        __syncwarp();
      }
      if (p0 + KEYS > len) {
        bool bad = false;
        for (int e = lane; e < KEYS * (HDP / 8); e += 32) {
          uint32_t v[4];
          const uint32_t at = vb + tile_at(first + e / (HDP / 8), e % (HDP / 8));
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                       : "r"(at)
                       : "memory");
#pragma unroll
          for (int k = 0; k < 4; ++k) bad = bad || finite2(v[k]) != v[k];
        }
        odd = __any_sync(0xffffffffu, bad);
      }
    }
    // The running reference and sum, two rows a thread (four threads a row). The reference is the
    // maximum, or kLift below it, rounded up, so that no probability passes 1, or 2^kLift.
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n) mx = fmaxf(mx, fmaxf(sc[n][2 * u], sc[n][2 * u + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      mx = fmaxf(m[u], __fmaf_ru(mx, scale, WIDE ? 0.0f : -float(kLift)));
      const float base = mx == -INFINITY ? 0.0f : mx;
      const float carry = ex2(m[u] - base);
      m[u] = mx;
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 2 * u; x < 2 * u + 2; ++x) {
          sc[n][x] = ex2(fmaf(sc[n][x], scale, -base));
          sum += sc[n][x];
        }
      l[u] = fmaf(l[u], carry, sum);
      if (__any_sync(0xffffffffu, carry != 1.0f))
#pragma unroll
        for (int n = 0; n < 2 * KS; ++n) {
          acc[n][2 * u] *= carry;
          acc[n][2 * u + 1] *= carry;
        }
    }
    const auto values = [&](auto clean) {
      uint32_t ph[NT / 2][4], pl[NT / 2][4];
#pragma unroll
      for (int kk = 0; kk < NT / 2; ++kk)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float p = sc[2 * kk + (x >> 1)][2 * (x & 1)];
          const float q = sc[2 * kk + (x >> 1)][2 * (x & 1) + 1];
          if constexpr (WIDE) split2_up<kLift>(p, q, ph[kk][x], pl[kk][x]);
          else ph[kk][x] = pack_half2(p, q);
        }
#pragma unroll
      for (int n = 0; n < KS; ++n) {
        // f32: a tile's products apart from the sums over the tiles, which f32 additions round: a
        // step of a tensor-core sum drops bits of its size. The low parts' first, scaled back.
        float part[2][4] = {};
        uint32_t b[NT / 2][4];
#pragma unroll
        for (int kk = 0; kk < NT / 2; ++kk) {
          ldsm4_t(b[kk], vb + tile_at(first + kk * 16 + (lane & 15), 2 * n + (lane >> 4)));
          if constexpr (decltype(clean)::value)
#pragma unroll
            for (int x = 0; x < 4; ++x) b[kk][x] = finite2(b[kk][x]);
          if constexpr (WIDE) {
            mma16(part[0], pl[kk], b[kk][0], b[kk][1]);
            mma16(part[1], pl[kk], b[kk][2], b[kk][3]);
          } else {
            mma16(acc[2 * n], ph[kk], b[kk][0], b[kk][1]);
            mma16(acc[2 * n + 1], ph[kk], b[kk][2], b[kk][3]);
          }
        }
        if constexpr (WIDE) {
#pragma unroll
          for (int x = 0; x < 8; ++x) part[x >> 2][x & 3] *= 1.0f / kLowUp;
#pragma unroll
          for (int kk = 0; kk < NT / 2; ++kk) {
            mma16(part[0], ph[kk], b[kk][0], b[kk][1]);
            mma16(part[1], ph[kk], b[kk][2], b[kk][3]);
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) acc[2 * n + (x >> 2)][x & 3] += part[x >> 2][x & 3];
        }
      }
    };
    if (!odd) {
      values(std::false_type());
    } else {
      // Infinities and NaN in V go one by one to the rows that see them, and the products get
      // zeros in their place (0 times infinity is not 0).
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
          const int from = (lane & ~3) | (j >> 1);
          float p[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float e = __shfl_sync(0xffffffffu, sc[n][2 * u], from);
            const float f = __shfl_sync(0xffffffffu, sc[n][2 * u + 1], from);
            p[u] = (j & 1) ? f : e;
          }
#pragma unroll
          for (int c = 0; c < 2 * KS; ++c) {
            uint32_t v;
            asm volatile("ld.shared.b32 %0, [%1];"
                         : "=r"(v)
                         : "r"(vb + tile_at(first + 8 * n + j, c) + 2 * c2)
                         : "memory");
            const uint32_t rest = v ^ finite2(v);
            if (rest == 0u) continue;
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&rest));
#pragma unroll
            for (int u = 0; u < 2; ++u)
              if (p[u] != 0.0f) {
                acc[c][2 * u] = fmaf(p[u], f.x, acc[c][2 * u]);
                acc[c][2 * u + 1] = fmaf(p[u], f.y, acc[c][2 * u + 1]);
              }
          }
        }
      values(std::true_type());
    }
    if (!(bits >> 31)) fence_proxy_async_smem();  // the zeros, before a later load
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.empty[st]);
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
  }


  // The warps' shares of the positions meet in shared memory, over the tiles.
  float *sum = reinterpret_cast<float *>(tiles);  // [WK][MT][HDP]
  warps_sync();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = wr * 16 + g + 8 * u;
    if ((lane & 3) == 0) {
      sh.m[w][g + 8 * u] = m[u];
      sh.l[w][g + 8 * u] = l[u];
    }
#pragma unroll
    for (int n = 0; n < 2 * KS; ++n)
      *reinterpret_cast<float2 *>(sum + (wk * MT + r) * HDP + 8 * n + c2) =
          make_float2(acc[n][2 * u], acc[n][2 * u + 1]);
  }
  warps_sync();
  if (sh.abort) return;  // a wait gave up: the outputs are left as they are
  const int quads = a.hd / 4;
  for (int e = tid; e < MT * quads; e += TF_WARPS * 32) {
    const int r = e / quads, c = (e - r * quads) * 4, rr = f.r0 + r;
    if (rr >= f.rows) break;
    const int i = rr / group, q = f.lo + i, head = f.kvh * group + rr - i * group;
    if (q >= a.rows) break;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < WK; ++k) top = fmaxf(top, sh.m[k * WR + (r >> 4)][r & 15]);
    const float base = top == -INFINITY ? 0.0f : top;
    float total = 0.0f, o[4] = {};
#pragma unroll
    for (int k = 0; k < WK; ++k) {
      const float x = ex2(sh.m[k * WR + (r >> 4)][r & 15] - base);
      const float4 v = *reinterpret_cast<const float4 *>(sum + (k * MT + r) * HDP + c);
      const float y = WIDE ? x * (1.0f / (1 << kLift)) : x;
      total = fmaf(x, sh.l[k * WR + (r >> 4)][r & 15], total);
      o[0] = fmaf(y, v.x, o[0]);
      o[1] = fmaf(y, v.y, o[1]);
      o[2] = fmaf(y, v.z, o[2]);
      o[3] = fmaf(y, v.w, o[3]);
    }
    if (a.splits == 1) {
      const float inv = total != 0.0f ? 1.0f / total : 0.0f;
      E *to = static_cast<E *>(a.o) + q * a.o_stride + (long long)head * a.hd + c;
#pragma unroll
      for (int x = 0; x < 4; ++x) to[x] = E(o[x] * inv);
    } else {
      float *to = a.part + (((long long)q * a.heads + head) * a.splits + f.split) * (a.hd + 4);
      *reinterpret_cast<float4 *>(to + c) = make_float4(o[0], o[1], o[2], o[3]);
      if (c == 0) *reinterpret_cast<float2 *>(to + a.hd) = make_float2(top, total);
    }
  }
}

template <int HDP, int MAXR, bool WIDE>
__global__ void __launch_bounds__(TF_THREADS, FewTile<HDP, MAXR, WIDE>::kCtas)
    attend_few_kernel(const __grid_constant__ CUtensorMap map, const AttendTreeArgs a) {
  using T = FewTile<HDP, MAXR, WIDE>;
  constexpr int ST = T::kStages;
  extern __shared__ uint8_t raw[];
  uint8_t *tiles = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                               ~uintptr_t(1023));
  __shared__ FewShared<ST> sh;
  const int tid = int(threadIdx.x), lane = tid & 31, w = int(warp_id());
  const Abort ab{&sh.abort, a.err};
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], TF_WARPS);
    }
    sh.abort = 0u;
    fence_mbar_init();
    prefetch_tmap(&map);
  }
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  __syncthreads();

  FewItem f;
  f.split = int(blockIdx.x) % a.splits;
  f.r0 = int(blockIdx.x) / a.splits * MAXR;
  f.kvh = int(blockIdx.y);
  f.s = int(blockIdx.z);
  f.lo = a.row_start ? a.row_start[f.s] : f.s;
  const int t = min(a.row_start ? a.row_start[f.s + 1] - f.lo : 1, a.max_rows);
  f.rows = t * (a.heads / a.kv_heads);  // token by token, the heads of each together
  if (f.r0 >= f.rows || f.lo < 0) return;
  f.len = max(a.lens[f.s], 0);
  const int keys = int(min((long long)f.len + (a.mask ? t : 0), (long long)a.max_len));
  f.k0 = f.split * a.chunk;
  f.k1 = min(keys, f.k0 + a.chunk);
  f.n_tiles = f.k1 > f.k0 ? (f.k1 - f.k0 + TF_KEYS - 1) / TF_KEYS : 0;

  if (w == TF_WARPS) {  // the producer: a lane a page of the tile, its block one tile ahead
    const int box = min(a.bs, TF_KEYS), boxes = TF_KEYS / box;
    const int *table = a.table + (long long)f.s * a.width;
    const auto block_of = [&](int i) {
      const int pos = f.k0 + i * TF_KEYS + lane * box;
      return i < f.n_tiles && lane < boxes && pos < keys ? table[pos / a.bs] : -1;
    };
    int next = block_of(0), i = 0;
    for (; i < f.n_tiles; ++i) {
      const int st = i % ST, pos = f.k0 + i * TF_KEYS + lane * box, b = next;
      next = block_of(i + 1);
      const bool in = b >= 0 && b < a.blocks;
      const uint32_t bits = __ballot_sync(0xffffffffu, in);
      if (i >= ST && !mbar_wait_warp(&sh.empty[st], ((i / ST) - 1) & 1, ab, kErrTimeoutProducer)) break;
      if (lane == 0) {
        const bool all = bits == (1u << boxes) - 1u &&
                         f.k0 + (i + 1) * TF_KEYS <= min(f.len, keys);
        sh.info[st] = bits | (all ? 1u << 31 : 0u);
        mbar_arrive_expect_tx(&sh.full[st], T::kStage);
      }
      __syncwarp();
      if (lane < boxes) {
        // A position outside the pool reads as zeros: block `blocks` is past the tensor's end.
        uint8_t *to = tiles + st * T::kStage + lane * box * 128;
        const int z = in ? b : a.blocks;
#pragma unroll
        for (int h = 0; h < HDP / 64; ++h) {
          tma_load_4d(to + h * TF_HALF, &map, &sh.full[st], 64 * h, pos % a.bs, f.kvh, z);
          tma_load_4d(to + (HDP / 64 + h) * TF_HALF, &map, &sh.full[st], 64 * h, pos % a.bs,
                      a.kv_heads + f.kvh, z);
        }
      }
    }
    // The shared memory stays until the last loads have landed, also where a wait gave up.
    for (int j = max(i - ST, 0); j < i; ++j)
      for (int k = 0; k < 2000 && !mbar_try_wait_sleep(&sh.full[j % ST], (j / ST) & 1, 100000u); ++k) {}
    return;
  }
  const int here = f.rows - f.r0;
  if (MAXR == 16 || here <= 16) few_rows<HDP, ST, 1, WIDE>(a, f, tiles, sh, ab);
  else few_rows<HDP, ST, 2, WIDE>(a, f, tiles, sh, ab);
}

// The ranges of a row joined: a CTA a (drafted row, request), four elements a thread.
template <typename E>
__global__ void __launch_bounds__(128) attend_few_join_kernel(const AttendTreeArgs a) {
  griddep_launch_dependents();
  griddep_wait();  // the previous kernel of the stream has completed (programmatic launch)
  const int i = int(blockIdx.x), s = int(blockIdx.z);
  const int lo = a.row_start ? a.row_start[s] : s;
  const int t = min(a.row_start ? a.row_start[s + 1] - lo : 1, a.max_rows), q = lo + i;
  if (i >= t || lo < 0 || q >= a.rows) return;
  const int quads = a.hd / 4;
  for (int e = int(blockIdx.y * blockDim.x + threadIdx.x); e < a.heads * quads;
       e += int(gridDim.y * blockDim.x)) {
    const int head = e / quads, c = (e - head * quads) * 4;
    const float *from = a.part + ((long long)q * a.heads + head) * a.splits * (a.hd + 4);
    float top = -INFINITY;
    for (int k = 0; k < a.splits; ++k) top = fmaxf(top, from[k * (a.hd + 4) + a.hd]);
    const float base = top == -INFINITY ? 0.0f : top;
    float total = 0.0f, o[4] = {};
    for (int k = 0; k < a.splits; ++k) {
      const float2 ml = *reinterpret_cast<const float2 *>(from + k * (a.hd + 4) + a.hd);
      const float4 v = *reinterpret_cast<const float4 *>(from + k * (a.hd + 4) + c);
      const float f = ex2(ml.x - base);
      total = fmaf(f, ml.y, total);
      o[0] = fmaf(f, v.x, o[0]);
      o[1] = fmaf(f, v.y, o[1]);
      o[2] = fmaf(f, v.z, o[2]);
      o[3] = fmaf(f, v.w, o[3]);
    }
    const float inv = total != 0.0f ? 1.0f / total : 0.0f;
    E *to = static_cast<E *>(a.o) + q * a.o_stride + (long long)head * a.hd + c;
#pragma unroll
    for (int x = 0; x < 4; ++x) to[x] = E(o[x] * inv);
  }
}

template <int HDP, int MAXR, bool WIDE>
cudaError_t launch_few(const CUtensorMap &map, const AttendTreeArgs &a, cudaStream_t s) {
  auto *kernel = attend_few_kernel<HDP, MAXR, WIDE>;
  constexpr size_t smem = FewTile<HDP, MAXR, WIDE>::kSmem;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !configured[dev]) {
    cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    if (dev < 64) configured[dev] = true;
  }
  const long long rows = (long long)a.max_rows * (a.heads / a.kv_heads);
  const int row_tiles = int((rows + MAXR - 1) / MAXR);
  return launch_pdl(kernel, dim3(a.splits * row_tiles, a.kv_heads, a.n), dim3(TF_THREADS), smem, s,
                    map, a);
}

template <int HDP, bool WIDE>
cudaError_t launch_rows(const CUtensorMap &map, const AttendTreeArgs &a, cudaStream_t s) {
  const long long rows = (long long)a.max_rows * (a.heads / a.kv_heads);
  return rows <= 16 ? launch_few<HDP, 16, WIDE>(map, a, s) : launch_few<HDP, TF_ROWS, WIDE>(map, a, s);
}

}  // namespace

AttendFewPlan attend_few_plan(int n, int max_rows, int max_len, int heads, int kv_heads, int hd,
                              int sms) {
  AttendFewPlan p;
  const long long rows = (long long)max_rows * (heads / kv_heads);
  const long long ctas = (long long)n * kv_heads * ((rows + TF_ROWS - 1) / TF_ROWS);
  // Ranges of 256 positions at least, as many as fill the SMs with three CTAs each (two for heads of
  // more than 64), also where an SM holds four or five.
  const long long slots = (hd <= 64 ? 3ll : 2ll) * sms;
  const long long want = std::max<long long>(1, slots / ctas);
  const long long most = std::max<long long>(1, (max_len + 255) / 256);
  p.splits = p.most = int(std::min<long long>(std::min(want, most), 128));
  p.chunk = int(((long long)max_len + p.splits - 1) / p.splits);
  p.chunk = std::max((p.chunk + TF_KEYS - 1) / TF_KEYS, 1) * TF_KEYS;
  p.splits = std::max((max_len + p.chunk - 1) / p.chunk, 1);
  return p;
}

size_t attend_few_part_bytes(const AttendFewPlan &p, int rows, int heads, int hd) {
  return p.splits > 1 ? size_t(rows) * heads * p.splits * (hd + 4) * sizeof(float) : 0;
}

cudaError_t launch_attend_few(const CUtensorMap &map, const AttendTreeArgs &a, int f16,
                              cudaStream_t s) {
  if (a.n <= 0 || a.max_rows <= 0) return cudaSuccess;
  cudaError_t e;
  if (a.hd <= 64) e = f16 ? launch_rows<64, false>(map, a, s) : launch_rows<64, true>(map, a, s);
  else e = f16 ? launch_rows<128, false>(map, a, s) : launch_rows<128, true>(map, a, s);
  if (e != cudaSuccess || a.splits == 1) return e;
  const dim3 grid(a.max_rows, std::min(8, (a.heads * a.hd / 4 + 127) / 128), a.n);
  return f16 ? launch_pdl(attend_few_join_kernel<__half>, grid, dim3(128), 0, s, a)
             : launch_pdl(attend_few_join_kernel<float>, grid, dim3(128), 0, s, a);
}

}  // namespace wv
