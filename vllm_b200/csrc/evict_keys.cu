// Cutting a paged cache back: of a request's n rows a kv head keeps m = min(n, keep), those of the lowest and the newest positions and of the others those
// of the highest scores (ties: the first row); kept rows behind row m move into the evicted rows in front of it, the i-th into the i-th.
//
// A row's place is a 32-bit key that orders like (protected, score); the m-th largest key is found digit by digit (8 bits) from counts in shared
// memory.  A request of up to 4096 rows is a CTA's for each kv head, longer ones a cluster's, whose CTAs add their counts through distributed
// shared memory; the keys are made once and stay in shared memory.  Warps hold runs of neighbours, so ranks among equal keys, evicted and moving rows
// are counts of bits in front.  What bounds it is the chain of passes and exchanges: digits of 11 bits, whose bins take longer to add up than a pass over
// the rows, took 29 us for 64 x 1200 rows of 8 heads and 86 us for 4 x 30000.
// A second kernel moves the rows: nothing is read that is written (sources lie behind m, targets in front), so the order does not matter.  Filling the
// gaps moves as many rows as were evicted in front of m, where keeping the order would move nearly all.
#include "cluster.cuh"

namespace evict {

constexpr int BINS = 256, DIGITS = 4;
constexpr uint32_t LOWEST = 0x007fffffu, PROTECTED = 0xffffffffu;        // -inf; above +inf
constexpr int CTA_ROWS = 4096;                                           // rows of a CTA, where eight are enough for them
constexpr int MANY = 296;                                                // CTAs from which they have 8 warps instead of 16: two for each SM
constexpr int FUSED_CTAS = 148, FUSED_MOVES = 1024;                      // up to which there is one kernel
constexpr int SMEM_ROWS = 50 * 1024;                                     // of which the keys fit; beyond 8 times that they are made anew in every pass

struct Params {
  const float* scores;
  const int* positions;      // null: a row's number
  const int* seq_lens;
  float* new_scores;         // [B, Hkv, L]
  int* new_positions;
  int* new_lens;
  int* count;                // [B Hkv]: rows that move
  int* target;               // [B Hkv][cap]
  int* source;
  int64_t sc_req, sc_head, po_req, po_head;
  int Hkv, L, max_rows, keep, first, recent, parts, cap;
};

VB_DEVICE uint32_t ordered(float x) {
  if (x != x) return LOWEST;
  const uint32_t u = __float_as_uint(x + 0.f);                            // (-0 is 0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Move {
  const float* scores;
  const int* positions;
  float* new_scores;
  int* new_positions;
  const int* count;
  const int* target;
  const int* source;
  uint16_t* cache;
  const int* block_table;
  int64_t sc_req, sc_head, po_req, po_head, bt_stride, num_blocks;
  int Hkv, L, cap, D, BS;
};

// Of up to N moves: places of the keys in the cache (to: -1, none), and of the values
template <int N> struct Places { int64_t from[N], to[N], vfrom[N], vto[N]; };

// A CTA moves the rows j0 .. j0 + n - 1 of a list, n <= N <= THREADS.  Transposed values: a lane per move, a dimension at a time, as neighbours in the list
// are near each other in source and target.  Nearly all of the 32-byte pieces of a page's values hold a row that moves or one that makes room,
// so those pages are read and written almost whole: 317 MB at 5.5 TB/s for 4 x 30000 rows down to 4096, 57 us.
template <int THREADS, int N> VB_DEVICE void move_rows(const Move& p, Places<N>& at, bool vt, int b, int h, int j0, int n) {
  const int row = b * p.Hkv + h;
  if ((int)threadIdx.x < n) {
    const int t = p.target[(int64_t)row * p.cap + j0 + threadIdx.x], s = p.source[(int64_t)row * p.cap + j0 + threadIdx.x];
    p.new_scores[(int64_t)row * p.L + t] = p.scores[b * p.sc_req + h * p.sc_head + s];
    p.new_positions[(int64_t)row * p.L + t] = p.positions ? p.positions[b * p.po_req + h * p.po_head + s] : s;
    const int64_t page = (int64_t)p.BS * p.D;
    int64_t bt = p.block_table[b * p.bt_stride + t / p.BS], bs = p.block_table[b * p.bt_stride + s / p.BS];
    const bool ok = (uint64_t)bt < (uint64_t)p.num_blocks && (uint64_t)bs < (uint64_t)p.num_blocks;   // (a table may not say else; nothing outside the
    if (!ok) bt = bs = 0;                                                                             // cache is touched)
    const int64_t kt = (bt * 2 * p.Hkv + h) * page, ks = (bs * 2 * p.Hkv + h) * page, v = p.Hkv * page;
    const int64_t to = kt + (int64_t)(t % p.BS) * p.D, from = ks + (int64_t)(s % p.BS) * p.D;
    at.to[threadIdx.x] = ok ? to : -1;
    at.from[threadIdx.x] = from;
    at.vto[threadIdx.x] = vt ? kt + v + t % p.BS : to + v;
    at.vfrom[threadIdx.x] = vt ? ks + v + s % p.BS : from + v;
  }
  __syncthreads();
  // transposed values, a warp: 32 moves, DIMS dimensions; the warp's first ones are on their way while the keys move
  constexpr int DIMS = N == 32 ? 16 : 32, UNITS = 128 / DIMS;
  const int lane = threadIdx.x & 31, units = vt ? (n + 31) / 32 * UNITS : 0;
  int unit = threadIdx.x >> 5;
  uint16_t x[DIMS];
  auto read = [&]() -> uint16_t* {                       // where they go, or null
    const int j = unit / UNITS * 32 + lane, d = unit % UNITS * DIMS;
    if (unit >= units || j >= n || at.to[j] < 0) return nullptr;
    const uint16_t* src = p.cache + at.vfrom[j] + d * p.BS;
#pragma unroll
    for (int u = 0; u < DIMS; ++u) x[u] = src[u * p.BS];
    return p.cache + at.vto[j] + d * p.BS;
  };
  uint16_t* to_x = read();
  const int ch = p.D / 8, items = n * ch;
  constexpr int U = 2;                                   // pieces on their way at a time
  for (int i0 = threadIdx.x; i0 < items; i0 += U * THREADS) {
    uint4 k[U], v[U];
    int64_t to[U], vto[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * THREADS, j = i / ch, c = i % ch * 8;
      to[u] = i < items ? at.to[j] : -1;
      if (to[u] >= 0) {
        k[u] = *reinterpret_cast<const uint4*>(p.cache + at.from[j] + c);
        if (!vt) v[u] = *reinterpret_cast<const uint4*>(p.cache + at.vfrom[j] + c);
        to[u] += c;
        vto[u] = at.vto[j] + c;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (to[u] >= 0) {
        if (!vt) *reinterpret_cast<uint4*>(p.cache + vto[u]) = v[u];
        *reinterpret_cast<uint4*>(p.cache + to[u]) = k[u];
      }
    }
  }
  while (unit < units) {
    if (to_x) {
#pragma unroll
      for (int u = 0; u < DIMS; ++u) to_x[u * p.BS] = x[u];
    }
    unit += THREADS / 32;
    to_x = read();
  }
}

constexpr int PAIRS = 32, MOVERS = 256;
// Grid (groups of 32 moves, kv heads, requests)
template <bool VT>
__global__ void __launch_bounds__(MOVERS) move_kernel(const Move p) {
  __shared__ Places<PAIRS> at;
  pdl_trigger();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z, j0 = blockIdx.x * PAIRS, n = min(p.count[b * p.Hkv + h] - j0, PAIRS);
  if (n > 0) move_rows<MOVERS, PAIRS>(p, at, VT, b, h, j0, n);
}

// KEPT: the keys are kept in shared memory.  FUSED (1: values in rows, 2: transposed): the CTA or the cluster moves its rows, too
template <bool KEPT, int THREADS, int FUSED>
__global__ void __launch_bounds__(THREADS) select_kernel(const Params p, const Move mv) {
  constexpr int WARPS = THREADS / 32;
  extern __shared__ uint32_t evict_smem[];
  uint32_t* hist = evict_smem;                           // [DIGITS][BINS]
  uint32_t* masks = hist + DIGITS * BINS;                // a bit per row: kept (of rows of a CTA / 32 words, rounded up)
  __shared__ int sums[2][WARPS], box[4];
  __shared__ int all_bins[BINS], found[3];
  pdl_wait();
  pdl_trigger();                                         // (here: the moving kernel is waiting when this one ends)
  const int rank = blockIdx.x % p.parts, row = blockIdx.x / p.parts, b = row / p.Hkv, h = row % p.Hkv;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n = min(max(p.seq_lens[b], 0), p.max_rows), m = min(n, p.keep);
  const int chunk = ((n + p.parts - 1) / p.parts + 31) & ~31;
  const int lo = min(rank * chunk, n), hi = min(lo + chunk, n);
  const int seg = ((hi - lo + WARPS - 1) / WARPS + 31) & ~31;
  const int w0 = min(lo + w * seg, hi), w1 = min(w0 + seg, hi);           // the warp's run
  uint32_t* keys = masks + (p.max_rows / p.parts + 63) / 32 + 1 - lo;     // keys[i] of row i
  const float* scores = p.scores + b * p.sc_req + h * p.sc_head;
  const int* positions = p.positions ? p.positions + b * p.po_req + h * p.po_head : nullptr;
  float* new_scores = p.new_scores + (int64_t)row * p.L;
  int* new_positions = p.new_positions + (int64_t)row * p.L;
  if (rank == 0 && h == 0 && threadIdx.x == 0) p.new_lens[b] = m;
  for (int i = threadIdx.x; i < DIGITS * BINS; i += THREADS) hist[i] = 0;

  int total = n;                                         // the next position
  if (positions) {
    int top = -1;
#pragma unroll 8
    for (int i = w0 + lane; i < w1; i += 32) top = max(top, positions[i]);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) sums[0][w] = top;
    __syncthreads();
    top = -1;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) top = max(top, sums[0][i]);
    if (p.parts > 1) {
      if (threadIdx.x == 0) box[0] = top;
      cluster_sync();
      for (int i = 0; i < p.parts; ++i) top = max(top, __float_as_int(ld_dsmem_f32(dsmem_addr(smem_u32(&box[0]), i))));
    }
    total = top + 1;
  }
  auto make = [&](int i) {
    const int place = positions ? positions[i] : i;
    return place < p.first || place >= total - p.recent ? PROTECTED : ordered(scores[i]);
  };
  auto key = [&](int i) { return KEPT ? keys[i] : make(i); };
  constexpr int U = 4;                                   // loads on their way at a time
  if (KEPT) {
    for (int i0 = w0 + lane; i0 < w1; i0 += 32 * U) {
      float x[U];
      int place[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = min(i0 + u * 32, w1 - 1);
        x[u] = scores[i];
        place[u] = positions ? positions[i] : i;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * 32 < w1) keys[i0 + u * 32] = place[u] < p.first || place[u] >= total - p.recent ? PROTECTED : ordered(x[u]);
    }
  }

  // ---- the m-th largest key, and how many of its equals stay
  uint32_t prefix = 0;
  int need = m;
  bool ties = false;                                     // not all of them
  if (m < n) {
    __syncthreads();
#pragma unroll 1
    for (int d = 0; d < DIGITS; ++d) {
      const int shift = 24 - 8 * d;
      const uint32_t above = d == 0 ? 0u : 0xffffffffu << (shift + 8);
      uint32_t* bins = hist + d * BINS;
      for (int i = w0 + lane; i < w1; i += 32) {
        const uint32_t k = key(i);
        if ((k & above) == prefix) atomicAdd(&bins[k >> shift & 255], 1u);
      }
      if (p.parts > 1) {
        cluster_sync();
        for (int bin = threadIdx.x; bin < BINS; bin += THREADS) {
          int c = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < p.parts) c += __float_as_int(ld_dsmem_f32(dsmem_addr(smem_u32(&bins[bin]), i)));
          all_bins[bin] = c;
        }
      }
      __syncthreads();
      if (w == 0) {                                      // eight bins a lane, from the highest down
        const int* from = p.parts > 1 ? all_bins : reinterpret_cast<const int*>(bins);
        int c[8], mine = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mine += c[j] = from[BINS - 1 - (lane * 8 + j)];
        int x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        int before = x - mine;
        if (before < need && before + mine >= need) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (before < need && before + c[j] >= need) {
              found[0] = BINS - 1 - (lane * 8 + j);
              found[1] = need - before;
              found[2] = c[j];
            }
            before += c[j];
          }
        }
      }
      __syncthreads();
      prefix |= (uint32_t)found[0] << shift;
      need = found[1];
      ties = need < found[2];
    }
  }
  // The same number of a warp in all its lanes: sums over the warps in front, in front in the cluster too, and over the cluster, for two of them.
  auto scan_two = [&](int& x, int& y, int& all_x, int slot) {
    __syncthreads();
    if (lane == 0) { sums[0][w] = x; sums[1][w] = y; }
    __syncthreads();
    int bx = 0, by = 0, ax = 0, ay = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      if (i < w) { bx += sums[0][i]; by += sums[1][i]; }
      ax += sums[0][i]; ay += sums[1][i];
    }
    if (p.parts > 1) {
      if (threadIdx.x == 0) { box[slot] = ax; box[slot + 1] = ay; }
      cluster_sync();
      const int own = ax;
      ax = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i < p.parts) {
          const int vx = i == rank ? own : __float_as_int(ld_dsmem_f32(dsmem_addr(smem_u32(&box[slot]), i)));
          const int vy = i < rank ? __float_as_int(ld_dsmem_f32(dsmem_addr(smem_u32(&box[slot + 1]), i))) : 0;
          if (i < rank) { bx += vx; by += vy; }
          ax += vx;
        }
      }
    }
    x = bx; y = by; all_x = ax;
  };
  // ---- which rows stay: a bit each
  int equal = 0, none = 0, all;
  if (ties) {
    for (int i = w0; i < w1; i += 32) equal += __popc(__ballot_sync(0xffffffffu, i + lane < w1 && key(i + lane) == prefix));
    scan_two(equal, none, all, 0);
  }
  int holes = 0, movers = 0;
  for (int i = w0; i < w1; i += 32) {
    const bool there = i + lane < w1;
    const uint32_t here = w1 - i >= 32 ? 0xffffffffu : (1u << (w1 - i)) - 1;
    uint32_t stay = here;
    if (m < n) {
      const uint32_t k = there ? key(i + lane) : 0u;
      if (ties) {
        const uint32_t same = __ballot_sync(0xffffffffu, there && k == prefix);
        stay = __ballot_sync(0xffffffffu, there && (k > prefix || (k == prefix && equal + __popc(same & ((1u << lane) - 1)) < need)));
        equal += __popc(same);
      } else {
        stay = __ballot_sync(0xffffffffu, there && k >= prefix);
      }
    }
    const uint32_t front = i >= m ? 0u : m - i >= 32 ? 0xffffffffu : (1u << (m - i)) - 1;
    holes += __popc(~stay & front & here);
    movers += __popc(stay & ~front);
    if (lane == 0) masks[(i - lo) >> 5] = stay;
  }
  __syncwarp();
  int n_holes;
  scan_two(holes, movers, n_holes, 2);
  if (rank == 0 && threadIdx.x == 0) p.count[row] = n_holes;
  // ---- lists, and scores and positions of the rows that do not move
  int* target = p.target + (int64_t)row * p.cap;
  int* source = p.source + (int64_t)row * p.cap;
  for (int i0 = w0; i0 < w1; i0 += 32 * U) {
    float x[U];
    int place[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * 32 + lane;
      x[u] = i < min(w1, m) ? scores[i] : 0.f;
      place[u] = positions && i < min(w1, m) ? positions[i] : i;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * 32;
      if (i >= w1) break;
      const uint32_t stay = masks[(i - lo) >> 5];
      const uint32_t front = i >= m ? 0u : m - i >= 32 ? 0xffffffffu : (1u << (m - i)) - 1;
      const uint32_t here = w1 - i >= 32 ? 0xffffffffu : (1u << (w1 - i)) - 1, me = 1u << lane;
      const uint32_t hole = ~stay & front & here, mover = stay & ~front;
      if (hole & me) target[holes + __popc(hole & (me - 1))] = i + lane;
      if (mover & me) source[movers + __popc(mover & (me - 1))] = i + lane;
      if (stay & front & me) {
        new_scores[i + lane] = x[u];
        new_positions[i + lane] = place[u];
      }
      holes += __popc(hole);
      movers += __popc(mover);
    }
  }
  for (int i = m + rank * THREADS + threadIdx.x; i < p.L; i += p.parts * THREADS) {
    new_scores[i] = 0.f;
    new_positions[i] = total + i - m;
  }
  if (p.parts > 1) cluster_sync();                       // the others may still read this CTA's counts and mailboxes (and have written their lists)
  if constexpr (FUSED != 0) {
    __shared__ Places<THREADS> at;
    const int share = (n_holes + p.parts - 1) / p.parts, last = min((rank + 1) * share, n_holes);
    for (int j0 = rank * share; j0 < last; j0 += THREADS) {
      __syncthreads();
      move_rows<THREADS, THREADS>(mv, at, FUSED == 2, b, h, j0, min(last - j0, THREADS));
    }
  }
}

}  // namespace evict

// `ws`: B Hkv (1 + 2 cap) ints, cap = max(0, min(keep, max_rows - keep)) moves of a row.  max_rows: rows of a request that the block table and the scores
// have room for.
EXPORT int vb_evict_keys(void* cache, int64_t num_blocks, const int* block_table, const int* seq_lens, const float* scores, const int* positions,
                         float* new_scores, int* new_positions, int* new_lens, int* ws, int B, int Hkv, int D, int BS, int L, int max_rows, int keep, int first,
                         int recent, int64_t bt_stride, int64_t sc_req, int64_t sc_head, int64_t po_req, int64_t po_head, int vt, cudaStream_t st) {
  using namespace evict;
  if (B <= 0 || Hkv <= 0) return 0;
  if (D % 8 || (vt && (D != 128 || BS != 64)) || keep < 1 || max_rows > L || max_rows < 0) return -1;
  const int spare = max_rows - keep, cap = spare <= 0 ? 0 : spare < keep ? spare : keep;
  Params p{scores, positions, seq_lens, new_scores, new_positions, new_lens, ws, ws + (int64_t)B * Hkv, ws + (int64_t)B * Hkv * (1 + cap),
           sc_req, sc_head, po_req, po_head, Hkv, L, max_rows, keep, first, recent, 1, cap};
  while (p.parts < 8 && max_rows > CTA_ROWS * p.parts) p.parts *= 2;
  const int rows = (max_rows + p.parts - 1) / p.parts + 32;
  const bool kept = rows <= SMEM_ROWS;
  const size_t smem = (size_t)(DIGITS * BINS + (max_rows / p.parts + 63) / 32 + 1 + (kept ? rows : 0)) * 4;
  if (smem > 227 * 1024) return -3;
  // Few CTAs wait for their chains, many for instructions that every warp has of its own.  us of both kernels with 8 and 16 warps: 1 request of 700 rows
  // (8 CTAs) 10.8 and 10.2, 16 of 2000 (64) 22.4 and 14.0, 64 of 1200 (512) 74.3 and 77.4, 4 of 30000 (256 in clusters) 97.5 and 82.9
  const bool many = p.parts == 1 && (int64_t)B * Hkv > MANY;
  const Move mv{scores, positions, new_scores, new_positions, p.count, p.target, p.source, reinterpret_cast<uint16_t*>(cache), block_table,
                sc_req, sc_head, po_req, po_head, bt_stride, num_blocks, Hkv, L, cap, D, BS};
  // One kernel where that leaves a CTA for every SM at most and few moves to each: a cut is called now and then, and a launch costs the host 3 us.  A call and
  // its kernels, us, in two and in one: 700 rows to 512, 8 heads 23.1 and 20.0 (10.1 and 12.4), 16 x 2000 to 1500, 4 heads of 64 24.2 and 21.0 (14.0 and 13.2)
  const bool fused = kept && !many && (int64_t)B * Hkv * p.parts <= FUSED_CTAS && cap <= FUSED_MOVES && rows <= CTA_ROWS + 32;
  auto k = !kept ? select_kernel<false, 512, 0>
           : many ? select_kernel<true, 256, 0>
           : !fused ? select_kernel<true, 512, 0>
           : vt ? select_kernel<true, 512, 2> : select_kernel<true, 512, 1>;
  if (smem > 24 * 1024 && cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return (int)cudaGetLastError();
  if (vb_launch_parts(k, dim3((unsigned)(B * Hkv * p.parts)), dim3(many ? 256 : 512), smem, st, (unsigned)p.parts, p, mv) != cudaSuccess)
    return (int)cudaGetLastError();
  if (cap > 0 && !fused) {
    const dim3 grid((cap + PAIRS - 1) / PAIRS, Hkv, B);
    if ((vt ? vb_launch(move_kernel<true>, grid, dim3(MOVERS), 0, st, mv) : vb_launch(move_kernel<false>, grid, dim3(MOVERS), 0, st, mv)) != cudaSuccess)
      return (int)cudaGetLastError();
  }
  return (int)cudaGetLastError();
}
