// Attention of one new token per request over a paged cache, which also adds to each cached key's score the weights that it got.
//
//   s[h, k] = c(scale q_h . K_k),  lse_h = log(sum_k e^s[h, k] + e^sink_h),  out_h = sum_k e^(s[h, k] - lse_h) V_k
//   scores[b, g, k] += sum over the query heads h of kv head g of e^(s[h, k] - lse_h)
//
// A weight is known when the last key has been seen, so there are two kernels.  The first reads keys and values once, leaves the scores s in a
// workspace (4 bytes a query head and key, beside 4 D bytes of the key and its value: 6 % more for 4 heads of 128, written and read in L2) and
// a running maximum, sum and output per part of a request's keys.  The second joins the parts, writes the output and adds
// the weights.
//
// First kernel: rows are pairs (request, kv head); all their tiles of 64 keys, in order, are dealt to the CTAs in equal runs, so that ragged and
// few long requests keep all SMs as busy as many equal ones.  In a run a warp takes every fourth strip of 16 keys through
// S^T = K Q^T (m16n8k16: keys are rows, the at most 16 query heads columns), an own running maximum and O^T += V^T P^T; its strips
// come by asynchronous copies of its own, STAGES of them on their way across the borders of rows, so warps meet only where a row
// ends.  Weights enter the second product as two 16-bit parts, P = hi + lo: the output is then as exact as its own rounding.
// Few short requests (scored_parts in ops/cuda.py) are one kernel's instead: a cluster has a row, its scores stay in shared memory, and the parts meet there.
//
// Decode is bound by the bytes of the cache; a tcgen05 product (128 keys x 16) would take the scores through tensor memory and
// barriers between roles for products that are a few percent of the time.  us for 64 requests of 1000 with 32 / 8 heads of 128 (bytes 40.9):
// 54, of which the first kernel takes 46 and the join 8; two of 95000 (121) 131; one of 700 (0.45) 6.3 in clusters and 8.6 without; 24 of 60 to 924 with
// 16 / 8 heads of 64, capped, fp16 (3.8) 15.7.
// The other way to the weights, a second pass over the keys, would read half the cache again.
#include "attention_prompt.cuh"
#include "cluster.cuh"
#include "device_once.h"

namespace sdec {

constexpr int TILE = 64, STRIP = 16;
constexpr int MAX_REQUESTS = 512;           // of a launch: their first tiles lie in shared memory
constexpr float LOG2E = 1.4426950408889634f;

struct Params {
  const void* q;
  const void* cache;
  const int* block_table;
  const int* seq_lens;
  void* out;
  float* scores;
  const float* sinks;
  float* raw;              // [request][kv head][raw_rows][G]: scores in powers of two
  float* part;             // [segment][16][D + 2]: output, maximum, sum
  int2* info;              // [row]: its first CTA, and how many
  int64_t q_stride, out_stride, bt_stride, sc_req, sc_head;
  int64_t num_blocks;
  int B, Hkv, G, D, BS, max_rows, raw_rows, ctas, chunks, extra, block, parts;      // chunks: of at most 16 query heads of a kv head
  float scale_log2, ku, c2;
};

VB_DEVICE int rows_of(const Params& p, int b) { return min(max(p.seq_lens[b], 0), p.max_rows); }

// A row's tiles, and what its end costs in tiles
VB_DEVICE int slots_of(const Params& p, int n) { return n > 0 ? (n + TILE - 1) / TILE + p.extra : 0; }

// first[b]: slots of all rows in front of request b, as if each request had one kv head; first[B]: of all
VB_DEVICE void scan_tiles(const Params& p, int* first, int* lens, int* warp_sums) {
  const int n_threads = blockDim.x, lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = n_threads >> 5;
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += n_threads) {
    const int b = b0 + threadIdx.x;
    const int n = b < p.B ? rows_of(p, b) : 0, mine = slots_of(p, n);
    if (b < p.B) lens[b] = n;
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[w] = x;
    __syncthreads();
    int before = base;
    for (int i = 0; i < nw; ++i) {
      if (i < w) before += warp_sums[i];
      base += warp_sums[i];
    }
    if (b < p.B) first[b] = before + x - mine;
    __syncthreads();
  }
  if (threadIdx.x == 0) first[p.B] = base;
  __syncthreads();
}

// A row: request, kv head, chunk of query heads; its slots are [begin, end) of the order of all
struct Row {
  int index, b, hc, begin, end;
};
VB_DEVICE void row_at(const int* first, int B, int H, int tile, Row& r) {      // the row that has this tile
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] * H <= tile) lo = mid; else hi = mid - 1;
  }
  const int n = first[lo + 1] - first[lo];               // > 0: the last request that begins at or in front of the tile
  r.b = lo;
  r.hc = (tile - first[lo] * H) / n;
  r.index = lo * H + r.hc;
  r.begin = first[lo] * H + r.hc * n;
  r.end = r.begin + n;
}
VB_DEVICE void next_row(const int* first, int H, Row& r) {                     // behind it there is one more
  if (++r.hc == H) {
    r.hc = 0;
    do { ++r.b; } while (first[r.b + 1] == first[r.b]);
  }
  r.index = r.b * H + r.hc;
  r.begin = r.end;
  r.end = r.begin + first[r.b + 1] - first[r.b];
}

// (the cache is read once and leaves L2 first, so that the scores that are read again stay in it: 64 x 1000 58 to 54 us, 2 x 95000 141 to 136)
VB_DEVICE void cp_async16(uint32_t dst, const void* src, bool real) {
  const int n = real ? 16 : 0;
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(n), "l"(L2_EVICT_FIRST) : "memory");
}
VB_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> VB_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

VB_DEVICE void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
VB_DEVICE void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> VB_DEVICE void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> VB_DEVICE void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> VB_DEVICE void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit values, two to a lane, with rows and columns exchanged
VB_DEVICE uint32_t turn8(uint32_t x) { uint32_t r; asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x)); return r; }

// DP: head size, rounded up to 64, 128 or 256 (what is behind it is zeros in shared memory); NT: groups of eight query heads
template <int DP_> struct Form {
  static constexpr int DP = DP_, WARPS = 4, THREADS = WARPS * 32, CTAS = DP == 256 ? 1 : 2;      // CTAS: of an SM
  static constexpr int STRIP_BYTES = STRIP * DP * 2;                       // of keys; values behind them
  static constexpr int STAGES = DP == 64 ? 6 : 3;
  static constexpr int RING = WARPS * STAGES * 2 * STRIP_BYTES;
  static constexpr int REGS = DP / 16 * 4 + 4;                             // of a group of heads: output, maxima, sums
  static constexpr int SMEM = RING + WARPS / 2 * REGS * 128 + (2 * MAX_REQUESTS + 1 + 32) * 4;
};

// FUSED: a row's tiles are the p.parts CTAs' of a cluster, and everything is done here: the scores stay in shared memory until the parts have met.
template <typename T, int DP, int NT, bool VT, bool CAP, bool FUSED>
__global__ void __launch_bounds__(Form<DP>::THREADS, Form<DP>::CTAS) decode_kernel(const Params p) {
  using F = Form<DP>;
  // The reference of a head's weights is its largest score less SHIFT, or up to 8 below that.  fp16 has no values under 2^-24: as multiples of 2^-32 of the
  // largest weight the tail of a long request is not lost.
  constexpr float SHIFT = sizeof(T) == 2 && DTypeOf<T>::v == DT_F16 ? 7.f : 0.f;
  constexpr int WARPS = F::WARPS, STAGES = F::STAGES, KD = DP / 16, CH = DP / 8;           // CH: 16-byte pieces of a key
  extern __shared__ __align__(128) unsigned char smem[];
  float* exch = reinterpret_cast<float*>(smem + F::RING);
  int* first = reinterpret_cast<int*>(smem + F::RING + WARPS / 2 * F::REGS * 128);
  int* lens = first + MAX_REQUESTS + 1;
  int* warp_sums = lens + MAX_REQUESTS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_trigger();             // (here: the joining kernel may read the lengths as soon as it starts)
  const int H = p.Hkv * p.chunks, PD = p.D + 2;
  int t0, t1, per;
  Row row;
  float *raw_s = nullptr, *part_s = nullptr, *factor_s = nullptr;          // FUSED: scores of the CTA's keys, its part, log-sum-exps and factors of the parts
  const int rank = FUSED ? blockIdx.x % p.parts : 0;
  if constexpr (FUSED) {
    row.index = blockIdx.x / p.parts;
    row.b = row.index / p.Hkv;
    row.hc = row.index % p.Hkv;
    row.begin = 0;
    row.end = (rows_of(p, row.b) + TILE - 1) / TILE;
    per = (row.end + p.parts - 1) / p.parts;
    t0 = min(rank * per, row.end);
    t1 = min(t0 + per, row.end);
    part_s = reinterpret_cast<float*>(first);
    factor_s = part_s + p.G * PD;
    raw_s = factor_s + p.G * 9 + (-(p.G * (PD + 9)) & 3);
  } else {
    scan_tiles(p, first, lens, warp_sums);
    const int total = first[p.B] * H;
    per = (total + p.ctas - 1) / p.ctas;
    t0 = blockIdx.x * per;
    t1 = min(t0 + per, total);
    if (t0 >= t1) return;
    row_at(first, p.B, H, t0, row);
  }
  int n = FUSED ? rows_of(p, row.b) : lens[row.b];

  // A warp's stages of keys, with its values behind each; transposed values (VT) come as whole pages of 64 keys, a warp's strip being a quarter of them:
  // each warp fetches 32 of their 128 rows, and the warps meet once a page.
  constexpr int STAGE = (VT ? 1 : 2) * F::STRIP_BYTES;
  static_assert(!VT || (DP == 128 && WARPS * STRIP == TILE), "a page of transposed values is a tile");
  const uint32_t ring = smem_u32(smem) + warp * (STAGES * STAGE), v_ring = smem_u32(smem) + WARPS * STAGES * F::STRIP_BYTES;
  const int64_t page = (int64_t)p.BS * p.D;                                // values of a page of one head
  // The warp's strips: flat numbers 4 t0 + warp + i WARPS.  Where they lie is looked up for 32 of them at once, a lane each: a block number comes
  // out of memory before the copies can be issued, and one at a time that was most of a short run.
  const int s_end = t1 * 4;
  int64_t my_page = 0;                                                      // of the lane's strip: place of the page, token in it (-1: nothing to fetch)
  int my_off = -1, fetched = 0;
  const int c0 = lane % CH, r0l = lane / CH;                                // CH = 8, 16, 32: a lane's piece of a key and its first key
  constexpr int RSTEP = CH >= 32 ? 1 : 32 / CH;
  const bool real = c0 * 8 < p.D;
  auto fetch = [&](int stage) {
    if ((fetched & 31) == 0) {
      const int s = t0 * 4 + warp + (fetched + lane) * WARPS;
      my_off = -1;
      if (s < s_end) {
        Row r = row;
        if (!FUSED) row_at(first, p.B, H, s >> 2, r);
        const int tok = VT ? ((s >> 2) - r.begin) * TILE : (s - r.begin * 4) * STRIP;      // VT: of the page
        if (tok < (FUSED ? n : lens[r.b])) {
          int64_t blk = p.block_table[r.b * p.bt_stride + tok / p.BS];
          if ((uint64_t)blk >= (uint64_t)p.num_blocks) blk = 0;             // (a table may not say that; nothing is read outside the cache)
          my_page = (blk * 2 * p.Hkv + r.hc / p.chunks) * page;
          my_off = tok % p.BS;
        }
      }
    }
    const int off = __shfl_sync(0xffffffffu, my_off, fetched & 31);
    const int64_t at = __shfl_sync(0xffffffffu, my_page, fetched & 31);
    ++fetched;
    if (off >= 0) {
      const T* k = reinterpret_cast<const T*>(p.cache) + at;
      const T* v = k + p.Hkv * page;
      const uint32_t to = ring + stage * STAGE;
      const T* src = k + (int64_t)(VT ? warp * STRIP : off) * p.D + (real ? c0 * 8 : 0);
#pragma unroll
      for (int i = 0; i < STRIP / RSTEP; ++i) {
        const int r = r0l + i * RSTEP;
        cp_async16(to + r * (DP * 2) + ((c0 ^ (r & 7)) << 4), src + (int64_t)r * p.D, real);
      }
      if constexpr (VT) {                                                  // values stored [dim][token of the page]
        const int c = lane & 7, d0 = warp * 32 + (lane >> 3);
        const uint32_t vt = v_ring + stage * (TILE * DP * 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = d0 + i * 4;
          cp_async16(vt + d * 128 + ((c ^ (d & 7)) << 4), v + d * TILE + c * 8, true);
        }
      } else {
        const T* sv = v + (int64_t)off * p.D + (real ? c0 * 8 : 0);
#pragma unroll
        for (int i = 0; i < STRIP / RSTEP; ++i) {
          const int r = r0l + i * RSTEP;
          cp_async16(to + F::STRIP_BYTES + r * (DP * 2) + ((c0 ^ (r & 7)) << 4), sv + (int64_t)r * p.D, real);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(i);

  const int r0 = lane >> 2, q0 = (lane & 3) * 2;
  const int mi = lane >> 3, l7 = lane & 7;
  int s = t0 * 4 + warp, turn = 0;
  uint32_t q[KD][NT][2];
  auto load_q = [&]() {
    const int g0 = row.hc % p.chunks * 16, G = min(p.G - g0, 16);
    const T* qp = reinterpret_cast<const T*>(p.q) + row.b * p.q_stride + (int64_t)(row.hc / p.chunks * p.G + g0) * p.D;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < KD; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = k * 16 + j * 8 + q0;
          q[k][nt][j] = nt * 8 + r0 < G && d < p.D ? *reinterpret_cast<const uint32_t*>(qp + (nt * 8 + r0) * p.D + d) : 0u;
        }
  };
  load_q();
  while (true) {
    const int seg_end = min(row.end, t1) * 4;
    const int g0 = row.hc % p.chunks * 16, G = min(p.G - g0, 16);
    if (!FUSED) n = lens[row.b];
    float o[KD][NT][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < KD; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][nt][j] = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) { m_run[nt][u] = -INFINITY; l_run[nt][u] = 0.f; }
    }
    for (; s < seg_end; s += WARPS) {
      const int stage = turn;
      turn = turn + 1 == STAGES ? 0 : turn + 1;
      cp_async_wait<STAGES - 2>();
      if constexpr (VT) __syncthreads();
      else __syncwarp();
      fetch(stage == 0 ? STAGES - 1 : stage - 1);                          // into the stage of the strip before, which the whole warp (VT: all warps) has read
      const int tok = (s - row.begin * 4) * STRIP;
      if (tok < n) {
        const uint32_t ks = ring + stage * STAGE, vs = VT ? v_ring + stage * (TILE * DP * 2) : ks + F::STRIP_BYTES;
        float sc[NT][4], sd[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[nt][i] = sd[nt][i] = 0.f;
        const uint32_t k_row = ks + ((mi & 1) * 8 + l7) * (DP * 2);
#pragma unroll
        for (int k = 0; k < KD; ++k) {
          uint32_t a[4];
          ldsm4(a, k_row + (((k * 2 + (mi >> 1)) ^ l7) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<T>(k & 1 ? sd[nt] : sc[nt], a, q[k][nt][0], q[k][nt][1]);
        }
        const bool cut = tok + STRIP > n;
        const bool in[2] = {!cut || tok + r0 < n, !cut || tok + 8 + r0 < n};
        float* raw = FUSED ? raw_s + (tok - t0 * TILE) * p.G : p.raw + ((int64_t)(row.b * p.Hkv + row.hc / p.chunks) * p.raw_rows + tok) * p.G + g0;
        uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float mx[2], alpha[2];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = sc[nt][i] + sd[nt][i];
            sc[nt][i] = in[i >> 1] ? (CAP ? prompt::cap_any(x * p.ku, p.c2) : x * p.scale_log2) : -INFINITY;
            const int g = nt * 8 + q0 + (i & 1);
            if (g < G) raw[(int64_t)(r0 + (i >> 1) * 8) * p.G + g] = sc[nt][i];
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) mx[u] = fmaxf(sc[nt][u], sc[nt][2 + u]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1)
#pragma unroll
            for (int u = 0; u < 2; ++u) mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], x));
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float was = m_run[nt][u];
            const float at = mx[u] - SHIFT;
            const bool up = at > was + 8.f || (was == -INFINITY && at > -INFINITY);            // else the old reference stays
            alpha[u] = up && was != -INFINITY ? ex2(was - at) : 1.f;
            m_run[nt][u] = up ? at : was;
          }
          if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int i = 0; i < KD; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[i][nt][j] *= alpha[j & 1];
            l_run[nt][0] *= alpha[0]; l_run[nt][1] *= alpha[1];
          }
          const float ref[2] = {m_run[nt][0] == -INFINITY ? 0.f : m_run[nt][0], m_run[nt][1] == -INFINITY ? 0.f : m_run[nt][1]};
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const float x = ex2(sc[nt][2 * t] - ref[0]), y = ex2(sc[nt][2 * t + 1] - ref[1]);
            l_run[nt][0] += x; l_run[nt][1] += y;
            const uint32_t hi = pack2<T>(x, y);
            ph[nt][t] = turn8(hi);
            const float2 back = unpack2<T>(hi);
            pl[nt][t] = turn8(pack2<T>(x - back.x, y - back.y));
          }
        }
        uint32_t keepm[2] = {0xffffffffu, 0xffffffffu};                     // of tokens q0, q0 + 1 of either group of eight
        if (cut) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int t = tok + j * 8 + q0;
            keepm[j] = (t < n ? 0xffffu : 0u) | (t + 1 < n ? 0xffff0000u : 0u);
          }
        }
#pragma unroll
        for (int i = 0; i < KD; ++i) {
          uint32_t a[4];
          if constexpr (VT) {
            const int d = i * 16 + (mi & 1) * 8 + l7;
            ldsm4(a, vs + d * 128 + (((warp * 2 + (mi >> 1)) ^ (d & 7)) << 4));
          } else {
            // stored [token][dim], turned by the load: matrices (dims 0-7, tokens 0-7), (dims 8-15, tokens 0-7), (dims 0-7, tokens 8-15), ...
            const int t = (mi >> 1) * 8 + l7;
            ldsm4_t(a, vs + t * (DP * 2) + (((i * 2 + (mi & 1)) ^ (t & 7)) << 4));
          }
          if (cut) {           // slots behind the sequence may hold what a weight of 0 does not cancel
            a[0] &= keepm[0]; a[1] &= keepm[0]; a[2] &= keepm[1]; a[3] &= keepm[1];
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816<T>(o[i][nt], a, ph[nt][0], ph[nt][1]);
            mma16816<T>(o[i][nt], a, pl[nt][0], pl[nt][1]);
          }
        }
      }
    }
    // ---- the warps' results of the segment: lanes hold the same places in every warp, so the upper half of the warps hands its registers over
    float* part = FUSED ? part_s : p.part + (int64_t)(row.index + blockIdx.x) * 16 * PD;
    const bool empty = !FUSED && max(row.begin, t0) >= row.begin + (n + TILE - 1) / TILE;      // nothing but the row's further slots
    if (!FUSED && !empty && row.begin >= t0 && threadIdx.x == 0)
      p.info[row.index] = make_int2(blockIdx.x, (row.begin + (n + TILE - 1) / TILE - 1) / per - blockIdx.x + 1);
    const bool more = !FUSED && row.end < t1;
    if (more) {                              // (the next row's queries are on their way meanwhile)
      next_row(first, H, row);
      load_q();
    }
    if (!empty)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l_run[nt][u] += __shfl_xor_sync(0xffffffffu, l_run[nt][u], x);
#pragma unroll
      for (int half = WARPS / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (warp >= half && warp < 2 * half) {
          float* to = exch + (warp - half) * F::REGS * 32 + lane;
#pragma unroll
          for (int i = 0; i < KD; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) to[(i * 4 + j) * 32] = o[i][nt][j];
#pragma unroll
          for (int u = 0; u < 2; ++u) { to[(KD * 4 + u) * 32] = m_run[nt][u]; to[(KD * 4 + 2 + u) * 32] = l_run[nt][u]; }
        }
        __syncthreads();
        if (warp < half) {
          const float* from = exch + warp * F::REGS * 32 + lane;
          float fa[2], fb[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float mb = from[(KD * 4 + u) * 32], top = fmaxf(m_run[nt][u], mb);
            fa[u] = m_run[nt][u] == -INFINITY ? 0.f : ex2(m_run[nt][u] - top);
            fb[u] = mb == -INFINITY ? 0.f : ex2(mb - top);
            m_run[nt][u] = top;
            l_run[nt][u] = l_run[nt][u] * fa[u] + from[(KD * 4 + 2 + u) * 32] * fb[u];
          }
#pragma unroll
          for (int i = 0; i < KD; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][nt][j] = o[i][nt][j] * fa[j & 1] + from[(i * 4 + j) * 32] * fb[j & 1];
        }
      }
      if (warp == 0) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int g = nt * 8 + q0 + u;
          if (g < G) {
            float* to = part + g * PD;
#pragma unroll
            for (int i = 0; i < KD; ++i) {
              if (i * 16 + r0 < p.D) to[i * 16 + r0] = o[i][nt][u];
              if (i * 16 + 8 + r0 < p.D) to[i * 16 + 8 + r0] = o[i][nt][2 + u];
            }
            if (r0 == 0) { to[p.D] = m_run[nt][u]; to[p.D + 1] = l_run[nt][u]; }
          }
        }
      }
    }
    if (!more) break;
  }
  cp_async_wait<0>();
  if constexpr (FUSED) {
    cluster_sync();
    const uint32_t parts_at = smem_u32(part_s);
    const int h = row.hc;
    for (int g = warp; g < p.G; g += WARPS) {            // a warp: log-sum-exp of a head, its parts and the sink
      const uint32_t at = parts_at + (g * PD + p.D) * 4;
      const float m0 = lane < p.parts ? ld_dsmem_f32(dsmem_addr(at, lane)) : -INFINITY, l0 = lane < p.parts ? ld_dsmem_f32(dsmem_addr(at + 4, lane)) : 0.f;
      const float sink = p.sinks ? p.sinks[h * p.G + g] * LOG2E : -INFINITY;
      const float m = warp_max(fmaxf(m0, sink)), top = m == -INFINITY ? 0.f : m;
      const float l = warp_sum(l0 * ex2(m0 - top)) + (p.sinks ? ex2(sink - top) : 0.f);
      const float lse = l > 0.f ? top + log2f(l) : INFINITY;                // no key and no sink: weights of 0
      if (lane < 8) factor_s[g * 9 + lane] = ex2(m0 - lse);
      if (lane == 8) factor_s[g * 9 + 8] = lse;
    }
    __syncthreads();
    for (int i = rank * F::THREADS + threadIdx.x; i < p.G * p.D; i += p.parts * F::THREADS) {
      const int g = i / p.D, d = i % p.D;
      float x[8], acc = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) x[c] = c < p.parts ? ld_dsmem_f32(dsmem_addr(parts_at + (g * PD + d) * 4, c)) : 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) acc += x[c] * factor_s[g * 9 + c];
      reinterpret_cast<T*>(p.out)[row.b * p.out_stride + (int64_t)h * p.G * p.D + i] = from_f32<T>(acc);
    }
    float* sc = p.scores + row.b * p.sc_req + h * p.sc_head;
    for (int k = t0 * TILE + threadIdx.x; k < min(t1 * TILE, n); k += F::THREADS) {
      float w = 0.f;
      for (int g = 0; g < p.G; ++g) w += ex2(raw_s[(k - t0 * TILE) * p.G + g] - factor_s[g * 9 + 8]);
      sc[k] += w;
    }
    cluster_sync();                                      // the others may still read this CTA's part
  }
}

// Grid (blocks of p.block keys, kv heads, requests): joins a row's outputs and adds the weights of its keys.  It is a chain of reads from memory (the row's
// parts, then what they say), so what does not wait for another read is read first, and there are as many blocks as the SMs hold at a time.
constexpr int JOIN = 256, JOINERS = 4, U = 4, KEYS = U * JOIN, FACTORS = 32;      // JOINERS: blocks of an SM
template <typename T>
__global__ void __launch_bounds__(JOIN, JOINERS) join_kernel(const Params p) {
  extern __shared__ float join_smem[];                // of the G heads: log-sum-exp in powers of two, then a factor for each of the first FACTORS parts
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.z, h = blockIdx.y, H = p.Hkv * p.chunks, lane = threadIdx.x & 31, w = threadIdx.x >> 5, PD = p.D + 2;
  const int n = rows_of(p, b), end = min(((int)blockIdx.x + 1) * p.block, n);
  int key0 = blockIdx.x * p.block;
  // the keys' scores so far, and what the first four heads say of them
  const float* raw = p.raw + (int64_t)(b * p.Hkv + h) * p.raw_rows * p.G;
  float* sc = p.scores + b * p.sc_req + h * p.sc_head;
  const bool four = p.G % 4 == 0;
  float old[U];
  float4 x4[U];
  auto read_keys = [&]() {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = key0 + u * JOIN + threadIdx.x;
      old[u] = k < end ? sc[k] : 0.f;
      x4[u] = four && k < end ? *reinterpret_cast<const float4*>(raw + (int64_t)k * p.G) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  read_keys();
  // parts of a head: segments of CTAs, at row + CTA
  const int64_t step = (int64_t)16 * PD;
  auto parts = [&](int g, int& count) -> const float* {
    const int row = b * H + h * p.chunks + g / 16;
    const int2 at = n > 0 ? p.info[row] : make_int2(0, 0);
    count = at.y;
    return p.part + ((int64_t)(row + at.x) * 16 + g % 16) * PD;
  };
  float* factors = join_smem + ((p.G + 3) & ~3);
  for (int g = w; g < p.G; g += JOIN / 32) {          // a warp: log-sum-exp of a head, its parts and the sink
    int count;
    const float* x = parts(g, count) + p.D;
    const float sink = p.sinks ? p.sinks[h * p.G + g] * LOG2E : -INFINITY;
    const float m0 = lane < count ? x[lane * step] : -INFINITY, l0 = lane < count ? x[lane * step + 1] : 0.f;
    float m = fmaxf(m0, sink);
    for (int c = 32 + lane; c < count; c += 32) m = fmaxf(m, x[c * step]);
    m = warp_max(m);
    const float top = m == -INFINITY ? 0.f : m;
    float l = l0 * ex2(m0 - top);
    for (int c = 32 + lane; c < count; c += 32) l += x[c * step + 1] * ex2(x[c * step] - top);
    l = warp_sum(l) + (p.sinks ? ex2(sink - top) : 0.f);
    const float lse = l > 0.f ? top + log2f(l) : INFINITY;                  // no key and no sink: weights of 0
    if (lane == 0) join_smem[g] = lse;
    factors[g * FACTORS + lane] = ex2(m0 - lse);
  }
  // the thread's first output: its first parts
  constexpr int AHEAD = 8;
  float o[AHEAD];
  auto read_parts = [&](const float* x, int from, int count) {
#pragma unroll
    for (int c = 0; c < AHEAD; ++c) o[c] = from + c < count ? x[(from + c) * step] : 0.f;
  };
  const int first = blockIdx.x * JOIN + threadIdx.x;
  if (first < p.G * p.D) {
    int count;
    const float* x = parts(first / p.D, count);
    read_parts(x + first % p.D, 0, count);
  }
  __syncthreads();
  for (int i = first; i < p.G * p.D; i += gridDim.x * JOIN) {
    const int g = i / p.D;
    int count;
    const float* x = parts(g, count) + i % p.D;
    float acc = 0.f;
    for (int from = 0; from < count; from += AHEAD) {
      if (from > 0 || i != first) read_parts(x, from, count);
#pragma unroll
      for (int c = 0; c < AHEAD; ++c) {
        const int at = from + c;
        if (at < count) acc += o[c] * (at < FACTORS ? factors[g * FACTORS + at] : ex2(x[at * step + p.D - i % p.D] - join_smem[g]));
      }
    }
    reinterpret_cast<T*>(p.out)[b * p.out_stride + (int64_t)h * p.G * p.D + i] = from_f32<T>(acc);
  }
  while (key0 < end) {
    float sum[U] = {0.f, 0.f, 0.f, 0.f};
    if (four) {
      for (int g = 0; g < p.G; g += 4) {
        const float4 l = *reinterpret_cast<const float4*>(join_smem + g);
        if (g > 0) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int k = key0 + u * JOIN + threadIdx.x;
            if (k < end) x4[u] = *reinterpret_cast<const float4*>(raw + (int64_t)k * p.G + g);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) sum[u] += (ex2(x4[u].x - l.x) + ex2(x4[u].y - l.y)) + (ex2(x4[u].z - l.z) + ex2(x4[u].w - l.w));
      }
    } else {
      for (int g = 0; g < p.G; ++g) {
        const float l = join_smem[g];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int k = key0 + u * JOIN + threadIdx.x;
          if (k < end) sum[u] += ex2(raw[(int64_t)k * p.G + g] - l);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = key0 + u * JOIN + threadIdx.x;
      if (k < end) sc[k] = old[u] + sum[u];
    }
    key0 += KEYS;
    if (key0 < end) read_keys();
  }
}

constexpr int FUSED_TILES = 4;                           // of a CTA, at most, where a cluster has a row
template <typename F> constexpr int EXCH_BYTES = F::WARPS / 2 * F::REGS * 128;

// `clusters`: nothing is launched, the clusters of a row that the device runs at a time are counted.
template <typename T, int DP, int NT, bool VT, bool CAP>
static int launch(const Params& p, cudaStream_t st, int* clusters) {
  using F = Form<DP>;
  if constexpr (DP <= 128) if (p.parts > 0) {
    auto k = decode_kernel<T, DP, NT, VT, CAP, true>;
    constexpr int MOST = F::RING + EXCH_BYTES<F> + (16 * (DP + 2 + 9) + 4 + FUSED_TILES * TILE * 16) * 4;
    static std::atomic<uint64_t> devices{0};
    if (vb_allow_smem(reinterpret_cast<const void*>(k), MOST, devices) != cudaSuccess) return (int)cudaGetLastError();
    const int tiles = (p.max_rows + TILE - 1) / TILE, per = (tiles + p.parts - 1) / p.parts;
    const size_t smem = F::RING + EXCH_BYTES<F> + (size_t)(p.G * (p.D + 2 + 9) + 4 + per * TILE * p.G) * 4;
    if (clusters) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr = {};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = p.parts; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
      cfg.gridDim = dim3(p.parts); cfg.blockDim = dim3(F::THREADS); cfg.dynamicSmemBytes = smem; cfg.attrs = &attr; cfg.numAttrs = 1;
      return (int)cudaOccupancyMaxActiveClusters(clusters, k, &cfg);
    }
    vb_launch_parts(k, dim3(p.B * p.Hkv * p.parts), dim3(F::THREADS), smem, st, (unsigned)p.parts, p);
    return (int)cudaGetLastError();
  }
  if (clusters) return -1;
  auto k = decode_kernel<T, DP, NT, VT, CAP, false>;
  static std::atomic<uint64_t> devices{0};
  if (vb_allow_smem(reinterpret_cast<const void*>(k), F::SMEM, devices) != cudaSuccess) return (int)cudaGetLastError();
  vb_launch(k, dim3(p.ctas), dim3(F::THREADS), (size_t)F::SMEM, st, p);
  vb_launch(join_kernel<T>, dim3((p.max_rows + p.block - 1) / p.block, p.Hkv, p.B), dim3(JOIN), (size_t)(((p.G + 3) & ~3) + p.G * FACTORS) * 4, st, p);
  return (int)cudaGetLastError();
}
template <typename T, int DP, bool VT>
static int pick(const Params& p, bool cap, cudaStream_t st, int* clusters) {
  if (p.G > 8) return cap ? launch<T, DP, 2, VT, true>(p, st, clusters) : launch<T, DP, 2, VT, false>(p, st, clusters);
  return cap ? launch<T, DP, 1, VT, true>(p, st, clusters) : launch<T, DP, 1, VT, false>(p, st, clusters);
}
template <typename T>
static int go(const Params& p, bool vt, bool cap, cudaStream_t st, int* clusters = nullptr) {
  if (vt) return p.D == 128 ? pick<T, 128, true>(p, cap, st, clusters) : -2;
  if (p.D <= 64) return pick<T, 64, false>(p, cap, st, clusters);
  if (p.D <= 128) return pick<T, 128, false>(p, cap, st, clusters);
  return pick<T, 256, false>(p, cap, st, clusters);
}

}  // namespace sdec

// Into `clusters`: how many clusters of `parts` CTAs, each with a row of up to `tiles` tiles of a kv head with G query heads, the device runs at a time.
EXPORT int vb_scored_clusters(int G, int D, int tiles, int parts, int vt, int cap, int dtype, int* clusters) {
  using namespace sdec;
  if (dtype == DT_F32 || D % 8 || D > 128 || G < 1 || G > 16 || parts < 2 || parts > 8 || tiles < 1 || tiles > FUSED_TILES * parts) return -1;
  Params p{};
  p.G = G; p.D = D; p.max_rows = tiles * TILE; p.parts = parts;
  return dtype == DT_BF16 ? go<__nv_bfloat16>(p, vt != 0, cap != 0, nullptr, clusters) : go<__half>(p, vt != 0, cap != 0, nullptr, clusters);
}

// `ws`: for rows = group Hkv ceil(G / 16), (rows + ctas) 16 (D + 2) + group Hq ceil(max_rows / 64) 64 + 2 rows floats.  group: requests of a launch, up to 512.
// extra: tiles that a row counts for beside its own.  parts: CTAs of a cluster that has a row (one kernel, no `ws`); 0: equal runs.  max_rows: rows of a request
// that the block table and the scores have room for.
EXPORT int vb_scored_decode(const void* q, const void* cache, int64_t num_blocks, const int* block_table, const int* seq_lens, void* out, float* scores,
                            const float* sinks, float* ws, int B, int Hq, int Hkv, int D, int BS, int max_rows, int64_t q_stride, int64_t out_stride,
                            int64_t bt_stride, int64_t sc_req, int64_t sc_head, int ctas, int sms, int extra, int parts, int group, float scale, float soft_cap, int vt, int dtype, cudaStream_t st) {
  using namespace sdec;
  if (B <= 0) return 0;
  if (group < 1 || group > MAX_REQUESTS) return -1;
  if (dtype == DT_F32 || D % 8 || D > 256 || BS % 16 || Hq % Hkv || ctas < 1 || max_rows < 1 || parts < 0 || parts > 8) return -1;
  if (parts > 0 && (parts < 2 || D > 128 || Hq / Hkv > 16 || B > group || (max_rows + TILE - 1) / TILE > FUSED_TILES * parts)) return -1;
  Params p;
  p.Hkv = Hkv; p.G = Hq / Hkv; p.D = D; p.BS = BS; p.max_rows = max_rows; p.chunks = (p.G + 15) / 16; p.extra = extra; p.parts = parts;
  p.q_stride = q_stride; p.out_stride = out_stride; p.bt_stride = bt_stride; p.sc_req = sc_req; p.sc_head = sc_head;
  p.num_blocks = num_blocks; p.cache = cache; p.sinks = sinks;
  p.raw_rows = (max_rows + TILE - 1) / TILE * TILE;
  p.scale_log2 = scale * LOG2E;
  p.ku = soft_cap > 0.f ? scale / soft_cap : 0.f; p.c2 = soft_cap * LOG2E;
  for (int b0 = 0; b0 < B; b0 += group) {
    p.B = B - b0 < group ? B - b0 : group;
    p.q = reinterpret_cast<const char*>(q) + b0 * q_stride * 2;
    p.out = reinterpret_cast<char*>(out) + b0 * out_stride * 2;
    p.block_table = block_table + b0 * bt_stride;
    p.seq_lens = seq_lens + b0;
    p.scores = scores + b0 * sc_req;
    const int64_t rows = (int64_t)p.B * Hkv * p.chunks, tiles = rows * ((max_rows + TILE - 1) / TILE + p.extra);
    if (tiles >= (1 << 29)) return -3;                 // flat strip numbers are 32 bits
    p.ctas = ctas < tiles ? ctas : (int)tiles;
    const int64_t blocks = JOINERS * (int64_t)sms / ((int64_t)p.B * Hkv), most = (max_rows + JOIN - 1) / JOIN;
    p.block = (int)((most + (blocks < 1 ? 1 : blocks) - 1) / (blocks < 1 ? 1 : blocks)) * JOIN;
    p.part = ws;
    p.raw = ws + (rows + p.ctas) * 16 * (D + 2);
    p.info = reinterpret_cast<int2*>(p.raw + (int64_t)p.B * Hq * p.raw_rows);
    const int rc = dtype == DT_BF16 ? go<__nv_bfloat16>(p, vt != 0, soft_cap > 0.f, st) : go<__half>(p, vt != 0, soft_cap > 0.f, st);
    if (rc) return rc;
  }
  return 0;
}
