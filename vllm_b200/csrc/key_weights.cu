// The weights that a prompt's query rows give to the cached keys, added to the keys' scores:
//
//   scores[b, h, k] += sum over the request's (last) query rows t >= k and the G query heads g of kv head h of e^(c(scale q[t, g] . K[k]) - lse[t, g])
//
// lse is that of the attention before, so a weight needs no second look at its row.  Keys are the rows of tcgen05 products of 128 keys and up to 128
// (token, head) pairs: a thread owns a key (a lane of tensor memory) and half of the columns, and the sum stays in its registers until the key's
// last query.  256 keys (two products, half the reads of queries) of a kv head are a block; the blocks' query tiles, all in one order, are dealt to
// the CTAs in equal runs, as a prompt's first keys have the most queries and a short prompt has few blocks.  Blocks that end up in
// several CTAs are joined by a second kernel, in order: no atomics, the same result in every run.
//
// An exponential per (token, head, key) bounds it: 16 a cycle and SM on the special-function unit, twice the time of the products of 128
// dimensions.  One in eight is a polynomial on the multiply-add units instead.  us for 8000 tokens of 32 / 8 heads (of 128) and for 512 behind 25000
// twice of 16 / 4 (of 64): a CTA per block with 8 warps for both key tiles 410 and 196; runs of equal length and 16 warps 442 and 170, where
// packed polynomials cost more instructions than exponentials time; tiles of 256 columns, each key tile with its own warps 354 and 144; the
// log-sum-exps in the products 341 and 138; one in eight exponentials a polynomial 328 and 132 (one in four 337 and 138);
// half of a piece summed while the other half comes out of tensor memory 312 and 127 (at 1965 MHz; under the power cap, after some tenths of a second, 345).
#include "attention_prompt.cuh"
#include "device_once.h"

namespace kweights {

constexpr int KEYS = 256, TILE = 128, COLS = 256;
constexpr int SUMMERS = 16, NUM_THREADS = 640;     // warp 0: copies, 1: products, 2 and 3: log-sum-exps, 4..11 and 12..19: sums
constexpr int MAX_REQUESTS = 1024;          // of a launch: their first tiles lie in shared memory
constexpr int BLK = TILE * 128;             // [128 rows x 64 values], 16 KB
constexpr float LOG2E = 1.4426950408889634f;

struct Params {
  const int* block_table;
  const int* seq_lens;
  const int* qsl;            // null: one row per request
  const float* lse;          // [T, Hq]
  float* scores;
  float* part;               // [CTA][2][KEYS]: sums of a block that began in an earlier CTA; of one that goes on in the next
  int4* info;                // [CTA]: where that begins which it continues as the first: request, kv head, block (-1: nothing), its CTAs from here on
  int* error;                // raised when a wait ran into its limit
  int64_t bt_stride, sc_req, sc_head, num_blocks;
  int B, row0, T, Hq, Hkv, G, TQ, D, BS, max_rows, last, box_rows, whole;      // TQ: tokens of a tile, a power of 2; whole: blocks are not split
  float one, lse_in;       // what the parts of a log-sum-exp are multiples of; -1 / (scale one)
  float scale_log2, ku, c2;               // capped: scale / cap, cap log2(e)
};

// What a request needs: the tiles of tokens lie side by side up to its last token.  Key block i has the last tiles(i) of them.
struct Request {
  int len, q_end, q_lo, c0, tf, f, nb;      // c0: tiles of len tokens, tf: of the tokens that count, f: key blocks that all of those see
  VB_DEVICE void load(const Params& p, int b) {
    len = max(p.seq_lens[b], 0);
    const int n = min(len, p.max_rows), q_begin = p.qsl ? p.qsl[b] : p.row0 + b;
    q_end = min(p.qsl ? p.qsl[b + 1] : q_begin + 1, p.T);
    int count = min(q_end - q_begin, len);
    if (p.last > 0) count = min(count, p.last);
    q_lo = q_end - count;
    if (count <= 0 || n <= 0) { nb = f = tf = c0 = 0; return; }
    c0 = (len + p.TQ - 1) / p.TQ;
    tf = (count + p.TQ - 1) / p.TQ;
    nb = (n + KEYS - 1) / KEYS;
    f = min(nb, (c0 - tf) / (KEYS / p.TQ) + 1);
  }
  VB_DEVICE int tiles(const Params& p, int i) const { return i < f ? tf : c0 - KEYS / p.TQ * i; }
  VB_DEVICE int before(const Params& p, int i) const {       // tiles of the blocks in front of block i
    if (i <= f) return i * tf;
    return (int)((int64_t)f * tf + (int64_t)(i - f) * c0 - (int64_t)(f + i - 1) * (i - f) / 2 * (KEYS / p.TQ));
  }
};

// A run of tiles of one block: request b, kv head h, key block i, tiles [j, j + n) of its count
struct Segment : Request {
  int b, h, i, j, n, count;
  VB_DEVICE void start(const Params& p, const int* first, int s, int s1) {          // s < first[B]
    int lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= s) lo = mid; else hi = mid - 1;
    }
    b = lo;
    load(p, b);
    const int per_head = (first[b + 1] - first[b]) / p.Hkv;                          // > 0: the last request that begins at or in front of s
    s -= first[b];
    h = s / per_head;
    s -= h * per_head;
    lo = 0; hi = nb - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before(p, mid) <= s) lo = mid; else hi = mid - 1;
    }
    i = lo;
    j = s - before(p, i);
    count = tiles(p, i);
    n = min(count - j, s1);
  }
  VB_DEVICE void next(const Params& p, const int* first, int rest) {                // rest: tiles that are left, > 0
    if (++i == nb) {
      i = 0;
      if (++h == p.Hkv) {
        h = 0;
        do { ++b; } while (first[b + 1] == first[b]);
        load(p, b);
      }
    }
    j = 0;
    count = tiles(p, i);
    n = min(count, rest);
  }
};

// first[b]: tiles of the requests in front of request b; first[B]: of all
VB_DEVICE void scan_requests(const Params& p, int* first, int* warp_sums) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    int mine = 0;
    if (b < p.B) {
      Request r;
      r.load(p, b);
      mine = r.before(p, r.nb) * p.Hkv;
    }
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

template <int KB> struct Form {              // KB: blocks of 64 dimensions
  static constexpr int QS = KB == 1 ? 4 : KB == 2 ? 2 : 1;
  static constexpr int COLUMNS = KB <= 3 ? COLS : COLS / 2;                   // of a product
  static constexpr int K_BYTES = 2 * KB * BLK, Q_BYTES = KB * (COLUMNS * 128);
  static constexpr int NEED = K_BYTES + QS * Q_BYTES + TILE * 32 + 2 * COLS * 32 + 2 * COLS * 4 + KEYS * 4 + (MAX_REQUESTS + 1 + 32) * 4 + 32 * 8 + 16 + 1024;
  static constexpr int SMEM = NEED > 116 * 1024 ? NEED : 116 * 1024;         // one CTA per SM: it has all of tensor memory
};

VB_DEVICE float rcp(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// Capped scores, c2 tanh(x): up to |x| = 1 by the polynomial of the attention kernels, off by a part of x where 1 - 2 / (1 + e^(2 x)) is off by a part of the cap
// (2e-6 of a weight for a cap of 50); the log-sum-exps are sums of the same values then.  8000 tokens of 32 / 8 heads, 512 behind 25000 twice of 16 / 4: 721 and
// 286 us where no score of a piece is above the cap, 1442 and 565 where some are everywhere (1 - 2 / (1 + e^(2 x)) for all: 779 and 316).
VB_DEVICE float cap_far(float x, float c2) { return copysignf(fmaf(-2.f, rcp(1.f + ex2(fabsf(x) * 2.8853900817779268f)), 1.f), x) * c2; }
VB_DEVICE float cap_near_or_far(float x, float c2) { return fabsf(x) <= 1.f ? prompt::cap_small(x, c2) : cap_far(x, c2); }

// Other scores: a column gets sixteen more dimensions, three of which hold -lse / scale in parts of 16 bits, the keys' are constant.  The product is
// then what the exponential takes but for a factor: no log-sum-exps out of shared memory, where 128-bit reads by all threads and the operands of the
// products want the same bandwidth.  fp16: they are multiples of a power of two that makes them lse / 4 to lse / 8, far from either end of the type.  Where they do
// not fit all the same (scales next to 0) the product gets zeros and the sum the log-sum-exp, as where scores are capped.  They are added a little behind the middle
// of a product: its sums are cut towards 0, and half of them are then above 0 and half below for the keys with much weight.  Relative error of the weights of 300
// tokens 4.4e-7 with them last, 8.6e-7 first, 1.3e-7 so (heads of 128); of 900 with heads of 256 1.1e-6, 2.5e-6 and 1.8e-7; 32-bit multiplications and additions
// have 1.2e-7.
template <typename T> constexpr float MOST = DTypeOf<T>::v == DT_F16 ? 60000.f : 1e38f;          // of a part
// rows of 32 bytes, 8-row groups 256 bytes apart, SWIZZLE_32B
VB_DEVICE uint64_t umma_desc_sw32(const void* smem_tile) {
  return (uint64_t)((smem_u32(smem_tile) & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(256 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)6 << 61;
}

// 2^x: x = n + f, |f| <= 1/2 (n by the rounding of an addition), 2^f by the polynomial that interpolates it at the Chebyshev points (2.2e-7 of it at most,
// 0.8e-7 in the mean), n added to its exponent.  2^-126 below, 2^127 above.
VB_DEVICE float ex2_poly(float x) {
  x = fminf(fmaxf(x, -126.f), 127.f);
  const float t = x + 12582912.f, f = x - (t - 12582912.f);
  float r = 0.0013390863314270973f;
  r = fmaf(r, f, 0.009676031768321991f);
  r = fmaf(r, f, 0.055503569543361664f);
  r = fmaf(r, f, 0.2402210682630539f);
  r = fmaf(r, f, 0.6931471824645996f);
  r = fmaf(r, f, 1.0000001192092896f);
  return __int_as_float(__float_as_int(r) + (__float_as_int(t) << 23));
}

// tmem_ld_wait for these registers: no use of them moves in front of it
VB_DEVICE void wait_for(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :: "memory");
}
VB_DEVICE void wait_for(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29])
               :: "memory");
  asm volatile("" : "+r"(r[30]), "+r"(r[31]));
}

template <typename T, int KB, bool CAP>
__global__ void __launch_bounds__(NUM_THREADS, 1)
weights_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const Params p) {
  using F = Form<KB>;
  constexpr int QS = F::QS;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* k_smem = smem;                                  // [key tile][KB]
  unsigned char* q_smem = k_smem + F::K_BYTES;                   // [stage][KB]
  unsigned char* one_smem = q_smem + QS * F::Q_BYTES;            // [TILE][16]: what a column's sixteen further dimensions are multiplied with
  unsigned char* aug_smem = one_smem + TILE * 32;                // [slot][COLS][16]: those: less the log-sum-exp, in three parts
  float* lse_smem = reinterpret_cast<float*>(aug_smem + 2 * COLS * 32);          // [slot][COLS]: less what the product has not of the log-sum-exp, in powers of two
  float* exch = lse_smem + 2 * COLS;                             // [KEYS]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(exch + KEYS);   // [key tile]
  uint64_t* k_empty = k_full + 2;
  uint64_t* s_full = k_empty + 2;            // [key tile]
  uint64_t* s_empty = s_full + 2;
  uint64_t* l_full = s_empty + 2;            // [slot]
  uint64_t* l_empty = l_full + 2;
  uint64_t* q_full = l_empty + 2;
  uint64_t* q_empty = q_full + QS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_empty + QS);
  int* first = reinterpret_cast<int*>(tmem_slot + 4);
  int* warp_sums = first + MAX_REQUESTS + 1;
  __shared__ int odd[2];                     // of a tile: some column gives no weights, or has its log-sum-exp outside the product

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int budget = MBAR_BUDGET;
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_q); tma_prefetch_desc(&tmap_k);
    for (int s = 0; s < QS; ++s) { mbar_init(&q_full[s], 1); mbar_init(&q_empty[s], 1); }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1);
      mbar_init(&s_full[s], 1); mbar_init(&s_empty[s], SUMMERS / 2);
      mbar_init(&l_full[s], 1); mbar_init(&l_empty[s], SUMMERS + 1);
    }
    mbar_fence_init();
  }
  const int used = p.TQ * p.G, pieces = (used + 31) / 32;        // columns, and groups of 32 of them
  if (used < pieces * 32)                                        // columns that no head has: zeros
    for (int i = threadIdx.x; i < QS * F::Q_BYTES / 16; i += NUM_THREADS) reinterpret_cast<uint4*>(q_smem)[i] = make_uint4(0, 0, 0, 0);
  if (!CAP) {
    for (int i = threadIdx.x; i < 2 * COLS * 2; i += NUM_THREADS) reinterpret_cast<uint4*>(aug_smem)[i] = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < TILE * 2; i += NUM_THREADS) {
      const int row = i >> 1;                                    // (pieces of 16 bytes; those of rows 4 to 7 of eight change places)
      const bool front = ((i ^ (row >> 2)) & 1) == 0;
      reinterpret_cast<uint4*>(one_smem)[i] = front ? make_uint4(pack2<T>(p.one, p.one), pack2<T>(p.one, 0.f), 0, 0) : make_uint4(0, 0, 0, 0);
    }
  }
  fence_proxy_async();
  pdl_wait();
  // All of tensor memory: behind the kernel in front, which may allocate its own only after a wait of its own on the same SM, and before the next may begin.
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    pdl_trigger();
  }
  scan_requests(p, first, warp_sums);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;                              // scores of key tile t: columns t * COLS ..
  const int total = first[p.B], per = (total + gridDim.x - 1) / gridDim.x;
  int s0 = min((int)blockIdx.x * per, total), s1 = min(s0 + per, total);
  if (p.whole) {                                                 // the blocks that begin in the run
    Segment g;
    if (s0 < total) { g.start(p, first, s0, 1); if (g.j > 0) s0 += g.count - g.j; }
    if (s1 < total) { g.start(p, first, s1, 1); if (g.j > 0) s1 += g.count - g.j; }
  }

  if (p.part && s0 >= s1 && threadIdx.x == 0) p.info[blockIdx.x] = make_int4(0, 0, -1, 0);
  if (s0 < s1) {
    Segment g;
    g.start(p, first, s0, s1 - s0);
    if (p.part && threadIdx.x == 2 * 32)
      p.info[blockIdx.x] = make_int4(g.b, g.h, g.j > 0 && g.j <= per ? g.i : -1, (s0 - g.j + g.count + per - 1) / per - blockIdx.x);
    if (warp == 0) {
      int tile = 0, seg = 0;
      for (int s = s0;;) {
        const int n = min(g.len, p.max_rows), k0 = g.i * KEYS;
        // page numbers of the block's at most 16 boxes, a lane each
        int64_t blk = 0;
        if (lane * p.box_rows < KEYS && k0 + lane * p.box_rows < n) blk = p.block_table[g.b * p.bt_stride + (k0 + lane * p.box_rows) / p.BS];
        if ((uint64_t)blk >= (uint64_t)p.num_blocks) blk = 0;                // (a table may not say that)
        auto load_q = [&](int j) {
          const int qs = tile % QS;
          if (lane == 0) {
            mbar_wait_lim(&q_empty[qs], ((tile / QS) & 1) ^ 1, budget);
            if (budget >= 0) {
              mbar_expect_tx(&q_full[qs], KB * used * 128);
#pragma unroll
              for (int kb = 0; kb < KB; ++kb)
                prompt::tma_load_3d(q_smem + qs * F::Q_BYTES + kb * (F::COLUMNS * 128), &tmap_q, kb * 64, g.h * p.G, g.q_end - (g.count - j) * p.TQ, &q_full[qs]);
            }
          }
          ++tile;
        };
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
          const int boxes = max(0, min(TILE, n - k0 - t * TILE) + p.box_rows - 1) / p.box_rows;
          if (lane == 0) {
            mbar_wait_lim(&k_empty[t], (seg & 1) ^ 1, budget);
            if (budget >= 0) mbar_expect_tx(&k_full[t], boxes * KB * p.box_rows * 128);      // (none of a tile behind the last row: the barrier falls by itself)
          }
          for (int i = 0; i < boxes; ++i) {
            const int r = i * p.box_rows;
            const int at = __shfl_sync(0xffffffffu, (int)blk, (t * TILE + r) / p.box_rows);
            if (lane == 0 && budget >= 0) {
#pragma unroll
              for (int kb = 0; kb < KB; ++kb)
                prompt::tma_load_3d(k_smem + (t * KB + kb) * BLK + r * 128, &tmap_k, kb * 64, (k0 + t * TILE + r) % p.BS, at * 2 * p.Hkv + g.h, &k_full[t]);
            }
          }
          if (t == 0) load_q(g.j);
        }
        for (int j = g.j + 1; j < g.j + g.n; ++j) load_q(j);
        s += g.n;
        ++seg;
        if (s >= s1 || __shfl_sync(0xffffffffu, budget, 0) < 0) break;
        g.next(p, first, s1 - s);
      }
      if (lane == 0 && budget < 0) { mbar_let_land(k_full, 2); mbar_let_land(q_full, QS); }
    } else if (warp == 1) {
      const uint32_t idesc = umma_idesc_f16(TILE, pieces * 32, DTypeOf<T>::v == DT_BF16);
      const uint64_t da = umma_desc_sw128(k_smem), d_one = umma_desc_sw32(one_smem), d_aug = umma_desc_sw32(aug_smem);
      int tile = 0, seg = 0;
      for (int s = s0;;) {
        const bool second = g.i * KEYS + TILE < min(g.len, p.max_rows);
        for (int j = 0; j < g.n; ++j, ++tile) {
          const int qs = tile % QS;
          mbar_wait_lim(&q_full[qs], (tile / QS) & 1, budget);
          const uint64_t db = umma_desc_sw128(q_smem + qs * F::Q_BYTES);
          if (!CAP) mbar_wait_lim(&l_full[tile & 1], (tile >> 1) & 1, budget);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j == 0) mbar_wait_lim(&k_full[t], seg & 1, budget);
            mbar_wait_lim(&s_empty[t], (tile & 1) ^ 1, budget);
            tc_fence_after();
            __syncwarp();
            if (t == 0 || second) {
#pragma unroll
              for (int k = 0; k < KB * 4; ++k) {
                warp_umma_f16(tmem + t * COLS, da + (uint64_t)((t * KB + (k >> 2)) * (BLK / 16) + (k & 3) * 2),
                              db + (uint64_t)((k >> 2) * (F::COLUMNS * 128 / 16) + (k & 3) * 2), idesc, k != 0);
                if (!CAP && k == KB * 2 + KB / 2) warp_umma_f16(tmem + t * COLS, d_one, d_aug + (uint64_t)((tile & 1) * (COLS * 32 / 16)), idesc, 1);
              }
            }
            warp_umma_commit(&s_full[t]);
            if (j == g.n - 1) warp_umma_commit(&k_empty[t]);
          }
          warp_umma_commit(&q_empty[qs]);
          warp_umma_commit(&l_empty[tile & 1]);
          __syncwarp();
        }
        s += g.n;
        ++seg;
        if (s >= s1) break;
        g.next(p, first, s1 - s);
      }
    } else if (warp < 4) {                   // one for each slot: a load takes as long as a tile
      constexpr int PER = COLS / 32;
      const float never = copysignf(INFINITY, p.lse_in);         // in the place of less the log-sum-exp: a weight of 0, with a scale of either sign
      int at[PER], head[PER];                // of the lane's columns: token of the tile (-1: none), query head of the kv head
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int c = lane + k * 32;
        at[k] = c < used ? c / p.G : -1;
        head[k] = c % p.G;
      }
      int tile = 0;
      for (int s = s0;;) {
        for (int j = g.j; j < g.j + g.n; ++j, ++tile) {
          const int slot = tile & 1, tok = g.q_end - (g.count - j) * p.TQ;
          if (slot != (warp & 1)) continue;
          float x[PER];
#pragma unroll
          for (int k = 0; k < PER; ++k)
            x[k] = at[k] >= 0 && tok + at[k] >= g.q_lo ? p.lse[(int64_t)(tok + at[k]) * p.Hq + g.h * p.G + head[k]] : -INFINITY;
          mbar_wait_lim(&l_empty[slot], ((tile >> 1) & 1) ^ 1, budget);
          __syncwarp();
          bool none = false;
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            const bool row = fabsf(x[k]) < INFINITY;             // else none, or one without keys: 0
            const float y = row ? x[k] * p.lse_in : never;
            const bool fits = !CAP && fabsf(y) <= MOST<T>;
            lse_smem[slot * COLS + lane + k * 32] = !row ? -INFINITY : fits ? 0.f : x[k] * -LOG2E;
            none |= at[k] >= 0 && !(row && (CAP || fits));
            if (!CAP && k < pieces) {
              const int c = lane + k * 32;
              const T hi = from_f32<T>(row && !fits ? 0.f : y);
              const float rest = fits ? y - to_f32(hi) : 0.f;
              const T mid = from_f32<T>(rest);
              *reinterpret_cast<uint2*>(aug_smem + slot * (COLS * 32) + c * 32 + (((c >> 2) & 1) << 4)) =
                  make_uint2(pack2<T>(to_f32(hi), to_f32(mid)), pack2<T>(rest - to_f32(mid), 0.f));
            }
          }
          if (!CAP) fence_proxy_async();
          none = __any_sync(0xffffffffu, none);
          __syncwarp();                      // (a vote orders no memory: all lanes' values are there before lane 0 says so)
          if (lane == 0) {
            odd[slot] = none;
            mbar_arrive(&l_full[slot]);
          }
        }
        s += g.n;
        if (s >= s1) break;
        g.next(p, first, s1 - s);
      }
    } else {
      // A warp has 32 keys of one key tile and every second piece of 32 columns, half of which is on its way out of tensor memory while the other half is
      // summed.  The eight warps of a key tile go through its products by themselves, so one tile's are issued while the other's are summed.
      const int qd = warp & 3, half = ((warp - 4) >> 2) & 1, t = (warp - 4) >> 3, mine = t * TILE + qd * 32 + lane;
      const int groups = (pieces - half + 1) / 2;                // 2 to 4
      const uint32_t from = tmem + t * COLS + half * 32 + ((uint32_t)(qd * 32) << 16);
      auto weight = [&](uint32_t s, float l, bool poly, bool add, bool near) {
        const float x = __uint_as_float(s);
        const float y = CAP ? (near ? prompt::cap_small(x * p.ku, p.c2) : cap_near_or_far(x * p.ku, p.c2)) + l : add ? fmaf(x, p.scale_log2, l) : x * p.scale_log2;
        return poly ? ex2_poly(y) : ex2(y);
      };
      int tile = 0;
      for (int s = s0;;) {
        const int key0 = g.i * KEYS + t * TILE, key = g.i * KEYS + mine, n = min(g.len, p.max_rows);
        float* score = p.scores + g.b * p.sc_req + g.h * p.sc_head + key;
        const bool whole = g.n == g.count, writes = half == 0 && key < n;
        const float old = writes && whole ? *score : 0.f;
        float sum = 0.f, rest = 0.f;                             // of all tiles: the sum, and what its additions have cut off
        for (int j = g.j; j < g.j + g.n; ++j, ++tile) {
          const int slot = tile & 1, pos = g.len - (g.count - j) * p.TQ;               // position of the tile's first token
          const float* ls = lse_smem + slot * COLS + half * 32;
          mbar_wait_lim(&l_full[slot], (tile >> 1) & 1, budget);
          mbar_wait_lim(&s_full[t], tile & 1, budget);
          __syncwarp();
          tc_fence_after();
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          const bool full = pos >= key0 + TILE - 1 && !odd[slot];                      // every row sees every key
          const int c_lo = min(max(key - pos, 0), COLS) * p.G - half * 32;             // columns that see the key begin here
          auto release = [&]() {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_empty[t]);
          };
          if (key0 < n && full) {
            auto weigh_as = [&](const uint32_t (&v)[16], const float* lc, bool near) {
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const float4 l = CAP ? *reinterpret_cast<const float4*>(lc + i) : make_float4(0.f, 0.f, 0.f, 0.f);
                acc[0] += weight(v[i], l.x, false, false, near);
                acc[1] += weight(v[i + 1], l.y, false, false, near);
                acc[2] += weight(v[i + 2], l.z, i % 8 == 4, false, near);
                acc[3] += weight(v[i + 3], l.w, false, false, near);
              }
            };
            auto weigh = [&](const uint32_t (&v)[16], const float* lc) {
              if constexpr (CAP) {                               // (the whole warp takes one way)
                float far = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) far = fmaxf(far, fabsf(__uint_as_float(v[i])));
                if (__all_sync(0xffffffffu, far * fabsf(p.ku) <= 1.f)) weigh_as(v, lc, true);
                else weigh_as(v, lc, false);
              } else {
                weigh_as(v, lc, false);
              }
            };
            uint32_t va[16], vb[16];
            tmem_ld_32x16(from, va);
#pragma unroll 1
            for (int c = 0; c < groups; ++c) {
              wait_for(va);
              tmem_ld_32x16(from + c * 64 + 16, vb);
              weigh(va, ls + c * 64);
              wait_for(vb);
              if (c + 1 < groups) tmem_ld_32x16(from + c * 64 + 64, va);
              else release();
              weigh(vb, ls + c * 64 + 16);
            }
          } else if (key0 < n) {
#pragma unroll 1
            for (int c = 0; c < groups; ++c) {
              uint32_t v[32];
              tmem_ld_32x32(from + c * 64, v);
              wait_for(v);
              if (c == groups - 1) release();
              const float* lc = ls + c * 64;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float l = lc[i], x = weight(v[i], l, false, true, false);
                acc[i & 3] += c * 64 + i < c_lo || l == -INFINITY ? 0.f : x;
              }
            }
          } else if (lane == 0) {
            mbar_arrive(&s_empty[t]);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&l_empty[slot]);
          const float x = ((acc[0] + acc[1]) + (acc[2] + acc[3])) - rest, y = sum + x;
          rest = (y - sum) - x;
          sum = y;
        }
        // the two halves of the columns
        if (half == 1) exch[mine] = sum;
        asm volatile("bar.sync %0, 256;" ::"r"(1 + t) : "memory");
        if (half == 0) {
          const float x = sum + exch[mine];
          if (!whole) p.part[((int64_t)blockIdx.x * 2 + (g.j == 0 ? 1 : 0)) * KEYS + mine] = x;
          else if (writes) *score = old + x;
        }
        asm volatile("bar.sync %0, 256;" ::"r"(1 + t) : "memory");                    // exch is free again
        s += g.n;
        if (s >= s1) break;
        g.next(p, first, s1 - s);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
  if (budget < 0 && p.error) *p.error = 1;
}

// Blocks that several CTAs have summed: one CTA for each border between runs, at work where the border is the first within a block.
__global__ void __launch_bounds__(KEYS) join_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x + 1;
  const int4 at = p.info[c];
  if (at.z < 0) return;
  const int key = at.z * KEYS + threadIdx.x, n = min(max(p.seq_lens[at.x], 0), p.max_rows);
  float* score = p.scores + at.x * p.sc_req + at.y * p.sc_head + key;
  const float old = key < n ? *score : 0.f;
  float sum = p.part[((int64_t)(c - 1) * 2 + 1) * KEYS + threadIdx.x];
#pragma unroll 4
  for (int i = c; i < c + at.w; ++i) sum += p.part[(int64_t)i * 2 * KEYS + threadIdx.x];
  if (key < n) *score = old + sum;
}

template <typename T, int KB, bool CAP>
static int launch(const CUtensorMap& tq, const CUtensorMap& tk, const Params& p, int ctas, cudaStream_t st) {
  auto k = weights_kernel<T, KB, CAP>;
  static std::atomic<uint64_t> devices{0};
  if (vb_allow_smem(reinterpret_cast<const void*>(k), Form<KB>::SMEM, devices) != cudaSuccess) return (int)cudaGetLastError();
  vb_launch(k, dim3(ctas), dim3(NUM_THREADS), (size_t)Form<KB>::SMEM, st, tq, tk, p);
  if (p.part && ctas > 1) vb_launch(join_kernel, dim3(ctas - 1), dim3(KEYS), 0, st, p);
  return (int)cudaGetLastError();
}
template <typename T, bool CAP>
static int pick(const CUtensorMap& tq, const CUtensorMap& tk, const Params& p, int ctas, cudaStream_t st) {
  switch ((p.D + 63) / 64) {
    case 1: return launch<T, 1, CAP>(tq, tk, p, ctas, st);
    case 2: return launch<T, 2, CAP>(tq, tk, p, ctas, st);
    case 3: return launch<T, 3, CAP>(tq, tk, p, ctas, st);
    default: return launch<T, 4, CAP>(tq, tk, p, ctas, st);
  }
}

}  // namespace kweights

// `error` (device or pinned int, may be null) becomes 1 when a wait inside the kernel ran into its limit.  max_rows: rows of a request that the
// block table and the scores have room for; max_query: of its query rows that count.  part: ctas x 516 floats, or null: no block is split between CTAs (a
// key's sum then does not depend on other requests).
EXPORT int vb_key_weights(const void* q, const void* cache, int64_t num_blocks, const int* block_table, const int* seq_lens, const int* qsl, const float* lse,
                          float* scores, float* part, int* error, int B, int T, int Hq, int Hkv, int D, int BS, int max_rows, int max_query, int last, int ctas,
                          int64_t q_stride, int64_t bt_stride, int64_t sc_req, int64_t sc_head, float scale, float soft_cap, int dtype,
                          cudaStream_t st) {
  using namespace kweights;
  if (B <= 0 || T <= 0 || max_rows <= 0) return 0;
  if (dtype == DT_F32 || D % 8 || D > 256 || BS % 16 || Hq % Hkv || Hq / Hkv > 128 || ctas < 1) return -1;
  auto enc = get_encode();
  if (!enc) return -10;
  const bool bf16 = dtype == DT_BF16;
  const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  Params p;
  p.block_table = block_table; p.seq_lens = seq_lens; p.qsl = qsl; p.lse = lse; p.scores = scores; p.part = part; p.error = error; p.info = reinterpret_cast<int4*>(part + (int64_t)ctas * 2 * KEYS);
  p.bt_stride = bt_stride; p.sc_req = sc_req; p.sc_head = sc_head; p.num_blocks = num_blocks;
  p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.D = D; p.BS = BS; p.max_rows = max_rows; p.last = last; p.whole = part == nullptr;
  p.box_rows = BS & -BS;                                         // a page is whole boxes
  if (p.box_rows > TILE) p.box_rows = TILE;
  const int columns = D <= 192 ? COLS : COLS / 2;
  p.TQ = columns;
  while (p.TQ * p.G > columns) p.TQ /= 2;
  p.scale_log2 = scale * LOG2E;
  p.one = 1.f;
  if (!bf16) {                                                   // (a power of two that fp16 has)
    const int e = ilogbf(scale);
    p.one = ldexpf(1.f, e > 16 ? -14 : e < -13 ? 15 : 2 - e);
  }
  p.lse_in = -1.f / (scale * p.one);
  p.ku = soft_cap > 0.f ? scale / soft_cap : 0.f; p.c2 = soft_cap * LOG2E;
  CUtensorMap tq, tk;
  cuuint32_t es[3] = {1, 1, 1};
  {
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)Hq, (cuuint64_t)T};
    cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)p.G, (cuuint32_t)p.TQ};
    if (enc(&tq, dt, 3, const_cast<void*>(q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return -11;
  }
  {
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)BS, (cuuint64_t)num_blocks * 2 * Hkv};
    cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)D * BS * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)p.box_rows, 1};
    if (enc(&tk, dt, 3, const_cast<void*>(cache), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return -12;
  }
  const int64_t tiles = (int64_t)Hkv * ((max_rows + KEYS - 1) / KEYS) * ((max_query + p.TQ - 1) / p.TQ);      // of a request, at most
  int step = MAX_REQUESTS;
  while (step > 1 && tiles * step > (1 << 30)) step /= 2;        // tile numbers are 32 bits
  if (tiles > (1 << 30)) return -3;
  for (int b0 = 0; b0 < B; b0 += step) {
    p.B = B - b0 < step ? B - b0 : step;
    p.block_table = block_table + b0 * bt_stride;
    p.seq_lens = seq_lens + b0;
    p.scores = scores + b0 * sc_req;
    p.qsl = qsl ? qsl + b0 : nullptr;
    p.row0 = b0;
    const int n = p.B * tiles < ctas ? (int)(p.B * tiles) : ctas;
    const int rc = bf16 ? (soft_cap > 0.f ? pick<__nv_bfloat16, true>(tq, tk, p, n, st) : pick<__nv_bfloat16, false>(tq, tk, p, n, st))
                        : (soft_cap > 0.f ? pick<__half, true>(tq, tk, p, n, st) : pick<__half, false>(tq, tk, p, n, st));
    if (rc) return rc;
  }
  return 0;
}
