// The weights that a prompt's query rows give to the cached keys, added to the keys' scores:
//
//   scores[b, h, k] += sum over the request's (last) query rows t >= k and the G query heads g of kv head h of e^(c(scale q[t, g] . K[k]) - lse[t, g])
//
// lse is that of the attention before, so a weight needs no second look at its row.  Keys are the rows of tcgen05 products, 128 x 128: a thread owns
// a key (a lane of tensor memory), its columns are (token, head) pairs, and the sum stays in its registers until the key's last query: one write per key, no
// exchange between threads, no atomics, the same order in every run.  A CTA takes 256 keys (two products share a tile of queries, half the reads of
// it) of one kv head and the queries that see them.
#include "attention_prompt.cuh"

namespace kweights {

constexpr int KEYS = 256, TILE = 128, COLS = 128;
constexpr int NUM_THREADS = 352;            // warp 0: copies, 1: products, 2..9: sums, 10: log-sum-exps
constexpr int BLK = TILE * 128;             // [128 rows x 64 values], 16 KB
constexpr float LOG2E = 1.4426950408889634f;

struct Params {
  const int* block_table;
  const int* seq_lens;
  const int* qsl;            // null: one row per request
  const float* lse;          // [T, Hq]
  float* scores;
  int* error;                // raised when a wait ran into its limit
  int64_t bt_stride, sc_req, sc_head, num_blocks;
  int T, Hq, Hkv, G, D, BS, max_rows, last, box_rows;
  float scale_log2, ku, c2;
};

template <int KB> struct Form {              // KB: blocks of 64 dimensions
  static constexpr int STAGES = KB <= 2 ? 3 : KB == 3 ? 2 : 1;
  static constexpr int K_BYTES = 2 * KB * BLK, Q_BYTES = KB * BLK;
  static constexpr int NEED = K_BYTES + STAGES * Q_BYTES + 2 * COLS * 4 + 32 * 8 + 16 + 1024;
  static constexpr int SMEM = NEED > 116 * 1024 ? NEED : 116 * 1024;         // one CTA per SM: it has all of tensor memory
};

template <typename T, int KB, bool CAP>
__global__ void __launch_bounds__(NUM_THREADS, 1)
weights_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const Params p) {
  using F = Form<KB>;
  constexpr int STAGES = F::STAGES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* k_smem = smem;                                  // [key tile][KB]
  unsigned char* q_smem = k_smem + F::K_BYTES;                   // [stage][KB]
  float* lse_smem = reinterpret_cast<float*>(q_smem + STAGES * F::Q_BYTES);      // [2][COLS], in powers of two
  uint64_t* k_full = reinterpret_cast<uint64_t*>(lse_smem + 2 * COLS);
  uint64_t* q_full = k_full + 1;
  uint64_t* q_empty = q_full + STAGES;
  uint64_t* s_full = q_empty + STAGES;       // [buffer]
  uint64_t* s_empty = s_full + 2;
  uint64_t* l_full = s_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(l_full + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int budget = MBAR_BUDGET;
  pdl_trigger();
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.z, k0 = blockIdx.y * KEYS;
  const int len = max(p.seq_lens[b], 0), n = min(len, p.max_rows);
  const int q_begin = p.qsl ? p.qsl[b] : b, q_end = min(p.qsl ? p.qsl[b + 1] : b + 1, p.T);
  const int TQ = COLS / p.G;                                     // tokens of a tile
  int t_first = max(q_begin, q_end - len + k0);                  // the first token that sees a key of the CTA
  if (p.last > 0) t_first = max(t_first, q_end - p.last);
  const int tiles = (q_end - t_first + TQ - 1) / TQ;
  if (k0 >= n || q_end <= t_first) return;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_q); tma_prefetch_desc(&tmap_k);
    mbar_init(k_full, 1);
    for (int s = 0; s < STAGES; ++s) { mbar_init(&q_full[s], 1); mbar_init(&q_empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&s_full[s], 1); mbar_init(&s_empty[s], 8); mbar_init(&l_full[s], 1); }
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  if (TQ * p.G < COLS)                                           // columns that no head has: zeros
    for (int i = threadIdx.x; i < STAGES * F::Q_BYTES / 16; i += NUM_THREADS) reinterpret_cast<uint4*>(q_smem)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;                              // scores of buffer u, key tile t: columns u * 256 + t * 128

  if (warp == 0) {
    if (lane == 0) {
      const int* bt = p.block_table + b * p.bt_stride;
      int boxes = 0;
      for (int r = 0; r < KEYS && k0 + r < n; r += p.box_rows) ++boxes;
      mbar_expect_tx(k_full, boxes * KB * p.box_rows * 128);
      for (int i = 0; i < boxes; ++i) {
        const int r = i * p.box_rows, key = k0 + r;
        int64_t blk = bt[key / p.BS];
        if ((uint64_t)blk >= (uint64_t)p.num_blocks) blk = 0;    // (a table may not say that)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          prompt::tma_load_3d(k_smem + ((r >> 7) * KB + kb) * BLK + (r & 127) * 128, &tmap_k, kb * 64, key % p.BS, (int)(blk * 2 * p.Hkv + h), k_full);
      }
      for (int j = 0; j < tiles; ++j) {
        const int s = j % STAGES;
        mbar_wait_lim(&q_empty[s], ((j / STAGES) & 1) ^ 1, budget);
        if (budget < 0) break;
        mbar_expect_tx(&q_full[s], KB * TQ * p.G * 128);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          prompt::tma_load_3d(q_smem + s * F::Q_BYTES + kb * BLK, &tmap_q, kb * 64, h * p.G, t_first + j * TQ, &q_full[s]);
      }
      if (budget < 0) { mbar_let_land(k_full, 1); mbar_let_land(q_full, STAGES); }
    }
  } else if (warp == 1) {
    const uint32_t idesc = umma_idesc_f16(TILE, COLS, DTypeOf<T>::v == DT_BF16);
    const int steps = (p.D + 15) / 16;
    const bool second = k0 + TILE < n;
    mbar_wait_lim(k_full, 0, budget);
    for (int j = 0; j < tiles; ++j) {
      const int s = j % STAGES, u = j & 1;
      mbar_wait_lim(&q_full[s], (j / STAGES) & 1, budget);
      mbar_wait_lim(&s_empty[u], ((j >> 1) & 1) ^ 1, budget);
      tc_fence_after();
      __syncwarp();
      for (int t = 0; t < (second ? 2 : 1); ++t)
        for (int k = 0; k < steps; ++k) {
          const uint64_t da = umma_desc_sw128(k_smem + (t * KB + (k >> 2)) * BLK) + (uint64_t)((k & 3) * 2);
          const uint64_t db = umma_desc_sw128(q_smem + s * F::Q_BYTES + (k >> 2) * BLK) + (uint64_t)((k & 3) * 2);
          warp_umma_f16(tmem + u * 256 + t * TILE, da, db, idesc, k != 0);
        }
      warp_umma_commit(&s_full[u]);
      warp_umma_commit(&q_empty[s]);
      __syncwarp();
    }
  } else if (warp < 10) {
    const int t = (warp - 2) >> 2, qd = warp & 3;
    const int key = k0 + t * TILE + qd * 32 + lane;
    const uint32_t at = tmem + t * TILE + ((uint32_t)(qd * 32) << 16);
    const int key_max = k0 + t * TILE + TILE - 1;
    float sum = 0.f, rest = 0.f;             // of all tiles: the sum and what its additions have cut off
    for (int j = 0; j < tiles; ++j) {
      const int u = j & 1;
      const int tok = t_first + j * TQ, pos = len - (q_end - tok);                 // of the tile's first token
      const int cols = min(TQ, q_end - tok) * p.G;
      mbar_wait_lim(&l_full[u], (j >> 1) & 1, budget);
      mbar_wait_lim(&s_full[u], (j >> 1) & 1, budget);
      __syncwarp();
      tc_fence_after();
      const bool full = pos >= key_max && cols == TQ * p.G;
      const int c_lo = min(max(key - pos, 0), COLS) * p.G;                       // columns that see the key: [c_lo, cols)
      const float4* l4 = reinterpret_cast<const float4*>(lse_smem + u * COLS);
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      if (k0 + t * TILE < n) {
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32(at + u * 256 + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 l = l4[(c + i) / 4];
            const float ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = __uint_as_float(v[i + e]);
              const float w = CAP ? ex2(prompt::cap_any(x * p.ku, p.c2) - ls[e]) : ex2(fmaf(x, p.scale_log2, -ls[e]));
              acc[e] += full || (c + i + e >= c_lo && c + i + e < cols) ? w : 0.f;
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[u]);
      const float x = ((acc[0] + acc[1]) + (acc[2] + acc[3])) - rest, y = sum + x;
      rest = (y - sum) - x;
      sum = y;
    }
    if (key < n) p.scores[b * p.sc_req + h * p.sc_head + key] += sum;
  } else {
    for (int j = 0; j < tiles; ++j) {
      const int u = j & 1, tok = t_first + j * TQ;
      mbar_wait_lim(&s_empty[u], ((j >> 1) & 1) ^ 1, budget);
      __syncwarp();
#pragma unroll
      for (int c = lane; c < COLS; c += 32) {
        const int i = tok + c / p.G;
        const float x = c < TQ * p.G && i < q_end ? p.lse[(int64_t)i * p.Hq + h * p.G + c % p.G] : -INFINITY;
        lse_smem[u * COLS + c] = x > -INFINITY ? x * LOG2E : INFINITY;             // no row, or one without keys: weights of 0
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_full[u]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
  if (budget < 0 && p.error) *p.error = 1;
}

template <typename T, int KB, bool CAP>
static int launch(const CUtensorMap& tq, const CUtensorMap& tk, const Params& p, int B, cudaStream_t st) {
  auto k = weights_kernel<T, KB, CAP>;
  static bool set = false;
  if (!set) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Form<KB>::SMEM) != cudaSuccess) return (int)cudaGetLastError();
    set = true;
  }
  vb_launch(k, dim3(p.Hkv, (p.max_rows + KEYS - 1) / KEYS, B), dim3(NUM_THREADS), (size_t)Form<KB>::SMEM, st, tq, tk, p);
  return (int)cudaGetLastError();
}
template <typename T, bool CAP>
static int pick(const CUtensorMap& tq, const CUtensorMap& tk, const Params& p, int B, cudaStream_t st) {
  switch ((p.D + 63) / 64) {
    case 1: return launch<T, 1, CAP>(tq, tk, p, B, st);
    case 2: return launch<T, 2, CAP>(tq, tk, p, B, st);
    case 3: return launch<T, 3, CAP>(tq, tk, p, B, st);
    default: return launch<T, 4, CAP>(tq, tk, p, B, st);
  }
}

}  // namespace kweights

// `error` (device or pinned int, may be null) becomes 1 when a wait inside the kernel ran into its limit.  max_rows: rows of a request that the
// block table and the scores have room for.
EXPORT int vb_key_weights(const void* q, const void* cache, int64_t num_blocks, const int* block_table, const int* seq_lens, const int* qsl, const float* lse,
                          float* scores, int* error, int B, int T, int Hq, int Hkv, int D, int BS, int max_rows, int last, int64_t q_stride, int64_t bt_stride,
                          int64_t sc_req, int64_t sc_head, float scale, float soft_cap, int dtype, cudaStream_t st) {
  using namespace kweights;
  if (B <= 0 || T <= 0 || max_rows <= 0) return 0;
  if (dtype == DT_F32 || D % 8 || D > 256 || BS % 16 || Hq % Hkv || Hq / Hkv > COLS) return -1;
  auto enc = get_encode();
  if (!enc) return -10;
  const bool bf16 = dtype == DT_BF16;
  const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  Params p;
  p.block_table = block_table; p.seq_lens = seq_lens; p.qsl = qsl; p.lse = lse; p.scores = scores; p.error = error;
  p.bt_stride = bt_stride; p.sc_req = sc_req; p.sc_head = sc_head; p.num_blocks = num_blocks;
  p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.D = D; p.BS = BS; p.max_rows = max_rows; p.last = last;
  p.box_rows = BS & -BS;                                         // a page is whole boxes
  if (p.box_rows > TILE) p.box_rows = TILE;
  p.scale_log2 = scale * LOG2E;
  p.ku = soft_cap > 0.f ? scale / soft_cap : 0.f; p.c2 = soft_cap * LOG2E;
  CUtensorMap tq, tk;
  cuuint32_t es[3] = {1, 1, 1};
  {
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)Hq, (cuuint64_t)T};
    cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)p.G, (cuuint32_t)(COLS / p.G)};
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
  if (bf16) return soft_cap > 0.f ? pick<__nv_bfloat16, true>(tq, tk, p, B, st) : pick<__nv_bfloat16, false>(tq, tk, p, B, st);
  return soft_cap > 0.f ? pick<__half, true>(tq, tk, p, B, st) : pick<__half, false>(tq, tk, p, B, st);
}
