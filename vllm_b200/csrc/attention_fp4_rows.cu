// Attention of prompts, or portions of them, over a paged key-value cache in 4 bits (fp4.cuh), for the head shapes that the tcgen05 kernel over 16-bit pages does not take.
//
//   s[r, k] = c(scale q_r . K_k) for the keys k that row r sees,  lse_r = log(sum_k e^s[r, k] + e^sink),  out_r = sum_k e^(s[r, k] - lse_r) V_k
//
// A CTA has 128 query rows of a request and a kv head (pairs of a new token and a query head, so all heads of the kv head share its keys) and goes through the keys in tiles
// of 64.  Codes and scales of the next tile are on their way into registers while this one is worked on; then every thread turns its groups of 16 into fp16 (exact)
// in shared memory, where two tiles take turns: one barrier a tile.  S = Q K^T and O += P V are m16n8k16 products; a warp has 32 rows (heads of up to 96: a
// fragment of keys or values then serves two products) or 16, and takes 64 or 32 keys at a time: weights go from the accumulators of the first
// product into the operands of the second.  The reference of a row's weights stays until a weight would be above 2^15 (attention_fp4.cu).
//
// Q is fp16, bf16 rows scaled by a power of two (exact, attention_fp4.cu).  Weights are fp16 (off by at most 2^-11 of themselves: as the result where that is fp16,
// an eighth of its rounding where it is bf16); sums are in 32 bits.
//
// Where there are fewer CTAs than the SMs hold, the keys are split and a second kernel joins the parts.
//
// It is bound by how few warps the registers leave, 8 on an SM: the matrix pipe, whose legacy instructions would give 560 TFLOP/s, is busy in 46 % of the cycles for heads of 64 and 35 %
// for 256, and instructions issue in 35 and 21 %.  A warp that has issued waits for the latency of its own instruction (64: 2.3 of 5.3 cycles an instruction) or for shared memory (256:
// 3.2 of 9.3).  220 to 240 TFLOP/s for heads of 64 to 192, 173 for 256.  us for two
// prompts of 2000 behind 1500, 20 / 4 heads of 64, 80, 96, 128, 192, 256: 206, 282, 310, 394, 575, 1063 (64 keys at a time; 32: 224, 282, 310, 416, 575, 1063, and 64 for 96 357); heads of
// up to 128 read back to 16-bit pages of 128 take 204 to 209 there on the tcgen05 kernel and are better off here only in short portions (fp4_kernels in ops/cuda.py).  256 rows of a CTA
// share the keys' conversion but wait for one another: 251 where 128 took 226 (500 new tokens behind 11 500, 16 / 4 heads of 64, now 204).
#include "attention_prompt.cuh"
#include "device_once.h"
#include "fp4.cuh"

namespace rfp4 {

constexpr int TILE = 64, ROWS = 128;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f, SHIFT = 7.f, NONE = -3e38f;

struct Params {
  const void* q;
  const uint8_t* cache;
  const int* block_table;
  const int* seq_lens;
  const int* qsl;
  void* out;
  float* lse;
  const float* sinks;
  float* part;               // [split][token, head][D + 2]: output, maximum, sum
  int64_t q_stride, out_stride, bt_stride, num_blocks, tokens;
  int Hkv, G, BS, max_rows, few, splits, window, bf16;
  float scale_log2, ku, c2, out_scale;
};

// The keys that a CTA's rows see, as tiles [lo, hi) of its split
struct Span {
  int n, t, r0, rows, lo, hi;
};
VB_DEVICE Span span_of(const Params& p, int b, int tile, int split) {
  Span s;
  s.n = min(max(p.seq_lens[b], 0), p.max_rows);
  s.t = p.qsl[b + 1] - p.qsl[b];
  s.r0 = tile * ROWS;
  s.rows = s.t > p.few ? min(ROWS, s.t * p.G - s.r0) : 0;
  s.lo = s.hi = 0;
  if (s.rows <= 0) { s.rows = 0; return s; }
  const int first = s.n - s.t + s.r0 / p.G, last = s.n - s.t + (s.r0 + s.rows - 1) / p.G;       // places of the first and the last row
  const int from = p.window > 0 ? max(first - p.window + 1, 0) / TILE : 0, to = last >= 0 ? last / TILE + 1 : 0, per = (max(to - from, 0) + p.splits - 1) / p.splits;
  s.lo = from + split * per;
  s.hi = min(s.lo + per, to);
  return s;
}

VB_DEVICE void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
VB_DEVICE void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
VB_DEVICE void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

VB_DEVICE uint32_t max2(uint32_t a, uint32_t b) { uint32_t r; asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }

VB_DEVICE float log_of(float base, float sum) { return sum > 0.f ? (base + log2f(sum)) * LN2 : sum == 0.f ? -INFINITY : sum; }

template <int D_> struct Form {
  static constexpr int D = D_, MT = D <= 96 ? 2 : 1, WARPS = ROWS / (16 * MT), THREADS = WARPS * 32;
  static constexpr int CTAS = D <= 96 ? 2 : 1;             // of an SM
  static constexpr int SUB = D <= 64 || D == 128 ? 64 : 32;              // keys that a warp takes at a time: as many as the registers hold scores of
  static constexpr int LD = 2 * D + 16;                                  // bytes of a row in shared memory: an odd number of 16, so that neighbouring rows begin in different banks
  static constexpr int SIDE = TILE * LD, BUF = 2 * SIDE, SMEM = 2 * BUF;
  static constexpr int GROUPS = TILE * D / 16, MINE = (GROUPS + THREADS - 1) / THREADS;      // of a side; of a thread
};

template <int D, bool BF16>
__global__ void __launch_bounds__(Form<D>::THREADS, Form<D>::CTAS) rows_kernel(const Params p) {
  using F = Form<D>;
  constexpr int MT = F::MT, KD = D / 16, SUB = F::SUB, NT = SUB / 8, MINE = F::MINE;
  extern __shared__ __align__(128) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();
  const int split = blockIdx.x % p.splits, tile = gridDim.x / p.splits - 1 - blockIdx.x / p.splits;       // (those that see the most keys first)
  const int h = blockIdx.y, b = blockIdx.z;
  const Span sp = span_of(p, b, tile, split);
  if (sp.rows == 0) return;
  const int first_q = p.qsl[b], g = lane >> 2, t4 = lane & 3;
  const int n = sp.n, low = p.window > 0 ? max(n - sp.t + sp.r0 / p.G - p.window + 1, 0) : 0;
  const bool capped = p.ku != 0.f;

  // ---- codes and scales of a tile: a thread's groups
  const int64_t page = fp4::page_bytes(p.BS, D), to_v = p.Hkv * page;
  int at_page[MINE], at_off[MINE];                     // of the tile that is looked up next
  int blk[MINE], off[MINE];                            // of the tile that is read next
  const int pages_on = TILE / p.BS, rest = TILE % p.BS;
#pragma unroll
  for (int j = 0; j < MINE; ++j) {
    const int tok = sp.lo * TILE + (j * F::THREADS + threadIdx.x) / KD;
    at_page[j] = tok / p.BS;
    at_off[j] = tok % p.BS;
  }
  uint2 codes[2][MINE];
  uint32_t scales[2][MINE];
  auto look = [&](int tl) {
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int gi = j * F::THREADS + threadIdx.x, tok = tl * TILE + gi / KD;
      blk[j] = (F::GROUPS % F::THREADS == 0 || gi < F::GROUPS) && tl < sp.hi && tok < n ? p.block_table[b * p.bt_stride + at_page[j]] : -1;
      off[j] = at_off[j];
      at_page[j] += pages_on;
      at_off[j] += rest;
      if (at_off[j] >= p.BS) { at_off[j] -= p.BS; ++at_page[j]; }
    }
  };
  auto read = [&](int tl) {
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int gi = j * F::THREADS + threadIdx.x, r = gi / KD, c = gi - r * KD, tok = tl * TILE + r;
      const bool there = (F::GROUPS % F::THREADS == 0 || gi < F::GROUPS) && tl < sp.hi && tok < n;
      const uint64_t at = (uint64_t)blk[j] < (uint64_t)p.num_blocks ? blk[j] : 0;      // (a table may not say that; nothing is read outside the cache)
      const uint8_t* k = p.cache + (uint32_t)(at * 2 * p.Hkv + h) * (uint64_t)(uint32_t)page;      // (pages of heads: below 2^31)
      const uint8_t* x = k + off[j] * (D / 2) + c * 8;
      const uint8_t* s = k + p.BS * (D / 2) + off[j] * (D / 16) + c;
      codes[0][j] = there ? *reinterpret_cast<const uint2*>(x) : make_uint2(0u, 0u);
      codes[1][j] = there ? *reinterpret_cast<const uint2*>(x + to_v) : make_uint2(0u, 0u);
      scales[0][j] = there ? s[0] : 0u;
      scales[1][j] = there && tok >= low ? s[to_v] : 0u;            // values that no row sees may be what a weight of 0 does not cancel
    }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int gi = j * F::THREADS + threadIdx.x, r = gi / KD, c = gi - r * KD;
      if (F::GROUPS % F::THREADS == 0 || gi < F::GROUPS) {
        const uint32_t two = fp4::scales2(scales[0][j] | scales[1][j] << 8);
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const uint32_t f = side ? fp4::high2(two) : fp4::low2(two);
          uint32_t x[4], y[4];
          fp4::unpack8(codes[side][j].x, x);
          fp4::unpack8(codes[side][j].y, y);
          uint4* to = reinterpret_cast<uint4*>(smem + buf * F::BUF + side * F::SIDE + r * F::LD + c * 32);
          to[0] = make_uint4(fp4::mul2(x[0], f), fp4::mul2(x[1], f), fp4::mul2(x[2], f), fp4::mul2(x[3], f));
          to[1] = make_uint4(fp4::mul2(y[0], f), fp4::mul2(y[1], f), fp4::mul2(y[2], f), fp4::mul2(y[3], f));
        }
      }
    }
  };
  look(sp.lo);

  // ---- queries: rows g and g + 8 of the warp's blocks of 16
  uint32_t q[MT][KD][4];
  float by[MT][2];                                     // of a row's sums: to powers of two, or to the cap
  int last[MT][2];                                     // last key that a row sees
  const int wr = warp * 16 * MT;                       // the warp's first row of the CTA's
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = wr + m * 16 + u * 8 + g, r = sp.r0 + i, tok = r / p.G;
      const bool there = i < sp.rows;
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(p.q) + (int64_t)(first_q + tok) * p.q_stride + (int64_t)(h * p.G + r - tok * p.G) * D + t4 * 2;
      last[m][u] = n - sp.t + tok;
#pragma unroll
      for (int k = 0; k < KD; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) q[m][k][u + 2 * j] = there ? *reinterpret_cast<const uint32_t*>(qp + k * 16 + j * 8) : 0u;
    }
  read(sp.lo);
  look(sp.lo + 1);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float mine = 1.f;
      if (BF16) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < KD; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 x = unpack2<__nv_bfloat16>(q[m][k][u + 2 * j]);
            top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max((int)(__float_as_uint(top) >> 23), 27), 254);                  // of the exponent's field
        const float f = __uint_as_float((uint32_t)(127 + 14 - e + 127) << 23);               // 2^(14 - (e - 127))
        mine = __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
        for (int k = 0; k < KD; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 x = unpack2<__nv_bfloat16>(q[m][k][u + 2 * j]);
            q[m][k][u + 2 * j] = pack2<__half>(x.x * f, x.y * f);
          }
      }
      by[m][u] = mine * (capped ? p.ku : p.scale_log2);
    }
  const int warp_first = n - sp.t + (sp.r0 + wr) / p.G, warp_last = wr < sp.rows ? n - sp.t + (sp.r0 + min(wr + 16 * MT, sp.rows) - 1) / p.G : -1;

  float o[MT][D / 8][4], m_run[MT][2], l_run[MT][2];
  bool huge = false;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[m][i][j] = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) { m_run[m][u] = NONE; l_run[m][u] = 0.f; }
  }
  if (sp.lo < sp.hi) store(0);
  const uint32_t base = smem_u32(smem);
  const int mi = lane >> 3, l7 = lane & 7;
  for (int tl = sp.lo; tl < sp.hi; ++tl) {
    const int buf = (tl - sp.lo) & 1;
    __syncthreads();                                   // the tile is there, and nobody reads the other one
    read(tl + 1);
    look(tl + 2);
#pragma unroll
    for (int k0 = 0; k0 < TILE; k0 += SUB) {
      const int key0 = tl * TILE + k0;
      if (key0 > warp_last || (p.window > 0 && key0 + SUB <= warp_first - p.window + 1)) continue;
      // ---- S = Q K^T
      float s[MT][NT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[m][i][j] = 0.f;
      const uint32_t ks = base + buf * F::BUF + (k0 + (mi >> 1) * 8 + l7) * F::LD + (mi & 1) * 16;
#pragma unroll
      for (int k = 0; k < KD; ++k)
#pragma unroll
        for (int i = 0; i < NT; i += 2) {
          uint32_t x[4];
          ldsm4(x, ks + i * 8 * F::LD + k * 32);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma16816(s[m][i], q[m][k], x[0], x[1]);
            mma16816(s[m][i + 1], q[m][k], x[2], x[3]);
          }
        }
      // ---- weights
      const bool cut = key0 + SUB > warp_first + 1 || (p.window > 0 && key0 <= warp_last - p.window);
      uint32_t w[MT][NT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float f[2] = {by[m][0], by[m][1]};
        if (capped || cut || huge) {
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float x = s[m][i][j] * by[m][j >> 1];
              if (capped) x = prompt::cap_any(x, p.c2);
              const int key = key0 + i * 8 + t4 * 2 + (j & 1), to = last[m][j >> 1];
              s[m][i][j] = key > to || (p.window > 0 && key <= to - p.window) ? -INFINITY : x;
            }
          f[0] = f[1] = 1.f;
        }
        uint32_t most = 0u;                              // the largest weights, two halves
        float add[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float x = ex2(fmaf(s[m][i][2 * u], f[u], -m_run[m][u])), y = ex2(fmaf(s[m][i][2 * u + 1], f[u], -m_run[m][u]));
            add[u] += x + y;
            w[m][i][u] = pack2<__half>(x, y);
            most = max2(most, w[m][i][u]);
          }
        if (__any_sync(0xffffffffu, (most & 0xffffu) > 0x7800u || most > 0x7800ffffu)) {          // above 2^15
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < NT; ++i) mx = fmaxf(mx, fmaxf(s[m][i][2 * u] * f[u], s[m][i][2 * u + 1] * f[u]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float was = m_run[m][u], at = fmaxf(mx - SHIFT, NONE);
            const bool up = at > was + 8.f;
            const float alpha = up ? ex2(was - at) : 1.f;
            m_run[m][u] = up ? at : was;
            l_run[m][u] *= alpha;
            add[u] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) { o[m][i][2 * u] *= alpha; o[m][i][2 * u + 1] *= alpha; }
          }
          huge |= __any_sync(0xffffffffu, (m_run[m][0] > NONE && fabsf(m_run[m][0]) > 0x1p20f) || (m_run[m][1] > NONE && fabsf(m_run[m][1]) > 0x1p20f)) != 0;
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {                // (the difference of two rounded numbers: nothing is left over where scores are huge)
              const float x = ex2(__fsub_rn(__fmul_rn(s[m][i][2 * u], f[u]), m_run[m][u])), y = ex2(__fsub_rn(__fmul_rn(s[m][i][2 * u + 1], f[u]), m_run[m][u]));
              add[u] += x + y;
              w[m][i][u] = pack2<__half>(x, y);
            }
        }
        l_run[m][0] += add[0];
        l_run[m][1] += add[1];
      }
      // ---- O += P V
      const uint32_t vs = base + buf * F::BUF + F::SIDE + (k0 + (mi & 1) * 8 + l7) * F::LD + (mi >> 1) * 16;
#pragma unroll
      for (int kk = 0; kk < SUB / 16; ++kk)
#pragma unroll
        for (int i = 0; i < D / 8; i += 2) {
          uint32_t x[4];
          ldsm4_t(x, vs + kk * 16 * F::LD + i * 16);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint32_t a[4] = {w[m][2 * kk][0], w[m][2 * kk][1], w[m][2 * kk + 1][0], w[m][2 * kk + 1][1]};
            mma16816(o[m][i], a, x[0], x[1]);
            mma16816(o[m][i + 1], a, x[2], x[3]);
          }
        }
    }
    if (tl + 1 < sp.hi) store(buf ^ 1);
  }
  // ---- outputs, or parts of them
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float l = l_run[m][u];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const int i = wr + m * 16 + u * 8 + g, r = sp.r0 + i, tok = r / p.G, head = h * p.G + r - tok * p.G;
      if (i >= sp.rows) continue;
      const bool none = m_run[m][u] == NONE && l == 0.f;       // (with a NaN sum: nothing but NaN was seen, and that comes out)
      const int64_t at = (int64_t)(first_q + tok) * p.Hkv * p.G + head;
      if (p.splits > 1) {
        float* to = p.part + (split * p.tokens * p.Hkv * p.G + at) * (D + 2);
        if (!none)
#pragma unroll
          for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(to + j * 8 + t4 * 2) = make_float2(o[m][j][2 * u], o[m][j][2 * u + 1]);
        if (t4 == 0) *reinterpret_cast<float2*>(to + D) = make_float2(none ? -INFINITY : m_run[m][u], l);
        continue;
      }
      const float sink = p.sinks ? p.sinks[head] * LOG2E : -INFINITY, top = none ? sink : fmaxf(m_run[m][u], sink), base2 = top == -INFINITY ? 0.f : top;
      const float back = none ? 0.f : ex2(m_run[m][u] - base2), all = (none ? 0.f : l * back) + (p.sinks ? ex2(sink - base2) : 0.f), f = all == 0.f ? 0.f : back / all * p.out_scale;
      uint16_t* to = reinterpret_cast<uint16_t*>(p.out) + (int64_t)(first_q + tok) * p.out_stride + (int64_t)head * D + t4 * 2;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        const float x = none ? 0.f : o[m][j][2 * u] * f, y = none ? 0.f : o[m][j][2 * u + 1] * f;
        *reinterpret_cast<uint32_t*>(to + j * 8) = BF16 ? pack2<__nv_bfloat16>(x, y) : pack2<__half>(x, y);
      }
      if (t4 == 0 && p.lse) p.lse[at] = log_of(base2, all);
    }
}

// Grid (runs of JOIN / 32 rows, kv heads, requests): joins the parts of split keys.  A warp has a row.
constexpr int JOIN = 256, PER_TILE = ROWS / (JOIN / 32), MOST_SPLITS = 32;       // (a lane of the join each)
__global__ void __launch_bounds__(JOIN) join_kernel(const Params p, int D) {
  pdl_trigger();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
  const Span sp = span_of(p, b, blockIdx.x / PER_TILE, 0);
  const int first_q = p.qsl[b];
  const int64_t step = p.tokens * p.Hkv * p.G * (D + 2);
  const int i = blockIdx.x % PER_TILE * (JOIN / 32) + (threadIdx.x >> 5);
  if (i < sp.rows) {
    const int r = sp.r0 + i, tok = r / p.G, head = h * p.G + r - tok * p.G;
    const int64_t at = (int64_t)(first_q + tok) * p.Hkv * p.G + head;
    const float* x = p.part + at * (D + 2);
    const float2 ml = lane < p.splits ? *reinterpret_cast<const float2*>(x + lane * step + D) : make_float2(-INFINITY, 0.f);
    const float sink = p.sinks ? p.sinks[head] * LOG2E : -INFINITY, top = fmaxf(warp_max(ml.x), sink), base = top == -INFINITY ? 0.f : top;
    const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - base);
    const float sum = warp_sum(ml.x == -INFINITY ? 0.f : ml.y * f) + (p.sinks ? ex2(sink - base) : 0.f), by = sum == 0.f ? 0.f : p.out_scale / sum;
    uint16_t* to = reinterpret_cast<uint16_t*>(p.out) + (int64_t)(first_q + tok) * p.out_stride + (int64_t)head * D;
    for (int d0 = 0; d0 < D; d0 += 64) {
      const int d = d0 + 2 * lane;
      float2 acc = make_float2(0.f, 0.f);
#pragma unroll 4
      for (int c = 0; c < p.splits; ++c) {
        const float g = __shfl_sync(0xffffffffu, f, c);
        if (g != 0.f && d < D) {                         // (a part without keys holds nothing)
          const float2 y = *reinterpret_cast<const float2*>(x + c * step + d);
          acc.x += y.x * g; acc.y += y.y * g;
        }
      }
      if (d < D) *reinterpret_cast<uint32_t*>(to + d) = p.bf16 ? pack2<__nv_bfloat16>(acc.x * by, acc.y * by) : pack2<__half>(acc.x * by, acc.y * by);
    }
    if (lane == 0 && p.lse) p.lse[at] = log_of(base, sum);
  }
}

template <int D, bool BF16>
static int launch(const Params& p, dim3 grid, cudaStream_t st, int* ctas) {
  using F = Form<D>;
  if (ctas) { *ctas = F::CTAS; return 0; }
  auto k = rows_kernel<D, BF16>;
  static std::atomic<uint64_t> devices{0};
  if (vb_allow_smem(reinterpret_cast<const void*>(k), F::SMEM, devices) != cudaSuccess) return (int)cudaGetLastError();
  vb_launch(k, dim3(grid.x * p.splits, grid.y, grid.z), dim3(F::THREADS), (size_t)F::SMEM, st, p);
  if (p.splits > 1) vb_launch(join_kernel, dim3(grid.x * PER_TILE, grid.y, grid.z), dim3(JOIN), (size_t)0, st, p, D);
  return (int)cudaGetLastError();
}
static int go(const Params& p, int D, dim3 grid, cudaStream_t st, int* ctas = nullptr) {
#define VB_CASE(DD) case DD: return p.bf16 ? launch<DD, true>(p, grid, st, ctas) : launch<DD, false>(p, grid, st, ctas)
  switch (D) {
    VB_CASE(32); VB_CASE(64); VB_CASE(80); VB_CASE(96); VB_CASE(128); VB_CASE(192); VB_CASE(256);
  }
#undef VB_CASE
  return -2;
}

}  // namespace rfp4

// CTAs of an SM, for heads of D
EXPORT int vb_rows_fp4_ctas(int D, int* ctas) {
  rfp4::Params p{};
  return rfp4::go(p, D, dim3(1), nullptr, ctas);
}

// Causal attention of requests of more than `few` new tokens, at most max_q; rows of q and out [tokens] of the others are not touched.  ws: for splits > 1, splits tokens Hq (D + 2)
// floats.  lse [tokens, Hq] or null.
EXPORT int vb_rows_fp4(const void* q, const void* cache, int64_t num_blocks, const int* block_table, const int* seq_lens, const int* qsl, void* out, float* lse,
                       const float* sinks, float* ws, int B, int64_t tokens, int max_q, int Hq, int Hkv, int D, int BS, int max_rows, int few, int64_t q_stride, int64_t out_stride,
                       int64_t bt_stride, int splits, int window, float scale, float soft_cap, float out_scale, int dtype, cudaStream_t st) {
  using namespace rfp4;
  if (B <= 0 || max_q <= few) return 0;
  if ((dtype != DT_BF16 && dtype != DT_F16) || BS < 16 || BS % 16 || Hkv < 1 || Hkv > 65535 || Hq % Hkv || B > 65535 || q_stride % 8 || out_stride % 8 || !qsl || max_rows < 0 ||
      splits < 1 || splits > MOST_SPLITS || (splits > 1 && !ws))
    return -1;
  Params p;
  p.q = q; p.cache = (const uint8_t*)cache; p.block_table = block_table; p.seq_lens = seq_lens; p.qsl = qsl; p.out = out; p.lse = lse; p.sinks = sinks; p.part = ws;
  p.q_stride = q_stride; p.out_stride = out_stride; p.bt_stride = bt_stride; p.num_blocks = num_blocks; p.tokens = tokens;
  p.Hkv = Hkv; p.G = Hq / Hkv; p.BS = BS; p.max_rows = max_rows; p.few = few; p.splits = splits; p.window = window; p.bf16 = dtype == DT_BF16;
  p.scale_log2 = scale * LOG2E;
  p.ku = soft_cap > 0.f ? scale / soft_cap : 0.f; p.c2 = soft_cap * LOG2E; p.out_scale = out_scale;
  if ((int64_t)max_q * p.G > (1 << 30)) return -3;
  return go(p, D, dim3((max_q * p.G + ROWS - 1) / ROWS, Hkv, B), st);
}
