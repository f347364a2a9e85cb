// Attention of few query rows (one new token per request, or some drafts) over a paged key-value cache in 4 bits (fp4.cuh).
//
//   s[r, k] = c(scale q_r . K_k) for the keys k that row r sees,  lse_r = log(sum_k e^s[r, k] + e^sink),  out_r = sum_k e^(s[r, k] - lse_r) V_k
//
// Query rows are pairs (new token, query head of a kv head), 8, 16 or (heads of up to 128) 24 of them at a time: with a request and a kv head they are a
// "row" of the schedule.  All rows' tiles of 64 keys, in order, are dealt to the CTAs in equal runs, so that ragged and few long requests keep all SMs as
// busy as many equal ones; a row that one CTA has is finished there, one that several have is joined by a second kernel.  Where rows are few and short a cluster
// has a row, and the parts meet in shared memory.
//
// A warp takes every fourth strip of 32 keys; codes and scales of a strip come by asynchronous copies of the warp's own, the next strips on their way across the
// borders of rows.  S^T = K Q^T (m16n8k16: keys are rows, query rows columns), an own running maximum, O^T += V^T P^T.
//
// Codes become fp16 in registers (one conversion for two of them, one multiplication by their scale: exact, fp4.cuh), in the order in which the matrix
// instruction wants them: dimensions of K may go to the instruction's k in any order that Q follows, so a lane reads D / 4 neighbouring
// values of a key at once; the products with V pair up keys, so the nibbles of two keys are brought together first (a shift and a bitwise select for eight values),
// and a lane has D / 8 neighbouring dimensions.  Q is fp16, bf16 rows scaled by a power of two to [2^14, 2^15): exact but for values below 2^-28 of the largest,
// whose error is below 2^-39 of it.  Weights are fp16 multiples of 2^-24 of up to 2^15: off by 2^-11 of themselves (a result in bf16 is rounded by up to 2^-8), in two
// such parts where the result is fp16.  Sums are in 32 bits.
//
// What bounds it: 9 / 16 of a byte a value would be 5.9 TB/s of codes at the rate of a 16-bit copy; turning them into operands takes about 160 instructions of the integer pipe for 16
// keys and their values of 128, which is 27 us of two requests of 95000 beside 33.5 of their bytes.  They take 49.4 (74 % of the copy's rate without the 5 of the join): the integer pipe is
// busy in 55 % of the cycles and instructions issue in 60 %, so what is left are the waits of a strip's chain (copy, conversion, product, exponential, product), which 12 warps do not cover.  Three CTAs of 168 registers keep the pipes busier than four of 128 (49.4 to 54.4).  64 requests of 700 to 1301 take 26.4 (bytes 11.4): 13 at that
// rate, 4 for the join, the rest for the chain at a CTA's start (lengths, pages, keys) and for ends of rows; one of 700 5.7; 24 of 60 to 924 with 16 / 8 heads of 64, capped, with
// sinks and a window, 9.4.  A tcgen05 product would want the codes in shared memory as fp16 first: as many conversions, and their stores.
#include "attention_prompt.cuh"
#include "cluster.cuh"
#include "device_once.h"
#include "fp4.cuh"

#include <type_traits>

namespace afp4 {

constexpr int TILE = 64, STRIP = 32, WARPS = 4, THREADS = WARPS * 32;
constexpr int MAX_REQUESTS = 512;            // of a launch: their first tiles and lengths lie in shared memory
constexpr int MOST_COLS = 24;               // query rows of a row of the schedule
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float SHIFT = 7.f;                 // the reference of a row's weights is its largest score less SHIFT, or up to 8 below that
constexpr float NONE = -3e38f;               // the reference of a row that has seen no key: any score is far above it

struct Params {
  const void* q;
  const uint8_t* cache;
  const int* block_table;
  const int* seq_lens;
  const int* qsl;            // null: a token each
  void* out;
  float* lse;
  const float* sinks;
  float* part;               // [CTA][a row that began in front of the CTA's tiles, the one it leaves unfinished][COLS][D + 2]: output, maximum, sum
  int2* info;                // [row]: its first CTA, and how many
  int64_t q_stride, out_stride, bt_stride, num_blocks;
  int B, Hkv, G, BS, max_rows, few, ctas, chunks, extra, parts, window, bf16, shift;      // shift: of BS where that is a power of two, or -1
  uint32_t over_g;           // 2^32 / G, rounded up (0: G is 1)
  float scale_log2, ku, c2, out_scale;
};

// Token of a query row: r / G for r below 2^16 and G up to 2^6 (a dozen divisions a row were a fifth of its end)
VB_DEVICE int token_of(const Params& p, int r) { return p.over_g ? (int)__umulhi((uint32_t)r, p.over_g) : r; }

struct Request {
  int n, t;                  // rows in the cache, new tokens among them (0: none of this kernel's)
  VB_DEVICE int first_key(const Params& p) const { return p.window > 0 ? max(n - t - p.window + 1, 0) : 0; }      // that any of its rows sees
  VB_DEVICE int first_tile(const Params& p) const { return first_key(p) / TILE; }
  VB_DEVICE int tiles(const Params& p) const { return n > 0 && t > 0 ? (n + TILE - 1) / TILE - first_tile(p) : 0; }
  VB_DEVICE int chunks(const Params& p, int cols) const { return (t * p.G + cols - 1) / cols; }
};
VB_DEVICE Request request(const Params& p, int b) {
  Request r;
  r.n = min(max(p.seq_lens[b], 0), p.max_rows);
  r.t = p.qsl ? p.qsl[b + 1] - p.qsl[b] : 1;
  if (r.t > p.few || r.t < 0) r.t = 0;
  return r;
}
VB_DEVICE int slots_of(const Params& p, const Request& r) {          // a row's tiles, and what its end costs in tiles
  const int n = r.tiles(p);
  return n > 0 ? n + p.extra : 0;
}

// first[b]: slots of all rows in front of request b, as if each request had one kv head; first[B]: of all
VB_DEVICE void scan_tiles(const Params& p, int cols, int* first, int2* reqs, int* warp_sums) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    int mine = 0;
    if (b < p.B) {
      const Request r = request(p, b);
      reqs[b] = make_int2(r.n, r.t);
      mine = slots_of(p, r) * r.chunks(p, cols);
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
    for (int i = 0; i < WARPS; ++i) {
      if (i < w) before += warp_sums[i];
      base += warp_sums[i];
    }
    if (b < p.B) first[b] = before + x - mine;
    __syncthreads();
  }
  if (threadIdx.x == 0) first[p.B] = base;
  __syncthreads();
}

// A row: request, kv head, chunk of query rows; its slots are [begin, end) of the order of all
struct Row {
  int b, h, c, begin, end;
};
VB_DEVICE void row_at(const Params& p, int cols, const int* first, const int2* reqs, int tile, Row& r) {      // the row that has this tile
  int lo = 0, hi = p.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] * p.Hkv <= tile) lo = mid; else hi = mid - 1;
  }
  const Request q{reqs[lo].x, reqs[lo].y};               // (it has slots: the last request that begins at or in front of the tile)
  const int n = slots_of(p, q), chunks = q.chunks(p, cols), i = (tile - first[lo] * p.Hkv) / n;
  r.b = lo;
  r.h = chunks == 1 ? i : i / chunks;
  r.c = i - r.h * chunks;
  r.begin = first[lo] * p.Hkv + i * n;
  r.end = r.begin + n;
}
VB_DEVICE void next_row(const Params& p, int cols, const int* first, const int2* reqs, Row& r) {                     // behind it there is one more
  Request q{reqs[r.b].x, reqs[r.b].y};
  if (++r.c == q.chunks(p, cols)) {
    r.c = 0;
    if (++r.h == p.Hkv) {
      r.h = 0;
      do { ++r.b; } while (first[r.b + 1] == first[r.b]);
      q = Request{reqs[r.b].x, reqs[r.b].y};
    }
  }
  r.begin = r.end;
  r.end = r.begin + slots_of(p, q);
}

VB_DEVICE void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
VB_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> VB_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

VB_DEVICE void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit values, two to a lane, with rows and columns exchanged
VB_DEVICE uint32_t turn8(uint32_t x) { uint32_t r; asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x)); return r; }

// N neighbouring bytes of shared memory as words; `at` is a multiple of what N is one of: 16, 8, 4, 2 or 1.  What the last word has behind them are copies: conversions of
// codes that the compiler (nvcc 12.9) knows to be 0 came out as others'.
template <int N> struct Bytes {
  static constexpr int WORDS = (N + 3) / 4;
  uint32_t w[WORDS];
  VB_DEVICE void load(const unsigned char* at) {
    if constexpr (N % 16 == 0) {
#pragma unroll
      for (int i = 0; i < N / 16; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(at + 16 * i);
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      }
    } else if constexpr (N % 8 == 0) {
#pragma unroll
      for (int i = 0; i < N / 8; ++i) {
        const uint2 x = *reinterpret_cast<const uint2*>(at + 8 * i);
        w[2 * i] = x.x; w[2 * i + 1] = x.y;
      }
    } else if constexpr (N % 4 == 0) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(at + 4 * i);
    } else {
      constexpr int S = N % 2 == 0 ? 2 : 1;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        uint32_t x = 0;
#pragma unroll
        for (int j = 0; j < 4; j += S)
          if (4 * i + j < N) x |= (S == 2 ? (uint32_t)*reinterpret_cast<const uint16_t*>(at + 4 * i + j) : (uint32_t)at[4 * i + j]) << (8 * j);
        w[i] = 4 * i + 4 <= N ? x : N % 4 == 2 ? x | x << 16 : N % 4 == 1 ? x * 0x01010101u : x | x << 24;
      }
    }
  }
};

template <int D_> struct Form {
  static constexpr int D = D_, KD = D / 16;
  static constexpr int CODES = STRIP * D / 2, SIDE = CODES + STRIP * D / 16, STAGE = 2 * SIDE;       // bytes of a strip's keys, values behind them
  static constexpr int STAGES = D <= 64 ? 3 : 2;
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int EXCH = WARPS * KD * 4 * 128, MAXIMA = WARPS * MOST_COLS * 8;   // the warps' outputs of eight query rows; maxima and sums of all
  static constexpr int lists(int B) { return ((3 * B + 2 + WARPS) * 4 + 15) & ~15; }                 // first tiles, lengths and new tokens of B requests
  static constexpr int PART = MOST_COLS * (D + 2 + 9) * 4;                 // of a CTA of a cluster, instead of the lists
  static constexpr int FIXED = RING + EXCH + MAXIMA;
  // a lane's D / 4 values of a key lie in GK groups, its D / 8 values of a value row in GV
  static constexpr int SK = D / 4, SV = D / 8;
  static constexpr int GK = SK % 16 == 0 ? SK / 16 : 16 % SK == 0 ? 1 : 2, GV = SV % 16 == 0 ? SV / 16 : 16 % SV == 0 ? 1 : 2;
  static constexpr bool STRAIGHT_K = SK % 16 == 0 || 16 % SK == 0, STRAIGHT_V = SV % 16 == 0 || 16 % SV == 0;
};

// BF16: type of queries and outputs, or fp16
template <int D, int NT, bool BF16, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) attention_kernel(const Params p) {
  using F = Form<D>;
  constexpr int KD = F::KD, STAGES = F::STAGES, COLS = 8 * NT, PD = D + 2;
  extern __shared__ __align__(128) unsigned char smem[];
  float* exch = reinterpret_cast<float*>(smem + F::RING);
  float2* maxima = reinterpret_cast<float2*>(smem + F::RING + F::EXCH);    // [warp][column]
  int2* reqs = reinterpret_cast<int2*>(smem + F::FIXED);
  int* first = reinterpret_cast<int*>(reqs + p.B);
  int* warp_sums = first + p.B + 1;
  float* part_s = reinterpret_cast<float*>(smem + F::FIXED);               // cluster: the CTA's part
  float* factor_s = part_s + COLS * PD;                                    // ... and factors of the parts
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool fused = p.parts > 0, capped = p.ku != 0.f;
  pdl_wait();
  pdl_trigger();             // (here: the joining kernel may read the lengths as soon as it starts)
  int t0, t1, per;
  Row row;
  Request req;
  const int rank = fused ? blockIdx.x : 0;
  if (fused) {
    row.b = blockIdx.z;
    row.h = p.chunks == 1 ? blockIdx.y : blockIdx.y / p.chunks;
    row.c = blockIdx.y - row.h * p.chunks;
    req = request(p, row.b);
    row.begin = 0;
    row.end = row.c < req.chunks(p, COLS) ? req.tiles(p) : 0;
    per = (row.end + p.parts - 1) / p.parts;
    t0 = min(rank * per, row.end);
    t1 = min(t0 + per, row.end);
  } else {
    scan_tiles(p, COLS, first, reqs, warp_sums);
    const int total = first[p.B] * p.Hkv;
    per = (total + p.ctas - 1) / p.ctas;
    t0 = blockIdx.x * per;
    t1 = min(t0 + per, total);
    if (t0 >= t1) return;
    row_at(p, COLS, first, reqs, t0, row);
    req = Request{reqs[row.b].x, reqs[row.b].y};
  }

  unsigned char* ring = smem + warp * (STAGES * F::STAGE);
  const int64_t page = fp4::page_bytes(p.BS, D);
  // The warp's strips: flat numbers PER_TILE t0 + warp + i WARPS.  Where their halves lie is looked up for 32 strips at once, a lane each: number of the page of a head
  // (below 2^31: pages have 144 bytes or more) and row in it (-1: nothing to fetch).  Where pages are multiples of a strip the halves lie together.
  constexpr int PER_TILE = TILE / STRIP;
  const int s_end = t1 * PER_TILE;
  const bool together = p.BS % STRIP == 0;
  uint32_t my_page[2] = {0u, 0u};
  int my_off[2] = {-1, -1}, fetched = 0;
  const int64_t to_v = p.Hkv * page, codes = (int64_t)p.BS * (D / 2);
  auto copy_codes = [&](uint32_t to, const uint8_t* from, auto pieces) {   // pieces of 16 bytes
    constexpr int N = decltype(pieces)::value;
#pragma unroll
    for (int i = 0; i < (N + 31) / 32; ++i) {
      const int j = i * 32 + lane;
      if (N % 32 == 0 || j < N) {
        const int d = D == 128 ? (j & ~3) | ((j & 3) ^ (j >> 3 & 2)) : j;  // (D = 128: pieces of a row change places so that lanes of a load meet in no bank)
        cp_async16(to + d * 16, from + j * 16);
        cp_async16(to + F::SIDE + d * 16, from + to_v + j * 16);
      }
    }
  };
  auto copy_scales = [&](uint32_t to, const uint8_t* from, auto pieces) {  // of keys, then of values
    constexpr int N = decltype(pieces)::value;
#pragma unroll
    for (int i = 0; i < (2 * N + 31) / 32; ++i) {
      const int j = i * 32 + lane, side = j >= N, jj = j - side * N;
      if (2 * N % 32 == 0 || j < 2 * N) cp_async16(to + F::CODES + side * F::SIDE + jj * 16, from + codes + (side ? to_v : 0) + jj * 16);
    }
  };
  auto fetch = [&](int stage) {
    if ((fetched & 31) == 0) {
      const int s = t0 * PER_TILE + warp + (fetched + lane) * WARPS;
      my_off[0] = my_off[1] = -1;
      if (s < s_end) {
        Row r = row;
        Request q = req;
        if (!fused) {
          row_at(p, COLS, first, reqs, s / PER_TILE, r);
          q = Request{reqs[r.b].x, reqs[r.b].y};
        }
        const int tok = (s / PER_TILE - r.begin + q.first_tile(p)) * TILE + s % PER_TILE * STRIP;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int at = tok + half * 16;
          if (at < q.n) {
            const int pg = p.shift >= 0 ? at >> p.shift : at / p.BS;
            int64_t blk = p.block_table[r.b * p.bt_stride + pg];
            if ((uint64_t)blk >= (uint64_t)p.num_blocks) blk = 0;           // (a table may not say that; nothing is read outside the cache)
            my_page[half] = (uint32_t)(blk * 2 * p.Hkv + r.h);
            my_off[half] = at - pg * p.BS;
          }
        }
      }
    }
    const uint32_t to = smem_u32(ring + stage * F::STAGE);
    const int off = __shfl_sync(0xffffffffu, my_off[0], fetched & 31);
    const uint8_t* base = p.cache + __shfl_sync(0xffffffffu, my_page[0], fetched & 31) * (uint64_t)(uint32_t)page;
    if (together) {                          // (rows of the page behind the last one come along)
      if (off >= 0) {
        copy_codes(to, base + off * (D / 2), std::integral_constant<int, D>{});
        copy_scales(to, base + off * (D / 16), std::integral_constant<int, D / 8>{});
      }
    } else {
      const int off2 = __shfl_sync(0xffffffffu, my_off[1], fetched & 31);
      const uint8_t* base2 = p.cache + __shfl_sync(0xffffffffu, my_page[1], fetched & 31) * (uint64_t)(uint32_t)page;
      if (off >= 0) {
        copy_codes(to, base + off * (D / 2), std::integral_constant<int, D / 2>{});
        copy_scales(to, base + off * (D / 16), std::integral_constant<int, D / 16>{});
      }
      if (off2 >= 0) {
        copy_codes(to + 8 * D, base2 + off2 * (D / 2), std::integral_constant<int, D / 2>{});
        copy_scales(to + D, base2 + off2 * (D / 16), std::integral_constant<int, D / 16>{});
      }
    }
    ++fetched;
    cp_async_commit();
  };
  const int r0 = lane >> 2, t4 = lane & 3, q0 = t4 * 2;
  // rows of a product in front of slots of the next: row r is key r ^ (r >> 1 & 1), so that the keys of neighbouring lanes lie in both halves of the banks
  const int key0 = r0 ^ (r0 >> 1 & 1);
  const int vkey[4] = {q0 + (t4 & 1), q0 + 1 - (t4 & 1), q0 + 8 + (t4 & 1), q0 + 9 - (t4 & 1)};
  int s = t0 * PER_TILE + warp, turn = 0;
  uint32_t q[KD][NT][2];
  float mult[NT][2];                                                        // of a column's sums: to powers of two, or to the cap
  int hi[NT][2];                                                            // last key that a column sees
  auto read_q = [&]() {                      // as they are
    const int first_q = p.qsl ? p.qsl[row.b] : row.b;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row.c * COLS + nt * 8 + r0, tok = token_of(p, r);
      const bool there = tok < req.t;
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(p.q) + (int64_t)(first_q + tok) * p.q_stride + (int64_t)(row.h * p.G + r - tok * p.G) * D + t4 * (D / 4);
      if constexpr (D % 32 == 0) {
#pragma unroll
        for (int k = 0; k < KD; k += 2) {
          const uint4 x = there ? *reinterpret_cast<const uint4*>(qp + k * 4) : make_uint4(0u, 0u, 0u, 0u);
          q[k][nt][0] = x.x; q[k][nt][1] = x.y; q[k + 1][nt][0] = x.z; q[k + 1][nt][1] = x.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < KD; ++k) {
          const uint2 x = there ? *reinterpret_cast<const uint2*>(qp + k * 4) : make_uint2(0u, 0u);
          q[k][nt][0] = x.x; q[k][nt][1] = x.y;
        }
      }
    }
  };
  auto convert_q = [&]() {                   // to fp16, with the factor of their products
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mine = 1.f;
      if (BF16) {
        uint32_t most = 0u;                  // of the halves' bits without their signs
#pragma unroll
        for (int k = 0; k < KD; ++k) most = __vmaxu2(most, __vmaxu2(q[k][nt][0] & 0x7fff7fffu, q[k][nt][1] & 0x7fff7fffu));
        most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = min(max((int)(max(most & 0xffffu, most >> 16) >> 7), 27), 254);        // of the exponent's field; [2^-100, 2^127]
        const float f = __uint_as_float((uint32_t)(127 + 14 - e + 127) << 23);               // 2^(14 - (e - 127)), at least 2^-113
        mine = __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
        for (int k = 0; k < KD; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 x = unpack2<__nv_bfloat16>(q[k][nt][j]);
            q[k][nt][j] = pack2<__half>(x.x * f, x.y * f);
          }
      }
      mine *= capped ? p.ku : p.scale_log2;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        mult[nt][u] = __shfl_sync(0xffffffffu, mine, (q0 + u) * 4);
        hi[nt][u] = req.n - req.t + token_of(p, row.c * COLS + nt * 8 + q0 + u);
      }
    }
  };
  read_q();                                  // (on their way together with the first strips)
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(i);
  while (true) {
    convert_q();
    const int seg_end = min(row.end, t1) * PER_TILE, n = req.n, tile0 = req.first_tile(p), low = req.first_key(p);
    float o[KD][NT][4], m_run[NT][2], l_run[NT][2];
    // a reference of 2^20 or more: products of scores and their factor are rounded before it is taken off, as the reference was.  What a fused subtraction would keep of them, up to 1/16
    // there, grows with them, and as an exponent becomes a weight of its own
    bool huge = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < KD; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][nt][j] = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) { m_run[nt][u] = NONE; l_run[nt][u] = 0.f; }
    }
    for (; s < seg_end; s += WARPS) {
      const int stage = turn;
      turn = turn + 1 == STAGES ? 0 : turn + 1;
      cp_async_wait<STAGES - 2>();
      __syncwarp();
      fetch(stage == 0 ? STAGES - 1 : stage - 1);                          // into the stage of the strip before, which the whole warp has read
      const int tok = (s / PER_TILE - row.begin + tile0) * TILE + s % PER_TILE * STRIP;
      if (tok >= n) continue;
      const unsigned char* ks = ring + stage * F::STAGE;
      const unsigned char* vs = ks + F::SIDE;
      // ---- values of the strip as they are, on their way while the scores are computed
      const int gv0 = r0 * F::SV / 16, crossv = (16 - r0 * F::SV % 16) / 2;
      Bytes<D / 16> vc[2][4];
      uint32_t sa[2][F::GV], sb[2][F::GV];                                           // scales of the keys of slots (0, 1) and (8, 9)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = r0 * (D / 16);
          vc[m][j].load(vs + (m * 16 + vkey[j]) * (D / 2) + (D == 128 ? (((at >> 4) ^ (vkey[j] >> 1 & 2)) << 4 | (at & 15)) : at));
        }
#pragma unroll
        for (int g = 0; g < F::GV; ++g) {
          const unsigned char* at = vs + F::CODES + m * D + min(gv0 + g, D / 16 - 1);
          uint32_t x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = at[vkey[j] * (D / 16)];
          if (tok + STRIP > n || tok < low)      // rows of nobody, or that no query row sees, may hold what a weight of 0 does not cancel
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = tok + m * 16 + vkey[j] < n && tok + m * 16 + vkey[j] >= low ? x[j] : 0u;
          sa[m][g] = fp4::scales2(x[0] | x[1] << 8);
          sb[m][g] = fp4::scales2(x[2] | x[3] << 8);
        }
      }
      // ---- S^T = K Q^T, 16 keys at a time
      float sc[2][NT][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[m][nt][i] = 0.f;
        Bytes<D / 8> c0, c1;
        const int key = m * 16 + key0, piece = D == 128 ? (t4 ^ (key0 >> 1 & 2)) * 16 : t4 * (D / 8);
        c0.load(ks + key * (D / 2) + piece);
        c1.load(ks + (key + 8) * (D / 2) + piece);
        uint32_t s0[F::GK], s1[F::GK];
        const int g0 = t4 * F::SK / 16, cross = (16 - t4 * F::SK % 16) / 4;          // (not STRAIGHT_K: the lane's values from the cross-th four on are the next group's)
        const unsigned char* sp = ks + F::CODES + key * (D / 16);
        if constexpr (F::GK % 2 == 0 && F::STRAIGHT_K && D / 16 % 2 == 0) {           // two scales of a key at once
#pragma unroll
          for (int g = 0; g < F::GK; g += 2) {
            const uint32_t x = fp4::scales2(*reinterpret_cast<const uint16_t*>(sp + g0 + g)), y = fp4::scales2(*reinterpret_cast<const uint16_t*>(sp + 8 * (D / 16) + g0 + g));
            s0[g] = fp4::low2(x); s0[g + 1] = fp4::high2(x);
            s1[g] = fp4::low2(y); s1[g + 1] = fp4::high2(y);
          }
        } else {
#pragma unroll
          for (int g = 0; g < F::GK; ++g) {
            const unsigned char* at = sp + min(g0 + g, D / 16 - 1);
            const uint32_t two = fp4::scales2(at[0] | (uint32_t)at[8 * (D / 16)] << 8);
            s0[g] = fp4::low2(two);
            s1[g] = fp4::high2(two);
          }
        }
#pragma unroll
        for (int w = 0; w < (KD + 1) / 2; ++w) {                                     // a word: two steps of the product
          uint32_t a[4], b[4];
          fp4::unpack8(c0.w[w], a);
          fp4::unpack8(c1.w[w], b);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int k = 2 * w + half;
            if (k < KD) {
              const uint32_t f0 = F::STRAIGHT_K ? s0[F::GK > 1 ? k / 4 : 0] : k < cross ? s0[0] : s0[F::GK - 1];
              const uint32_t f1 = F::STRAIGHT_K ? s1[F::GK > 1 ? k / 4 : 0] : k < cross ? s1[0] : s1[F::GK - 1];
              const uint32_t a0 = fp4::mul2(a[2 * half], f0), a2 = fp4::mul2(a[2 * half + 1], f0), a1 = fp4::mul2(b[2 * half], f1), a3 = fp4::mul2(b[2 * half + 1], f1);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816(sc[m][nt], a0, a1, a2, a3, q[k][nt][0], q[k][nt][1]);
            }
          }
        }
      }
      // ---- weights
      const bool cut = tok + STRIP > n - req.t + 1 || (p.window > 0 && tok < n - p.window);
      uint32_t ph[2][NT][2], pl[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float by[2] = {mult[nt][0], mult[nt][1]};
        if (capped || cut || huge) {
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float x = sc[m][nt][i] * mult[nt][i & 1];
              if (capped) x = prompt::cap_any(x, p.c2);
              const int key = tok + m * 16 + key0 + (i >> 1) * 8, last = hi[nt][i & 1];
              sc[m][nt][i] = key > last || (p.window > 0 && key <= last - p.window) ? -INFINITY : x;
            }
          by[0] = by[1] = 1.f;
        }
        float y[2][4], most[2];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) y[m][i] = fmaf(sc[m][nt][i], by[i & 1], -m_run[nt][i & 1]);
#pragma unroll
        for (int u = 0; u < 2; ++u) most[u] = fmaxf(fmaxf(y[0][u], y[0][2 + u]), fmaxf(y[1][u], y[1][2 + u]));
        // the old reference stays where no weight is above 2^(8 + SHIFT)
        if (__any_sync(0xffffffffu, fmaxf(most[0], most[1]) > 8.f + SHIFT)) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float mx = fmaxf(fmaxf(sc[0][nt][u], sc[0][nt][2 + u]), fmaxf(sc[1][nt][u], sc[1][nt][2 + u])) * by[u];
            if (by[u] < 0.f) mx = fminf(fminf(sc[0][nt][u], sc[0][nt][2 + u]), fminf(sc[1][nt][u], sc[1][nt][2 + u])) * by[u];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            const float was = m_run[nt][u], at = fmaxf(mx - SHIFT, NONE);
            const bool up = at > was + 8.f;
            const float alpha = up ? ex2(was - at) : 1.f;
            m_run[nt][u] = up ? at : was;
            l_run[nt][u] *= alpha;
#pragma unroll
            for (int i = 0; i < KD; ++i) { o[i][nt][u] *= alpha; o[i][nt][2 + u] *= alpha; }
          }
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[m][i] = __fsub_rn(__fmul_rn(sc[m][nt][i], by[i & 1]), m_run[nt][i & 1]);
          huge |= __any_sync(0xffffffffu, (m_run[nt][0] > NONE && fabsf(m_run[nt][0]) > 0x1p20f) || (m_run[nt][1] > NONE && fabsf(m_run[nt][1]) > 0x1p20f));
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const float a = ex2(y[m][2 * t]), b = ex2(y[m][2 * t + 1]);
            l_run[nt][0] += a; l_run[nt][1] += b;
            const uint32_t h = pack2<__half>(a, b);
            ph[m][nt][t] = turn8(h);
            if (!BF16) {
              const float2 back = unpack2<__half>(h);
              pl[m][nt][t] = turn8(pack2<__half>(a - back.x, b - back.y));
            }
          }
      }
      // ---- O^T += V^T P^T, 16 keys at a time
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int w = 0; w < Bytes<D / 16>::WORDS; ++w) {
          // the nibbles of two keys next to each other: bytes of even values, and of odd ones
          constexpr uint32_t LOW = 0x0f0f0f0fu;
          uint32_t e01[4], o01[4], e23[4], o23[4];
          fp4::unpack8((vc[m][0].w[w] & LOW) | ((vc[m][1].w[w] << 4) & ~LOW), e01);
          fp4::unpack8(((vc[m][0].w[w] >> 4) & LOW) | (vc[m][1].w[w] & ~LOW), o01);
          fp4::unpack8((vc[m][2].w[w] & LOW) | ((vc[m][3].w[w] << 4) & ~LOW), e23);
          fp4::unpack8(((vc[m][2].w[w] >> 4) & LOW) | (vc[m][3].w[w] & ~LOW), o23);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = 4 * w + j;
            if (i < KD) {
              const uint32_t f0 = F::STRAIGHT_V ? sa[m][F::GV > 1 ? i / 8 : 0] : i < crossv ? sa[m][0] : sa[m][F::GV - 1];
              const uint32_t f1 = F::STRAIGHT_V ? sb[m][F::GV > 1 ? i / 8 : 0] : i < crossv ? sb[m][0] : sb[m][F::GV - 1];
              const uint32_t a0 = fp4::mul2(e01[j], f0), a1 = fp4::mul2(o01[j], f0), a2 = fp4::mul2(e23[j], f1), a3 = fp4::mul2(o23[j], f1);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816(o[i][nt], a0, a1, a2, a3, ph[m][nt][0], ph[m][nt][1]);
                if (!BF16) mma16816(o[i][nt], a0, a1, a2, a3, pl[m][nt][0], pl[m][nt][1]);
              }
            }
          }
        }
      }
    }
    // ---- the warps' results of the segment meet in shared memory
    const int index = (row.b * p.Hkv + row.h) * p.chunks + row.c, live = row.begin + req.tiles(p);       // (behind its tiles a row has further slots)
    const bool empty = !fused && max(row.begin, t0) >= live;
    const bool whole = !fused && row.begin >= t0 && live <= t1;
    if (!fused && !empty && row.begin >= t0 && threadIdx.x == 0) p.info[index] = make_int2(blockIdx.x, whole ? 1 : (live - 1) / per - (int)blockIdx.x + 1);
    const Row done = row;
    const Request done_req = req;
    const bool more = !fused && row.end < t1;
    if (more) {                              // (the next row's queries are on their way meanwhile)
      next_row(p, COLS, first, reqs, row);
      req = Request{reqs[row.b].x, reqs[row.b].y};
      read_q();
    }
    if (!empty) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l_run[nt][u] += __shfl_xor_sync(0xffffffffu, l_run[nt][u], x);
          if (m_run[nt][u] == NONE) m_run[nt][u] = l_run[nt][u] == 0.f ? -INFINITY : 0.f;        // (nothing seen, or nothing but NaN)
          if (r0 == 0) maxima[warp * MOST_COLS + nt * 8 + q0 + u] = make_float2(m_run[nt][u], l_run[nt][u]);
        }
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top[2], total[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float2 ml[WARPS];
#pragma unroll
          for (int w = 0; w < WARPS; ++w) ml[w] = maxima[w * MOST_COLS + nt * 8 + q0 + u];
          top[u] = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
          total[u] = 0.f;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) total[u] += ml[w].x == -INFINITY ? 0.f : ml[w].y * ex2(ml[w].x - top[u]);
          const float f = m_run[nt][u] == -INFINITY ? 0.f : ex2(m_run[nt][u] - top[u]);
#pragma unroll
          for (int i = 0; i < KD; ++i) { o[i][nt][u] *= f; o[i][nt][2 + u] *= f; }
        }
        float* to = exch + warp * (KD * 128) + lane;
#pragma unroll
        for (int i = 0; i < KD; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) to[(i * 4 + j) * 32] = o[i][nt][j];
        __syncthreads();
        // a thread: a column's values of half of a lane's dimensions
        constexpr int HALF = (KD + 1) / 2;
        const int u = warp & 1, i0 = warp >> 1 ? HALF : 0, g = nt * 8 + q0 + u, r = done.c * COLS + g, tok = token_of(p, r), d0 = r0 * (D / 8) + 2 * i0;
        const float m = u ? top[1] : top[0], l = u ? total[1] : total[0];
        float2 x[HALF];
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
          x[i] = make_float2(0.f, 0.f);
          if (KD % 2 == 0 || i0 + i < KD) {
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
              const float* from = exch + w * (KD * 128) + ((i0 + i) * 4 + u) * 32 + lane;
              x[i].x += from[0];
              x[i].y += from[64];
            }
          }
        }
        if (tok < done_req.t) {
          if (whole) {                       // nobody else has keys of the row
            const int head = done.h * p.G + r - tok * p.G, first_q = p.qsl ? p.qsl[done.b] : done.b;
            const float sink = p.sinks ? p.sinks[head] * LOG2E : -INFINITY, most = fmaxf(m, sink), base = most == -INFINITY ? 0.f : most;
            const float sum = (m == -INFINITY ? 0.f : l * ex2(m - base)) + (p.sinks ? ex2(sink - base) : 0.f);
            const float f = sum == 0.f || m == -INFINITY ? 0.f : ex2(m - base) / sum * p.out_scale;
            uint32_t y[HALF];
#pragma unroll
            for (int i = 0; i < HALF; ++i) y[i] = BF16 ? pack2<__nv_bfloat16>(x[i].x * f, x[i].y * f) : pack2<__half>(x[i].x * f, x[i].y * f);
            uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + (int64_t)(first_q + tok) * p.out_stride + (int64_t)head * D + d0;
            if constexpr (HALF == 4 && KD == 8) {
              *reinterpret_cast<uint4*>(out) = make_uint4(y[0], y[1], y[2], y[3]);
            } else {
#pragma unroll
              for (int i = 0; i < HALF; ++i)
                if (KD % 2 == 0 || i0 + i < KD) reinterpret_cast<uint32_t*>(out)[i] = y[i];
            }
            if (p.lse && r0 == 0 && i0 == 0) p.lse[(int64_t)(first_q + tok) * p.Hkv * p.G + head] = sum > 0.f ? (base + log2f(sum)) * LN2 : sum == 0.f ? -INFINITY : sum;
          } else {
            float* part = (fused ? part_s : p.part + (int64_t)(2 * blockIdx.x + (done.begin >= t0)) * COLS * PD) + g * PD;
#pragma unroll
            for (int i = 0; i < HALF; ++i)
              if (KD % 2 == 0 || i0 + i < KD) *reinterpret_cast<float2*>(part + d0 + 2 * i) = x[i];
            if (r0 == 0 && i0 == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
          }
        }
        if (nt + 1 < NT) __syncthreads();                // (in front of the next row: the barrier behind the maxima)
      }
    }
    if (!more) break;
  }
  cp_async_wait<0>();
  if (fused) {
    cluster_sync();
    const uint32_t parts_at = smem_u32(part_s);
    const int live = min(max(req.t * p.G - row.c * COLS, 0), COLS), first_q = p.qsl ? p.qsl[row.b] : row.b;
    for (int g = warp; g < live; g += WARPS) {           // a warp: log-sum-exp of a column, its parts and the sink
      const uint32_t at = parts_at + (g * PD + D) * 4;
      const int r = row.c * COLS + g, tok = token_of(p, r), head = row.h * p.G + r - tok * p.G;
      const float m0 = lane < p.parts ? ld_dsmem_f32(dsmem_addr(at, lane)) : -INFINITY, l0 = lane < p.parts ? ld_dsmem_f32(dsmem_addr(at + 4, lane)) : 0.f;
      const float sink = p.sinks ? p.sinks[head] * LOG2E : -INFINITY;
      const float m = warp_max(fmaxf(m0, sink)), top = m == -INFINITY ? 0.f : m;
      const float l = warp_sum(m0 == -INFINITY ? 0.f : l0 * ex2(m0 - top)) + (p.sinks ? ex2(sink - top) : 0.f);
      if (lane < 8) factor_s[g * 9 + lane] = m0 == -INFINITY ? 0.f : ex2(m0 - top) / l * p.out_scale;
      if (lane == 0 && rank == 0 && p.lse) p.lse[(int64_t)(first_q + tok) * p.Hkv * p.G + head] = l > 0.f ? (top + log2f(l)) * LN2 : l == 0.f ? -INFINITY : l;
    }
    __syncthreads();
    for (int i = rank * THREADS + threadIdx.x; i < live * (D / 2); i += p.parts * THREADS) {
      const int g = i / (D / 2), d = i % (D / 2) * 2, r = row.c * COLS + g, tok = token_of(p, r);
      float2 x[8], acc = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 8; ++c) x[c] = c < p.parts ? ld_dsmem_f32x2(dsmem_addr(parts_at + (g * PD + d) * 4, c)) : make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float f = factor_s[g * 9 + c];
        if (c < p.parts) { acc.x += x[c].x * f; acc.y += x[c].y * f; }
      }
      *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.out) + (int64_t)(first_q + tok) * p.out_stride + (int64_t)(row.h * p.G + r - tok * p.G) * D + d) =
          BF16 ? pack2<__nv_bfloat16>(acc.x, acc.y) : pack2<__half>(acc.x, acc.y);
    }
    cluster_sync();                                      // the others may still read this CTA's part
  }
}

// Grid (columns of a row, rows of a request, requests): the outputs of rows that several CTAs had, and of rows without keys.  EACH: warps of a column; the block has JOINERS /
// EACH columns.  The first parts are on their way before it is known what they count for.
constexpr int JOINERS = 4, JOIN = JOINERS * 32, PAIRS = 4, AHEAD = 4;
template <int EACH>
__global__ void __launch_bounds__(JOIN) join_kernel(const Params p, int cols, int D) {
  __shared__ float2 sums[EACH > 1 ? EACH : 1][EACH > 1 ? 32 * PAIRS : 1];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.z, h = p.chunks == 1 ? blockIdx.y : blockIdx.y / p.chunks, c = blockIdx.y - h * p.chunks, index = b * p.Hkv * p.chunks + blockIdx.y, PD = D + 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = EACH > 1 ? warp : 0, col = blockIdx.x * (JOINERS / EACH) + (EACH > 1 ? 0 : warp), pairs = D / 2;
  const int2 at = p.info[index];                         // (says something where the request has keys and the row is one)
  const Request req = request(p, b);
  const int r = c * cols + col, tok = token_of(p, r);
  if (col >= cols || tok >= req.t) return;
  const int count = req.n > 0 ? at.y : 0;
  if (count == 1) return;                                // done where its keys were
  // of part i: the first is what its CTA left unfinished, the others are the first rows of theirs
  const float* x = p.part + ((int64_t)(count ? 2 * at.x : 0) * cols + col) * PD;
  auto part = [&](int i) { return x + (int64_t)(2 * i + (i == 0)) * cols * PD; };
  auto read = [&](int from, float2 (&y)[AHEAD][PAIRS]) { // parts from, from + EACH, ...
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
      for (int j = 0; j < PAIRS; ++j)
        if (from + k * EACH < count && lane + 32 * j < pairs) y[k][j] = *reinterpret_cast<const float2*>(part(from + k * EACH) + 2 * (lane + 32 * j));
  };
  float2 y[AHEAD][PAIRS];
  float2 ml = lane < count ? *reinterpret_cast<const float2*>(part(lane) + D) : make_float2(-INFINITY, 0.f);
  read(w, y);
  const int head = h * p.G + r - tok * p.G;
  const int64_t token = (p.qsl ? p.qsl[b] : b) + tok;
  const float sink = p.sinks ? p.sinks[head] * LOG2E : -INFINITY;
  float top = fmaxf(sink, ml.x);
  for (int i = 32 + lane; i < count; i += 32) top = fmaxf(top, part(i)[D]);
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - base), total = ml.x == -INFINITY ? 0.f : ml.y * f;
  for (int i = 32 + lane; i < count; i += 32) {
    const float2 v = *reinterpret_cast<const float2*>(part(i) + D);
    if (v.x > -INFINITY) total += v.y * ex2(v.x - base);
  }
  total = warp_sum(total) + (p.sinks ? ex2(sink - base) : 0.f);
  float2 acc[PAIRS];
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) acc[j] = make_float2(0.f, 0.f);
  for (int i = w, block = 0; i < count; i += AHEAD * EACH) {
    if (i / 32 != block) {                               // factors of the next 32 parts, a lane each (AHEAD EACH divides 32)
      block = i / 32;
      const float m = block * 32 + lane < count ? part(block * 32 + lane)[D] : -INFINITY;
      f = m == -INFINITY ? 0.f : ex2(m - base);
    }
    if (i != w) read(i, y);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const float g = __shfl_sync(0xffffffffu, f, (i + k * EACH) & 31);
      if (i + k * EACH < count)
#pragma unroll
        for (int j = 0; j < PAIRS; ++j)
          if (lane + 32 * j < pairs) { acc[j].x += y[k][j].x * g; acc[j].y += y[k][j].y * g; }
    }
  }
  if (lane == 0 && w == 0 && p.lse) p.lse[token * p.Hkv * p.G + head] = total > 0.f ? (base + log2f(total)) * LN2 : total == 0.f ? -INFINITY : total;
  const float by = total == 0.f ? 0.f : p.out_scale / total;
  uint16_t* to = reinterpret_cast<uint16_t*>(p.out) + token * p.out_stride + (int64_t)head * D;
  auto write = [&](int i, float2 v) { *reinterpret_cast<uint32_t*>(to + 2 * i) = p.bf16 ? pack2<__nv_bfloat16>(v.x * by, v.y * by) : pack2<__half>(v.x * by, v.y * by); };
  if constexpr (EACH == 1) {
#pragma unroll
    for (int j = 0; j < PAIRS; ++j)
      if (lane + 32 * j < pairs) write(lane + 32 * j, acc[j]);
  } else {
#pragma unroll
    for (int j = 0; j < PAIRS; ++j)
      if (lane + 32 * j < pairs) sums[w][lane + 32 * j] = acc[j];
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += JOIN) {
      float2 v = sums[0][i];
#pragma unroll
      for (int j = 1; j < EACH; ++j) { v.x += sums[j][i].x; v.y += sums[j][i].y; }
      write(i, v);
    }
  }
}

constexpr int ctas_of(int D, int NT) { return D <= 128 ? (NT == 1 ? 3 : 5 - NT) : 2; }            // of an SM

// Groups of eight query rows of a row of the schedule, for requests of up to `rows` of them
static int groups_of(int D, int rows) { return rows <= 8 ? 1 : rows <= 16 || D > 128 ? 2 : 3; }

// `clusters`: nothing is launched, the clusters of a row that the device runs at a time are counted.
template <int D, int NT, bool BF16>
static int launch(const Params& p, cudaStream_t st, int* clusters, int* ctas) {
  using F = Form<D>;
  auto k = attention_kernel<D, NT, BF16, ctas_of(D, NT)>;
  static std::atomic<uint64_t> devices{0};
  constexpr int MOST = F::FIXED + (F::lists(MAX_REQUESTS) > F::PART ? F::lists(MAX_REQUESTS) : F::PART);
  if (vb_allow_smem(reinterpret_cast<const void*>(k), MOST, devices) != cudaSuccess) return (int)cudaGetLastError();
  if (ctas) { *ctas = ctas_of(D, NT); return 0; }
  if (clusters) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = p.parts; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(p.parts); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = F::FIXED + F::PART; cfg.attrs = &attr; cfg.numAttrs = 1;
    return (int)cudaOccupancyMaxActiveClusters(clusters, k, &cfg);
  }
  if (p.parts > 0) {
    vb_launch_parts(k, dim3(p.parts, p.Hkv * p.chunks, p.B), dim3(THREADS), (size_t)(F::FIXED + F::PART), st, (unsigned)p.parts, p);
    return (int)cudaGetLastError();
  }
  vb_launch(k, dim3(p.ctas), dim3(THREADS), (size_t)(F::FIXED + F::lists(p.B)), st, p);
  // many columns have few parts each, and a warp will do (behind 64 x 1000: 4.3 us, where four warps a column took 6.6)
  const int cols = min(8 * NT, p.few * p.G);
  if ((int64_t)cols * p.Hkv * p.chunks * p.B >= 1024)
    vb_launch(join_kernel<1>, dim3((cols + JOINERS - 1) / JOINERS, p.Hkv * p.chunks, p.B), dim3(JOIN), (size_t)0, st, p, 8 * NT, D);
  else
    vb_launch(join_kernel<JOINERS>, dim3(cols, p.Hkv * p.chunks, p.B), dim3(JOIN), (size_t)0, st, p, 8 * NT, D);
  return (int)cudaGetLastError();
}
template <int D>
static int pick(const Params& p, int nt, cudaStream_t st, int* clusters, int* ctas) {
  if constexpr (D <= 128)
    if (nt == 3) return p.bf16 ? launch<D, 3, true>(p, st, clusters, ctas) : launch<D, 3, false>(p, st, clusters, ctas);
  if (p.bf16) return nt == 2 ? launch<D, 2, true>(p, st, clusters, ctas) : launch<D, 1, true>(p, st, clusters, ctas);
  return nt == 2 ? launch<D, 2, false>(p, st, clusters, ctas) : launch<D, 1, false>(p, st, clusters, ctas);
}
static int go(const Params& p, int D, int nt, cudaStream_t st, int* clusters = nullptr, int* ctas = nullptr) {
  switch (D) {
    case 32: return pick<32>(p, nt, st, clusters, ctas);
    case 64: return pick<64>(p, nt, st, clusters, ctas);
    case 80: return pick<80>(p, nt, st, clusters, ctas);
    case 96: return pick<96>(p, nt, st, clusters, ctas);
    case 128: return pick<128>(p, nt, st, clusters, ctas);
    case 192: return pick<192>(p, nt, st, clusters, ctas);
    case 256: return pick<256>(p, nt, st, clusters, ctas);
  }
  return -2;
}

}  // namespace afp4

// Of heads of D and `rows` query rows (new tokens x query heads of a kv head) at most: columns of a row, CTAs of an SM, and, where parts > 0, clusters of that
// many CTAs that the device runs at a time.
EXPORT int vb_attention_fp4_plan(int D, int rows, int parts, int* cols, int* ctas, int* clusters) {
  using namespace afp4;
  Params p{};
  p.parts = parts;
  const int nt = groups_of(D, rows);
  *cols = 8 * nt;
  int rc = go(p, D, nt, nullptr, nullptr, ctas);
  if (rc == 0 && parts > 0) rc = parts > 8 ? -1 : go(p, D, nt, nullptr, clusters);
  return rc;
}

// Requests of at most `few` new tokens (qsl null: one each); rows of q and out of the others are not touched.  `ws`: 2 ctas cols (D + 2) + 2 group Hkv chunks
// floats, chunks = ceil(few Hq / Hkv / cols).  group: requests of a launch, up to 512.  extra: tiles that a row counts for
// beside its own.  parts: CTAs of a cluster that has a row (one kernel, no `ws`); 0: equal runs.  max_rows: rows of a request that the block table has room for.
// lse [T, Hq] or null.
EXPORT int vb_attention_fp4(const void* q, const void* cache, int64_t num_blocks, const int* block_table, const int* seq_lens, const int* qsl, void* out, float* lse,
                            const float* sinks, float* ws, int B, int Hq, int Hkv, int D, int BS, int max_rows, int few, int64_t q_stride, int64_t out_stride,
                            int64_t bt_stride, int ctas, int extra, int parts, int group, int window, float scale, float soft_cap, float out_scale, int dtype,
                            cudaStream_t st) {
  using namespace afp4;
  if (B <= 0) return 0;
  if (group < 1 || group > MAX_REQUESTS || few < 1 || max_rows < 0 || ctas < 1 || extra < 0 || parts < 0 || parts > 8) return -1;
  if ((dtype != DT_BF16 && dtype != DT_F16) || BS < 16 || BS % 16 || Hkv < 1 || Hq % Hkv || q_stride % 8 || out_stride % 8) return -1;
  if (parts > 0 && B > group) return -1;
  Params p;
  p.Hkv = Hkv; p.G = Hq / Hkv; p.BS = BS; p.max_rows = max_rows; p.few = few; p.extra = extra; p.parts = parts; p.window = window; p.bf16 = dtype == DT_BF16;
  if ((int64_t)few * p.G > 4096 || p.G > 64) return -1;
  const int nt = groups_of(D, few * p.G);
  p.chunks = (few * p.G + 8 * nt - 1) / (8 * nt);
  if ((int64_t)Hkv * p.chunks > 65535) return -1;      // (a dimension of the grids)
  p.q_stride = q_stride; p.out_stride = out_stride; p.bt_stride = bt_stride; p.num_blocks = num_blocks; p.cache = (const uint8_t*)cache; p.sinks = sinks;
  p.scale_log2 = scale * LOG2E;
  p.ku = soft_cap > 0.f ? scale / soft_cap : 0.f; p.c2 = soft_cap * LOG2E; p.out_scale = out_scale;
  p.lse = lse;
  p.over_g = p.G > 1 ? (uint32_t)(((1ull << 32) + p.G - 1) / p.G) : 0u;
  p.shift = 0;
  while (1 << p.shift < BS) ++p.shift;
  if (1 << p.shift != BS) p.shift = -1;
  for (int b0 = 0; b0 < B; b0 += group) {
    p.B = B - b0 < group ? B - b0 : group;
    // with offsets, rows are where they say; without, request b0 + i has row b0 + i
    p.q = qsl ? q : reinterpret_cast<const char*>(q) + b0 * q_stride * 2;
    p.out = qsl ? out : reinterpret_cast<char*>(out) + b0 * out_stride * 2;
    p.lse = qsl || !lse ? lse : lse + (int64_t)b0 * Hq;
    p.qsl = qsl ? qsl + b0 : nullptr;
    p.block_table = block_table + b0 * bt_stride;
    p.seq_lens = seq_lens + b0;
    const int64_t rows = (int64_t)p.B * Hkv * p.chunks, tiles = rows * ((max_rows + TILE - 1) / TILE + extra);
    if (tiles >= (1 << 29)) return -3;                 // flat strip numbers are 32 bits
    p.ctas = (int)max((int64_t)1, min((int64_t)ctas, tiles));
    p.part = ws;
    p.info = reinterpret_cast<int2*>(ws + (int64_t)2 * p.ctas * 8 * nt * (D + 2));
    const int rc = go(p, D, nt, st);
    if (rc) return rc;
  }
  return 0;
}
