// A key-value cache in 4 bits (fp4.cuh): what writes it, and what reads it back in 16 bits.
//
// Write: keys (and queries, in place) are turned by their positions where there are any, x' = (a cos - b sin, b cos + a sin) in 32 bits, rounded once
// to the type as an unquantised cache would hold them; then keys and values are quantised.  With several axes a token has a position on each, and `axes`
// says which of them turns a pair.  The 32-bit steps are rounded one by one (no fused multiply-add) and quotients are IEEE divisions, so that codes
// are those of the definition, bit by bit: a value next to the border of two codes would move by half of itself.
//
// Read: rows of requests one after the other, or (for the attention kernels over 16-bit pages) as pages of a workspace.
//
// Both are bound by the bytes they move: cached rows of 64 requests of 700 to 1301, 8 heads of 128, 60 us (bytes 51, 5.6 TB/s); a prompt of 8000 with 32 / 8 heads of
// 128 44 us for the write (173 MB, 3.9 TB/s; 47 where nothing is in L2) and 12 for the read.  Queries, which only turn, are three quarters of the write's bytes; its 30.7 M instructions of
// a warp issue in 63 % of the cycles, the integer pipe is busy in 41 %, and the 64 registers of four blocks an SM spill some: no one thing bounds it.
#include "fp4.cuh"

namespace {

constexpr int N = 8;                // values of a lane: half a group

struct Turn {
  const int64_t* positions;         // [axes, T]
  int64_t pos_stride;
  const int* axes;                  // [rot / 2] or null
  const float* table;               // [table_rows, rot]: cosines, sines
  int table_rows, rot, n_axes;
};
// Cosines and sines of the pairs of a block's tokens into shared memory, [tokens][2][rot / 2]: every head of a token takes them
VB_DEVICE void angles(const Turn& r, int t0, int tokens, float* to) {
  const int half = r.rot / 2;
  for (int i = threadIdx.x; i < tokens * half; i += blockDim.x) {
    const int t = i / half, pair = i - t * half, a = r.axes ? min(max(r.axes[pair], 0), r.n_axes - 1) : 0;
    int64_t p = r.positions[a * r.pos_stride + t0 + t];
    p = p < 0 ? 0 : p >= r.table_rows ? r.table_rows - 1 : p;     // (nothing is read outside the table)
    const float* row = r.table + p * r.rot + pair;
    to[t * r.rot + pair] = row[0];
    to[t * r.rot + half + pair] = row[half];
  }
  __syncthreads();
}
template <int M> VB_DEVICE void take(const float* at, float (&x)[M]) {          // M: 4 or 8; at a multiple of four
#pragma unroll
  for (int i = 0; i < M; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(at + i);
    x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
  }
}
VB_DEVICE float turn_a(float a, float b, float co, float si) { return __fsub_rn(__fmul_rn(a, co), __fmul_rn(b, si)); }
VB_DEVICE float turn_b(float a, float b, float co, float si) { return __fadd_rn(__fmul_rn(b, co), __fmul_rn(a, si)); }

// Quotients of values of 16 bits and a scale, for their codes: y r, r the rounded reciprocal, is off by less than 2^-20.  Borders of codes times a scale have seven significant
// bits, y has at most eleven, so a quotient that is not on a border is 2^-13 or more from it: as multiples of 2^-13 all quotients are on their side.  (A division for each value
// was a third of the kernel's instructions.)
VB_DEVICE float on_side(float y, float r) {
  constexpr float C = 1536.f;
  return __fsub_rn(__fadd_rn(__fmul_rn(y, r), C), C);
}

// Eight codes without the signs of zeros
VB_DEVICE uint32_t unsigned_zeros(uint32_t x) { return x & (0x77777777u | x << 1 | x << 2 | x << 3); }      // (the sign bit stays where one of the three below it is set)

// ROT: 0 none, 1 halves are pairs, 2 neighbours are pairs.  DC: head size and rotated part, or 0.  A lane has a group of 16 values.  A block has some tokens one after the
// other (several where there are many: their angles, which have to be waited for, come together); a thread's first rows are on their way before the angles are.
template <typename T, int ROT, int DC>
__global__ void __launch_bounds__(256, 4) write_kernel(T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, Turn turn, int Hq, int Hkv, int D_,
                                                    int64_t q_stride, int64_t k_stride, int64_t v_stride, uint8_t* __restrict__ cache, int64_t num_slots,
                                                    const int64_t* __restrict__ slots, int BS, int shift, float k_factor, float v_factor, int T_, int tokens) {
  extern __shared__ __align__(16) float angles_s[];
  pdl_trigger();
  pdl_wait();
  const int first_t = blockIdx.x * tokens, last_t = min(first_t + tokens, T_), D = DC ? DC : D_, rot = DC ? DC : turn.rot, half = rot / 2;
  const int groups = D / 16, side = Hkv * groups, n = 2 * side, per = ROT == 0 ? 1 : (ROT == 1 ? half : rot) / N, nq = ROT && q ? Hq * per : 0;
  struct Item { int part, h, g; };
  auto item = [&](int i) {
    const int part = i >= side, h = (i - part * side) / groups;
    return Item{part, h, i - part * side - h * groups};
  };
  auto turned = [&](const Item& m, int u) { return ROT && !m.part && m.g * 16 + u * N < rot; };       // u: half of the group
  auto load = [&](int t, const Item& m, Vec16<T> (&x)[2], Vec16<T> (&other)[2]) {
    const T* row = (m.part ? v + t * v_stride : k + t * k_stride) + m.h * D + m.g * 16;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      x[u] = ld16(row + u * N);
      if (ROT == 1 && turned(m, u)) other[u] = ld16(row + u * N + (m.g * 16 + u * N < half ? half : -half));
    }
  };
  auto q_row = [&](int t, int i) { const int h = i / per; return q + t * q_stride + h * D + (i - h * per) * N; };
  const int64_t bytes = fp4::page_bytes(BS, D);
  for (int t = first_t; t < last_t; ++t) {
    const float* angle_s = angles_s + (t - first_t) * rot;
    const int64_t slot = slots[t];
    const bool kept = slot >= 0 && slot < num_slots;
    Item m = item(threadIdx.x);
    Vec16<T> x[2], other[2], qa, qb;
    if (kept && (int)threadIdx.x < n) load(t, m, x, other);
    if ((int)threadIdx.x < nq) {
      qa = ld16(q_row(t, threadIdx.x));
      if (ROT == 1) qb = ld16(q_row(t, threadIdx.x) + half);
    }
    if (ROT && t == first_t) angles(turn, first_t, last_t - first_t, angles_s);
    if (kept) {
      const int64_t blk = shift >= 0 ? slot >> shift : slot / BS;       // (a division of 64 bits was a fifth of the kernel)
      const int off = (int)(slot - blk * BS);
      uint8_t* block = cache + blk * 2 * Hkv * bytes;
      for (int i = threadIdx.x; i < n; i += blockDim.x) {
        if (i >= (int)blockDim.x) {
          m = item(i);
          load(t, m, x, other);
        }
        float y[2][N];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int e = 0; e < N; ++e) y[u][e] = to_f32(x[u].e[e]);
          if (turned(m, u)) {
            const int c = m.g * 2 + u;
            if (ROT == 1) {
              const bool first = c * N < half;
              const float* at = angle_s + c * N - (first ? 0 : half);
              float co[N], si[N];
              take(at, co);
              take(at + half, si);
#pragma unroll
              for (int e = 0; e < N; ++e) y[u][e] = turn_b(to_f32(other[u].e[e]), y[u][e], co[e], first ? -si[e] : si[e]);      // (x - y is x + -y)
            } else {
              float co[N / 2], si[N / 2];
              take(angle_s + c * (N / 2), co);
              take(angle_s + half + c * (N / 2), si);
#pragma unroll
              for (int e = 0; e < N; e += 2) {
                const float a = y[u][e], b = y[u][e + 1];
                y[u][e] = turn_a(a, b, co[e / 2], si[e / 2]);
                y[u][e + 1] = turn_b(a, b, co[e / 2], si[e / 2]);
              }
            }
#pragma unroll
            for (int e = 0; e < N; e += 2) {
              const float2 r = unpack2<T>(pack2<T>(y[u][e], y[u][e + 1]));
              y[u][e] = r.x;
              y[u][e + 1] = r.y;
            }
          }
        }
        const float factor = m.part ? v_factor : k_factor;
        if (factor != 1.f)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) y[u][e] = __fdiv_rn(y[u][e], factor);
        uint32_t top = 0u;                                              // (of the bits: a NaN is above all numbers)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(y[u][e]) & 0x7fffffffu);
        const bool nan = top > 0x7f800000u;
        const uint32_t e8 = nan ? 0x7fu : fp4::scale_of(__uint_as_float(top));
        const float e4 = fp4::scale_value(e8);
        if (e8 == 0u || nan) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) y[u][e] = 0.f;
        } else if (factor != 1.f) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) y[u][e] = __fdiv_rn(y[u][e], e4);
        } else {
          const float r = __frcp_rn(e4);
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) y[u][e] = on_side(y[u][e], r);
        }
        uint2 codes = make_uint2(fp4::pack8(y[0]), fp4::pack8(y[1]));
        codes.x = unsigned_zeros(codes.x);
        codes.y = unsigned_zeros(codes.y);
        uint8_t* page = block + (m.part * Hkv + m.h) * bytes;
        *reinterpret_cast<uint2*>(page + off * (D / 2) + m.g * 8) = codes;
        page[BS * (D / 2) + off * (D / 16) + m.g] = (uint8_t)e8;
      }
    }
    if (ROT) {
      for (int i = threadIdx.x; i < nq; i += blockDim.x) {
        T* row = q_row(t, i);
        const int c = i % per;
        if (i >= (int)blockDim.x) {
          qa = ld16(row);
          if (ROT == 1) qb = ld16(row + half);
        }
        if (ROT == 1) {
          float co[N], si[N];
          take(angle_s + c * N, co);
          take(angle_s + half + c * N, si);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float a = to_f32(qa.e[e]), b = to_f32(qb.e[e]);
            qa.e[e] = from_f32<T>(turn_a(a, b, co[e], si[e]));
            qb.e[e] = from_f32<T>(turn_b(a, b, co[e], si[e]));
          }
          st16(row + half, qb);
        } else {
          float co[N / 2], si[N / 2];
          take(angle_s + c * (N / 2), co);
          take(angle_s + half + c * (N / 2), si);
#pragma unroll
          for (int e = 0; e < N; e += 2) {
            const float a = to_f32(qa.e[e]), b = to_f32(qa.e[e + 1]);
            qa.e[e] = from_f32<T>(turn_a(a, b, co[e / 2], si[e / 2]));
            qa.e[e + 1] = from_f32<T>(turn_b(a, b, co[e / 2], si[e / 2]));
          }
        }
        st16(row, qa);
      }
    }
  }
}

// A chunk of eight values of a row in T
template <typename T> VB_DEVICE Vec16<T> row_chunk(uint32_t codes, uint32_t scale, float factor) {
  uint32_t r[4];
  fp4::unpack8(codes, r);
  const uint32_t s2 = fp4::low2(fp4::scales2(scale));
  Vec16<T> o;
  uint32_t* w = &o.u.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = fp4::mul2(r[i], s2);
    if (DTypeOf<T>::v != DT_F16 || factor != 1.f) {
      float2 x = unpack2<__half>(w[i]);
      if (factor != 1.f) { x.x *= factor; x.y *= factor; }
      w[i] = pack2<T>(x.x, x.y);
    }
  }
  return o;
}

struct Source {
  const uint8_t* cache;
  int64_t num_blocks;
  const int* block_table;
  int64_t bt_stride;
  int width, BS, D, Hkv, shift;              // shift: of BS where that is a power of two, or -1
};
int shift_of(int BS) {
  int shift = 0;
  while (1 << shift < BS) ++shift;
  return 1 << shift == BS ? shift : -1;
}
Source source(const void* cache, int64_t num_blocks, const int* block_table, int64_t bt_stride, int width, int BS, int D, int Hkv) {
  return Source{(const uint8_t*)cache, num_blocks, block_table, bt_stride, width, BS, D, Hkv, shift_of(BS)};
}
// Codes and scales of a chunk of a row's keys and values
VB_DEVICE void load_chunk(const Source& s, int b, int h, int tok, int c, uint32_t (&codes)[2], uint32_t (&scale)[2]) {
  const int p = s.shift >= 0 ? tok >> s.shift : tok / s.BS, off = tok - p * s.BS, bytes = (int)fp4::page_bytes(s.BS, s.D);
  int64_t blk = s.block_table[b * s.bt_stride + p];
  if ((uint64_t)blk >= (uint64_t)s.num_blocks) blk = 0;             // (a table may not say that; nothing is read outside the cache)
  const uint8_t* k = s.cache + (uint32_t)(blk * 2 * s.Hkv + h) * (uint64_t)(uint32_t)bytes;      // (pages of heads have 144 bytes or more: below 2^31 of them)
  const int64_t to_v = (int64_t)s.Hkv * bytes;
  const int at = off * (s.D / 2) + c * 4, sc = s.BS * (s.D / 2) + off * (s.D / 16) + c / 2;
  codes[0] = *reinterpret_cast<const uint32_t*>(k + at);
  codes[1] = *reinterpret_cast<const uint32_t*>(k + to_v + at);
  scale[0] = k[sc];
  scale[1] = k[to_v + sc];
}

// Grid (runs of rows, requests): rows [first, first + n) of a request to rows [cu[b], cu[b + 1]) of k and v.  A block has all heads of a run of rows, so that what it
// writes lies together; a thread's loads are on their way before it writes.  EVEN: the chunks of a row divide the block, so that a thread stays with its chunk.
constexpr int READERS = 256, AHEAD = 4;
template <typename T, bool EVEN>
__global__ void __launch_bounds__(READERS) gather_kernel(Source s, const int* __restrict__ cu, const int* __restrict__ starts, T* __restrict__ k, T* __restrict__ v,
                                                         int64_t k_stride, int64_t v_stride, int64_t num_rows, int run, float k_factor, float v_factor) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, to = cu[b], n = cu[b + 1] - to, first = starts ? starts[b] : 0, chunks = s.D / N, wide = s.Hkv * chunks;
  const int r0 = blockIdx.x * run, rows = min(run, n - r0), items = rows * wide;
  const int r1 = threadIdx.x / wide, hc = threadIdx.x - r1 * wide, step = READERS / (EVEN ? wide : 1);
  for (int i0 = threadIdx.x, turn = 0; i0 < items; i0 += READERS * AHEAD, turn += AHEAD) {
    uint32_t codes[AHEAD][2], scale[AHEAD][2];
    auto row_of = [&](int j) { return EVEN ? r1 + (turn + j) * step : (i0 + j * READERS) / wide; };
    auto place_of = [&](int j) { return EVEN ? hc : (i0 + j * READERS) % wide; };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = i0 + j * READERS, r = row_of(j), at = place_of(j), h = at / chunks;
      const int64_t tok = (int64_t)first + r0 + r;
      codes[j][0] = codes[j][1] = scale[j][0] = scale[j][1] = 0u;
      if (i < items && tok >= 0 && tok < (int64_t)s.width * s.BS) load_chunk(s, b, h, (int)tok, at - h * chunks, codes[j], scale[j]);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = i0 + j * READERS, r = row_of(j), at = place_of(j);
      const int64_t row = (int64_t)to + r0 + r;
      if (i >= items || (uint64_t)row >= (uint64_t)num_rows) continue;
      st16(k + row * k_stride + at * N, row_chunk<T>(codes[j][0], scale[j][0], k_factor));
      st16(v + row * v_stride + at * N, row_chunk<T>(codes[j][1], scale[j][1], v_factor));
    }
  }
}

// Grid (pages of PS rows, kv heads, requests): the rows of requests with more than `few` new tokens as pages [pages, 2, Hkv, PS, W] of a workspace (W >= D, zeros behind
// the rows' values; VT: values of a page transposed, W = 128 and pages of 64), with the block table [B, gridDim.x] and the lengths that say so.  A request has as many pages
// as its rows need, behind those of the requests in front of it; the others have none, and a length of 0.  Rows behind the last one are zeros.
template <typename T, bool VT>
__global__ void __launch_bounds__(READERS) pages_kernel(Source s, const int* __restrict__ seq_lens, const int* __restrict__ qsl, int few, T* __restrict__ pages, int num_pages,
                                                        int PS, int W, int* __restrict__ table, int* __restrict__ lens) {
  __shared__ float red[32];
  __shared__ __align__(16) T tile[VT ? 64 * 130 : 1];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.z, h = blockIdx.y, p = blockIdx.x, real = s.D / N, width = gridDim.x;
  const int chunks = VT ? 128 / N : W / N;
  auto rows_of = [&](int i) {
    const int n = min(max(seq_lens[i], 0), s.width * s.BS);
    return qsl && qsl[i + 1] - qsl[i] <= few ? 0 : n;
  };
  const int n = rows_of(b);
  if (p * PS >= n) {
    if (h == 0 && threadIdx.x == 0) {
      table[(int64_t)b * width + p] = 0;
      if (p == 0) lens[b] = 0;
    }
    return;
  }
  int before = 0;
  for (int i = threadIdx.x; i < b; i += READERS) before += (rows_of(i) + PS - 1) / PS;
  const int base = (int)block_sum((float)before, red), page = base + p;           // (whole numbers below 2^24)
  const int room = min(max(num_pages - base, 0), width);                          // (the caller's workspace holds all)
  if (h == 0 && threadIdx.x == 0) {
    if (p == 0) lens[b] = min(n, room * PS);
    table[(int64_t)b * width + p] = p < room ? page : 0;
  }
  if (p >= room) return;
  const int w = VT ? 128 : W;
  T* kp = pages + ((int64_t)page * 2 * s.Hkv + h) * PS * w;
  T* vp = kp + (int64_t)s.Hkv * PS * w;
  for (int i = threadIdx.x; i < PS * chunks; i += READERS) {
    const int r = i / chunks, c = i % chunks, tok = p * PS + r;
    uint32_t codes[2] = {0u, 0u}, scale[2] = {0u, 0u};
    if (tok < n && c < real) load_chunk(s, b, h, tok, c, codes, scale);
    st16(kp + r * w + c * N, row_chunk<T>(codes[0], scale[0], 1.f));
    const Vec16<T> x = row_chunk<T>(codes[1], scale[1], 1.f);
    if (VT) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(tile + r * 130 + c * N);
      dst[0] = x.u.x; dst[1] = x.u.y; dst[2] = x.u.z; dst[3] = x.u.w;
    } else {
      st16(vp + r * w + c * N, x);
    }
  }
  if (VT) {
    __syncthreads();
    for (int i = threadIdx.x; i < 128 * 8; i += READERS) {
      const int d = i & 127, r = (i >> 7) * N;                        // (neighbouring lanes read neighbouring values of a row)
      Vec16<T> o;
#pragma unroll
      for (int e = 0; e < N; ++e) o.e[e] = tile[(r + e) * 130 + d];
      st16(vp + d * 64 + r, o);
    }
  }
}

// Rows [T, H, G, D] to [T, H, G2, D2] (chunks of eight values; zeros where there are none), or back
template <typename T>
__global__ void __launch_bounds__(READERS) fit_kernel(const T* __restrict__ x, T* __restrict__ y, int64_t n, int G, int G2, int from, int to, int64_t x_stride, int64_t y_stride,
                                                      int heads) {
  pdl_trigger();
  pdl_wait();
  for (int64_t i = (int64_t)blockIdx.x * READERS + threadIdx.x; i < n; i += (int64_t)gridDim.x * READERS) {
    const int c = (int)(i % to), hg = (int)(i / to % heads), h = hg / G2, g = hg - h * G2;      // (heads: of a row of y)
    const int64_t t = i / to / heads;
    Vec16<T> v;
    v.u = make_uint4(0u, 0u, 0u, 0u);
    if (c < from && g < G) v = ld16(x + t * x_stride + ((int64_t)(h * G + g) * from + c) * N);
    st16(y + t * y_stride + ((int64_t)hg * to + c) * N, v);
  }
}

bool bad_shape(int D, int BS, int dtype) { return (dtype != DT_BF16 && dtype != DT_F16) || D < 16 || D % 16 || BS < 16 || BS % 16; }

}  // namespace

// q [T, Hq D] is turned in place (null, or rot 0: none is); k, v [T, Hkv D] go to slots [T] (below 0 or behind the cache: nowhere).  positions [n_axes, T] with
// pos_stride between axes; axes [rot / 2] or null: the first.  All rows at 16-byte addresses.
EXPORT int vb_write_fp4(const int64_t* positions, int64_t pos_stride, int n_axes, const int* axes, const float* table, int table_rows, int rot, int neox, void* q,
                        const void* k, const void* v, int T, int Hq, int Hkv, int D, int64_t q_stride, int64_t k_stride, int64_t v_stride, void* cache,
                        int64_t num_blocks, const int64_t* slots, int BS, float k_factor, float v_factor, int dtype, cudaStream_t st) {
  if (T <= 0) return 0;
  if (bad_shape(D, BS, dtype) || Hkv < 1 || rot < 0 || rot > D || rot % 16 || (rot && (!positions || !table || table_rows < 1 || n_axes < 1))) return -1;
  const Turn turn{positions, pos_stride, axes, table, table_rows, rot, n_axes};
  const int items = max(2 * Hkv * (D / 16), rot ? Hq * (rot / (neox ? 2 * N : N)) : 0), threads = min(256, (items + 31) / 32 * 32);
  // tokens of a block: two halve the waits for angles, but need many blocks to fill the SMs, which hold 592.  us with 1 and 2 of them (4), 2000, 4000, 5331, 8000 and 16000 tokens: 32 / 8
  // heads of 128 14.5 and 13.4 (14.2), 25.8 and 24.5, 34.9 and 31.8 (34.0), 55.0 and 47.4 (47.0), 105 and 90 (85); 12 / 12 of 128 on three axes 12.1 and 12.7, 21.6 and 20.7, 28.8 and 26.6,
  // 44.9 and 39.8, 87 and 76; 16 / 4 of 64 6.1 and 9.6, 9.9 and 10.8, 12.8 and 13.2, 17.8 and 17.1, 33.3 and 31.2; 1000 tokens 8.2 and 8.2, 7.9 and 8.8, 5.5 and 8.9
  const int tokens = T >= 4096 ? 2 : 1;
  DISPATCH_HALF(dtype, TT, {
    auto kernel = rot == 0 ? write_kernel<TT, 0, 0> : !neox ? write_kernel<TT, 2, 0> : rot == 128 && D == 128 ? write_kernel<TT, 1, 128> : write_kernel<TT, 1, 0>;
    vb_launch(kernel, dim3((T + tokens - 1) / tokens), dim3(threads), (size_t)tokens * rot * 4, st, (TT*)q, (const TT*)k, (const TT*)v, turn, Hq, Hkv, D, q_stride, k_stride, v_stride,
              (uint8_t*)cache, num_blocks * BS, slots, BS, shift_of(BS), k_factor, v_factor, T, tokens);
  });
  return (int)cudaGetLastError();
}

// Rows [starts[b], ...) (null: from the first) of request b, cu[b + 1] - cu[b] <= max_rows of them, to rows from cu[b] on of k and v [num_rows, Hkv D]; a row that the
// block table [B, width] has no page for is zeros.
EXPORT int vb_gather_fp4(const void* cache, int64_t num_blocks, const int* block_table, int64_t bt_stride, int width, const int* cu, const int* starts, void* k, void* v,
                         int64_t k_stride, int64_t v_stride, int64_t num_rows, int B, int max_rows, int Hkv, int D, int BS, float k_factor, float v_factor, int dtype,
                         cudaStream_t st) {
  if (B <= 0 || max_rows <= 0 || num_rows <= 0) return 0;
  if (bad_shape(D, BS, dtype) || Hkv < 1 || Hkv > 65535 || B > 65535 || width < 0) return -1;
  const Source s = source(cache, num_blocks, block_table, bt_stride, width, BS, D, Hkv);
  const int wide = Hkv * (D / N), run = max(1, 1024 / wide);          // (four items of keys and values for every thread)
  if (((int64_t)max_rows + run - 1) / run > 0x7fffffff) return -1;
  DISPATCH_HALF(dtype, TT, {
    auto kernel = wide <= READERS && READERS % wide == 0 ? gather_kernel<TT, true> : gather_kernel<TT, false>;
    vb_launch(kernel, dim3((max_rows + run - 1) / run, B), dim3(READERS), 0, st, s, cu, starts, (TT*)k, (TT*)v, k_stride, v_stride, num_rows, run, k_factor, v_factor);
  });
  return (int)cudaGetLastError();
}

// Pages of a workspace [num_pages, 2, Hkv, PS, W] with table [B, table_width] and lens [B] of them, without the factors of keys and values.  few: requests of at most
// so many new tokens (qsl [B + 1]; null: all take part) are left out.
EXPORT int vb_pages_fp4(const void* cache, int64_t num_blocks, const int* block_table, int64_t bt_stride, int width, const int* seq_lens, const int* qsl, int few, void* pages,
                        int num_pages, int PS, int W, int vt, int* table, int table_width, int* lens, int B, int Hkv, int D, int BS, int dtype, cudaStream_t st) {
  if (B <= 0) return 0;
  if (bad_shape(D, BS, dtype) || Hkv < 1 || Hkv > 65535 || B > 65535 || width < 0 || table_width < 1 || PS < 1 || num_pages < 0 || W < D || W % N ||
      (vt && (W != 128 || PS != 64)))
    return -1;
  const Source s = source(cache, num_blocks, block_table, bt_stride, width, BS, D, Hkv);
  DISPATCH_HALF(dtype, TT, {
    auto kernel = vt ? pages_kernel<TT, true> : pages_kernel<TT, false>;
    vb_launch(kernel, dim3(table_width, Hkv, B), dim3(READERS), 0, st, s, seq_lens, qsl, few, (TT*)pages, num_pages, PS, W, table, lens);
  });
  return (int)cudaGetLastError();
}

// x [T, H, G, D] (row stride x_stride) to y [T, H, G2, D2]: values and heads behind the last are zeros, or left out.
EXPORT int vb_fit_rows(const void* x, void* y, int T, int H, int G, int D, int G2, int D2, int64_t x_stride, int64_t y_stride, int sms, int dtype, cudaStream_t st) {
  if (T <= 0) return 0;
  if ((dtype != DT_BF16 && dtype != DT_F16) || D % N || D2 % N || H < 1 || G < 1 || G2 < 1) return -1;
  const int64_t n = (int64_t)T * H * G2 * (D2 / N), blocks = (n + READERS - 1) / READERS;
  DISPATCH_HALF(dtype, TT, vb_launch(fit_kernel<TT>, dim3((unsigned)(blocks < 8 * sms ? blocks : 8 * sms)), dim3(READERS), 0, st, (const TT*)x, (TT*)y, n, G, G2, D / N, D2 / N,
                                     x_stride, y_stride, H * G2));
  return (int)cudaGetLastError();
}
