// A key-value cache in 4 bits (fp4.cuh): what writes it, and what reads it back in 16 bits.
//
// Write: keys (and queries, in place) are turned by their positions where there are any, x' = (a cos - b sin, b cos + a sin) in 32 bits, rounded once
// to the type as an unquantised cache would hold them; then keys and values are quantised.  With several axes a token has a position on each, and `axes`
// says which of them turns a pair.  The 32-bit steps are rounded one by one (no fused multiply-add) and quotients are IEEE divisions, so that codes
// are those of the definition, bit by bit: a value next to the border of two codes would move by half of itself.
//
// Read: rows of requests one after the other, or (for the attention kernels over 16-bit pages) as pages of a workspace.
//
// Both are bound by the bytes they move.
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
VB_DEVICE void angle(const Turn& r, int t, int pair, float& co, float& si) {
  const int a = r.axes ? min(max(r.axes[pair], 0), r.n_axes - 1) : 0;
  int64_t p = r.positions[a * r.pos_stride + t];
  p = p < 0 ? 0 : p >= r.table_rows ? r.table_rows - 1 : p;       // (nothing is read outside the table)
  const float* row = r.table + p * r.rot;
  co = row[pair];
  si = row[r.rot / 2 + pair];
}
VB_DEVICE float turn_a(float a, float b, float co, float si) { return __fsub_rn(__fmul_rn(a, co), __fmul_rn(b, si)); }
VB_DEVICE float turn_b(float a, float b, float co, float si) { return __fadd_rn(__fmul_rn(b, co), __fmul_rn(a, si)); }

// ROT: 0 none, 1 halves are pairs, 2 neighbours are pairs
template <typename T, int ROT>
__global__ void __launch_bounds__(256) write_kernel(T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, Turn turn, int Hq, int Hkv, int D,
                                                    int64_t q_stride, int64_t k_stride, int64_t v_stride, uint8_t* __restrict__ cache, int64_t num_slots,
                                                    const int64_t* __restrict__ slots, int BS, float k_factor, float v_factor) {
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, half = turn.rot / 2;
  const int64_t slot = slots[t];
  if (slot >= 0 && slot < num_slots) {
    const int64_t blk = slot / BS, bytes = fp4::page_bytes(BS, D);
    const int off = (int)(slot - blk * BS), chunks = D / N, side = Hkv * chunks, n = 2 * side;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
      const int i = i0 + threadIdx.x, j = min(i, n - 1), part = j >= side, h = (j - part * side) / chunks, c = (j - part * side) - h * chunks;
      if (i0 + (int)(threadIdx.x & ~31u) >= n) break;                 // (whole warps)
      const T* row = (part ? v + t * v_stride : k + t * k_stride) + (int64_t)h * D;
      const Vec16<T> x = ld16(row + c * N);
      float y[N];
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = to_f32(x.e[e]);
      if (ROT && !part && c * N < turn.rot) {
        if (ROT == 1) {
          const bool first = c * N < half;
          const Vec16<T> o = ld16(row + c * N + (first ? half : -half));
#pragma unroll
          for (int e = 0; e < N; ++e) {
            float co, si;
            angle(turn, t, c * N + e - (first ? 0 : half), co, si);
            const float other = to_f32(o.e[e]);
            y[e] = first ? turn_a(y[e], other, co, si) : turn_b(other, y[e], co, si);
          }
        } else {
#pragma unroll
          for (int e = 0; e < N; e += 2) {
            float co, si;
            angle(turn, t, (c * N + e) / 2, co, si);
            const float a = y[e], b = y[e + 1];
            y[e] = turn_a(a, b, co, si);
            y[e + 1] = turn_b(a, b, co, si);
          }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = to_f32(from_f32<T>(y[e]));
      }
      const float factor = part ? v_factor : k_factor;
      float top = 0.f;
      bool nan = false;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (factor != 1.f) y[e] = __fdiv_rn(y[e], factor);
        top = fmaxf(top, fabsf(y[e]));
        nan |= y[e] != y[e];
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));         // the other half of the group: D / 8 is even
      nan |= __shfl_xor_sync(0xffffffffu, (int)nan, 1) != 0;
      const uint32_t e8 = nan ? 0x7fu : fp4::scale_of(top);
      const float e4 = fp4::scale_value(e8);
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = e8 == 0u || nan ? 0.f : __fdiv_rn(y[e], e4) + 0.f;      // (no code of -0 for a -0)
      if (i < n) {
        uint8_t* page = cache + ((blk * 2 + part) * Hkv + h) * bytes;
        *reinterpret_cast<uint32_t*>(page + (int64_t)off * (D / 2) + c * (N / 2)) = fp4::pack8(y);
        if ((c & 1) == 0) page[(int64_t)BS * (D / 2) + (int64_t)off * (D / 16) + c / 2] = (uint8_t)e8;
      }
    }
  }
  if (ROT && q) {
    const int per = (ROT == 1 ? half : turn.rot) / N;
    for (int i = threadIdx.x; i < Hq * per; i += blockDim.x) {
      T* row = q + t * q_stride + (int64_t)(i / per) * D + (i % per) * N;
      Vec16<T> a = ld16(row), b;
      if (ROT == 1) {
        b = ld16(row + half);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          float co, si;
          angle(turn, t, (i % per) * N + e, co, si);
          const float x = to_f32(a.e[e]), y = to_f32(b.e[e]);
          a.e[e] = from_f32<T>(turn_a(x, y, co, si));
          b.e[e] = from_f32<T>(turn_b(x, y, co, si));
        }
        st16(row + half, b);
      } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          float co, si;
          angle(turn, t, ((i % per) * N + e) / 2, co, si);
          const float x = to_f32(a.e[e]), y = to_f32(a.e[e + 1]);
          a.e[e] = from_f32<T>(turn_a(x, y, co, si));
          a.e[e + 1] = from_f32<T>(turn_b(x, y, co, si));
        }
      }
      st16(row, a);
    }
  }
}

// A chunk of eight values of a row in T
template <typename T> VB_DEVICE Vec16<T> row_chunk(uint32_t codes, uint32_t scale, float factor) {
  uint32_t r[4];
  fp4::unpack8(codes, r);
  const uint32_t s2 = fp4::low2(fp4::scales2(scale));
  Vec16<T> o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = unpack2<__half>(fp4::mul2(r[i], s2));
    o.e[2 * i] = from_f32<T>(x.x * factor);
    o.e[2 * i + 1] = from_f32<T>(x.y * factor);
  }
  return o;
}

struct Source {
  const uint8_t* cache;
  int64_t num_blocks;
  const int* block_table;
  int64_t bt_stride;
  int width, BS, D, Hkv;
};
VB_DEVICE const uint8_t* page_of(const Source& s, int b, int part, int h, int tok) {
  int64_t blk = s.block_table[b * s.bt_stride + tok / s.BS];
  if ((uint64_t)blk >= (uint64_t)s.num_blocks) blk = 0;             // (a table may not say that; nothing is read outside the cache)
  return s.cache + ((blk * 2 + part) * s.Hkv + h) * fp4::page_bytes(s.BS, s.D);
}
VB_DEVICE void load_chunk(const Source& s, int b, int part, int h, int tok, int c, uint32_t& codes, uint32_t& scale) {
  const uint8_t* page = page_of(s, b, part, h, tok);
  const int off = tok % s.BS;
  codes = *reinterpret_cast<const uint32_t*>(page + (int64_t)off * (s.D / 2) + c * 4);
  scale = page[(int64_t)s.BS * (s.D / 2) + (int64_t)off * (s.D / 16) + c / 2];
}

// Grid (runs of ROWS rows, kv heads, requests): rows [first, first + n) of a request to rows [cu[b], cu[b + 1]) of k and v
constexpr int ROWS = 64, READERS = 256;
template <typename T>
__global__ void __launch_bounds__(READERS) gather_kernel(Source s, const int* __restrict__ cu, const int* __restrict__ starts, T* __restrict__ k, T* __restrict__ v,
                                                         int64_t k_stride, int64_t v_stride, int64_t num_rows, float k_factor, float v_factor) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.z, h = blockIdx.y, to = cu[b], n = cu[b + 1] - to, first = starts ? starts[b] : 0, chunks = s.D / N;
  const int r0 = blockIdx.x * ROWS, r1 = min(r0 + ROWS, n);
  for (int i = threadIdx.x; i < (r1 - r0) * chunks; i += READERS) {
    const int r = r0 + i / chunks, c = i % chunks;
    const int64_t tok = (int64_t)first + r;
    if ((uint64_t)((int64_t)to + r) >= (uint64_t)num_rows) continue;
    const bool real = tok >= 0 && tok < (int64_t)s.width * s.BS;
    uint32_t codes[2] = {0u, 0u}, scale[2] = {0u, 0u};
    if (real) {
      load_chunk(s, b, 0, h, (int)tok, c, codes[0], scale[0]);
      load_chunk(s, b, 1, h, (int)tok, c, codes[1], scale[1]);
    }
    st16(k + (int64_t)(to + r) * k_stride + (int64_t)h * s.D + c * N, row_chunk<T>(codes[0], scale[0], k_factor));
    st16(v + (int64_t)(to + r) * v_stride + (int64_t)h * s.D + c * N, row_chunk<T>(codes[1], scale[1], v_factor));
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
    if (tok < n && c < real) {
      load_chunk(s, b, 0, h, tok, c, codes[0], scale[0]);
      load_chunk(s, b, 1, h, tok, c, codes[1], scale[1]);
    }
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
  const int items = max(2 * Hkv * (D / N), rot ? Hq * (rot / (neox ? 2 * N : N)) : 0), threads = min(256, (items + 31) / 32 * 32);
  DISPATCH_HALF(dtype, TT, {
    auto kernel = rot == 0 ? write_kernel<TT, 0> : neox ? write_kernel<TT, 1> : write_kernel<TT, 2>;
    vb_launch(kernel, dim3(T), dim3(threads), 0, st, (TT*)q, (const TT*)k, (const TT*)v, turn, Hq, Hkv, D, q_stride, k_stride, v_stride, (uint8_t*)cache,
              num_blocks * BS, slots, BS, k_factor, v_factor);
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
  const Source s{(const uint8_t*)cache, num_blocks, block_table, bt_stride, width, BS, D, Hkv};
  DISPATCH_HALF(dtype, TT, vb_launch(gather_kernel<TT>, dim3((max_rows + ROWS - 1) / ROWS, Hkv, B), dim3(READERS), 0, st, s, cu, starts, (TT*)k, (TT*)v, k_stride, v_stride,
                                     num_rows, k_factor, v_factor));
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
  const Source s{(const uint8_t*)cache, num_blocks, block_table, bt_stride, width, BS, D, Hkv};
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
