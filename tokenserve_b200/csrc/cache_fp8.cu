// Writing K/V rows into the 8-bit paged cache, rotary positions fused with that write, and
// reading rows back.
//
// The cache keeps, for K and V each, e4m3 codes [num_blocks][Hkv][block_size][D] and float32
// scales [num_blocks][Hkv][block_size]; fp8.cuh has the row format. Slots and block tables are
// those of the 16-bit pool (src/tokenserve/backends/base.py:40-45): slot s is row
// (s / block_size, h, s % block_size).
//
// All three are bound by HBM. A row's D elements are spread over D * size / 16 neighbouring lanes
// (one 16-byte vector each), so the row's amax is a few shuffles, the row is read once, and the
// half-layout rotary partner comes from another lane of the row instead of a second load. A thread
// has the vectors of four rows in flight, and no 64-bit division stands before them. Rows that do
// not split that way (odd sizes or alignment) take a warp per row with scalar accesses. Measured with
// heads of 128: append of 32,768 tokens x 8 bf16 heads 38 us (0.82 of the copy rate), rotary + append
// of 16,381 tokens of 32/8 heads 71 us (0.79), reading 64 ragged contexts back 87 us (0.84).
#include "fp8.cuh"

namespace {

template <typename T>
struct alignas(16) Vec {
  static constexpr int E = 16 / sizeof(T);
  T v[E];
};

template <int N>
struct alignas(N * 4) Words {
  uint32_t w[N];
};

__host__ __forceinline__ bool aligned(const void* p, uintptr_t n) {
  return reinterpret_cast<uintptr_t>(p) % n == 0;
}

// Maximum over the LPR lanes of a row.
template <int LPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Block and offset of a slot; `shift` is log2(block_size), or -1 if that is no power of two.
struct Place {
  int64_t block;
  int off;
  __device__ __forceinline__ Place(int64_t slot, int block_size, int shift) {
    block = shift >= 0 ? slot >> shift : slot / block_size;
    off = int(slot - block * block_size);
  }
};

int log2_or_minus_one(int n) {
  for (int s = 0; s < 31; ++s)
    if (n == 1 << s) return s;
  return -1;
}

constexpr int kInFlight = 4;  // rows of a thread at a time

__device__ __forceinline__ void flag(int32_t* error_flag) {
  if (error_flag != nullptr) atomicExch(error_flag, 1);
}

// One lane's E values of a row -> E codes at row + c * E, the scale from the row's first lane; with
// VPL > 1 the lane has E / VPL values of each of VPL parts of the row. Every lane of the warp takes
// part (shuffles); `live` rows are stored. BRANCH: rows of a small scale have code of their own
// (append 37.7 us, 42.8 without; rotary + append 71.3 without, 72.1 with).
template <int E, int LPR, int VPL, bool BRANCH>
__device__ __forceinline__ void store_row_fp8(const float (&x)[E], int c, bool live, uint8_t* row,
                                              float* scale) {
  float m = ts::amax3(x[0], x[1], x[2]);
#pragma unroll
  for (int e = 3; e < E; e += 2) m = ts::amax3(m, x[e], x[e + 1 < E ? e + 1 : e]);
  const float sc = ts::fp8_row_scale(row_max<LPR>(__float_as_uint(m)));
  const ts::Fp8Divide by(sc);
  constexpr int P = E / VPL;
  Words<P / 4> w[VPL];
  if (BRANCH && !by.small()) {
#pragma unroll
    for (int i = 0; i < E / 4; ++i)
      w[i / (P / 4)].w[i % (P / 4)] = by.pack4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < E / 4; ++i)
      w[i / (P / 4)].w[i % (P / 4)] = by.pack4(x[4 * i] * by.up, x[4 * i + 1] * by.up,
                                               x[4 * i + 2] * by.up, x[4 * i + 3] * by.up);
  }
  if (live) {
#pragma unroll
    for (int q = 0; q < VPL; ++q)
      *reinterpret_cast<Words<P / 4>*>(row + (q * LPR + c) * P) = w[q];
    if (c == 0) *scale = sc;
  }
}

// ------------------------------------------------------------------------------ append

struct AppendArgs {
  const void* key;
  const void* value;
  int64_t key_stride, value_stride;  // elements
  uint8_t* key_pool;
  uint8_t* value_pool;
  float* key_scales;
  float* value_scales;
  const int64_t* slots;
  int64_t num_tokens;
  int heads, d, block_size, block_shift, tok_shift;  // tok_shift: log2(2 * heads) or -1
  int64_t num_slots;
  const int32_t* tags;
  int32_t* tag_pool;
  int32_t* error_flag;
};

// Slot of token t, -1 if nothing is written for it.
__device__ __forceinline__ int64_t live_slot(const int64_t* slots, int64_t t, int64_t num_slots) {
  const int64_t s = __ldg(slots + t);
  return s < num_slots ? s : -1;
}

// Tags and the flag of out-of-range slots, once per token.
__device__ __forceinline__ void token_side(const AppendArgs& a, int64_t t) {
  const int64_t s = __ldg(a.slots + t);
  if (s >= a.num_slots) flag(a.error_flag);
  if (s >= 0 && s < a.num_slots && a.tag_pool != nullptr) a.tag_pool[s] = __ldg(a.tags + t);
}

// Rows (token, K|V, head) in order: LPR lanes each with VPL 16-byte vectors, LPR vectors apart (half
// the lanes with two vectors each take half the shuffles and scale arithmetic), ROWS rows a thread.
template <typename T, int LPR, int VPL, int ROWS>
__global__ void __launch_bounds__(256) append_fp8_kernel(const AppendArgs a) {
  ts::allow_dependents();
  constexpr int E = Vec<T>::E, D = LPR * E * VPL, RPC = 256 / LPR;
  const int c = threadIdx.x % LPR;
  const uint32_t per_tok = 2 * a.heads;
  const uint32_t row0 = blockIdx.x * (RPC * ROWS) + threadIdx.x / LPR;
  Vec<T> v[ROWS][VPL];
  uint32_t tok[ROWS], r[ROWS];
  int64_t slot[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    tok[i] = a.tok_shift >= 0 ? (row0 + i * RPC) >> a.tok_shift : (row0 + i * RPC) / per_tok;
    r[i] = row0 + i * RPC - tok[i] * per_tok;
    slot[i] = tok[i] < a.num_tokens ? live_slot(a.slots, tok[i], a.num_slots) : -1;
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const bool is_v = r[i] >= uint32_t(a.heads);
    const T* src = static_cast<const T*>(is_v ? a.value : a.key) +
                   int64_t(tok[i]) * (is_v ? a.value_stride : a.key_stride) +
                   (is_v ? r[i] - a.heads : r[i]) * D + c * E;
#pragma unroll
    for (int q = 0; q < VPL; ++q) {
      if (slot[i] >= 0) {
        v[i][q] = *reinterpret_cast<const Vec<T>*>(src + q * LPR * E);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[i][q].v[e] = ts::from_float<T>(0.f);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const bool is_v = r[i] >= uint32_t(a.heads), live = slot[i] >= 0;
    if (tok[i] < a.num_tokens && r[i] == 0 && c == 0) token_side(a, tok[i]);
    float x[E * VPL];
#pragma unroll
    for (int e = 0; e < E * VPL; ++e) x[e] = ts::to_float(v[i][e / E].v[e % E]);
    const Place at(live ? slot[i] : 0, a.block_size, a.block_shift);
    const uint32_t prow =
        (uint32_t(at.block) * a.heads + (is_v ? r[i] - a.heads : r[i])) * a.block_size + at.off;
    store_row_fp8<E * VPL, LPR, VPL, true>(x, c, live,
                                     (is_v ? a.value_pool : a.key_pool) + uint64_t(prow) * D,
                                     (is_v ? a.value_scales : a.key_scales) + prow);
  }
}

// Any head_dim, stride and alignment: one warp per row.
template <typename T>
__global__ void __launch_bounds__(256) append_fp8_any_kernel(const AppendArgs a) {
  const int lane = threadIdx.x % 32;
  const int per_tok = 2 * a.heads;
  const int64_t rows = a.num_tokens * per_tok;
  for (int64_t row = (int64_t(blockIdx.x) * 256 + threadIdx.x) / 32; row < rows;
       row += int64_t(gridDim.x) * 8) {
    const int64_t t = row / per_tok;
    const int r = int(row - t * per_tok);
    const bool is_v = r >= a.heads;
    const int h = is_v ? r - a.heads : r;
    if (r == 0 && lane == 0) token_side(a, t);
    const int64_t slot = live_slot(a.slots, t, a.num_slots);
    if (slot < 0) continue;
    const T* src = static_cast<const T*>(is_v ? a.value : a.key) +
                   t * (is_v ? a.value_stride : a.key_stride) + int64_t(h) * a.d;
    uint32_t m = 0;
    for (int i = lane; i < a.d; i += 32) m = max(m, ts::abs_bits(ts::to_float(src[i])));
    const float sc = ts::fp8_row_scale(row_max<32>(m));
    const ts::Fp8Divide by(sc);
    const int64_t blk = slot / a.block_size;
    const int64_t prow = (blk * a.heads + h) * a.block_size + slot - blk * a.block_size;
    uint8_t* dst = (is_v ? a.value_pool : a.key_pool) + prow * a.d;
    for (int i = lane; i < a.d; i += 32) dst[i] = by.one(ts::to_float(src[i]));
    if (lane == 0) (is_v ? a.value_scales : a.key_scales)[prow] = sc;
  }
}

// Lanes a row of d elements of `es` bytes splits over, 0 if it does not.
int row_lanes(int d, int es) {
  const int bytes = d * es;
  if (bytes % 16) return 0;
  const int n = bytes / 16;
  return n == 4 || n == 8 || n == 16 || n == 32 ? n : 0;
}

template <typename T>
int launch_append(const AppendArgs& a, cudaStream_t s) {
  const int es = sizeof(T);
  int lpr = row_lanes(a.d, es);
  const int cb = 16 / es;  // code bytes a lane stores
  if (!aligned(a.key, 16) || !aligned(a.value, 16) || (a.key_stride * es) % 16 ||
      (a.value_stride * es) % 16 || !aligned(a.key_pool, cb) || !aligned(a.value_pool, cb))
    lpr = 0;
  const int64_t rows = a.num_tokens * 2 * a.heads;
  // The fast kernel counts the step's and the pool's rows in 32 bits.
  constexpr int64_t kMost = int64_t(4294967295) - 65536;
  if (lpr == 0 || rows >= kMost || a.num_slots >= kMost / a.heads) {
    const int64_t g = (rows + 7) / 8;
    append_fp8_any_kernel<T><<<unsigned(g < 65536 ? g : 65536), 256, 0, s>>>(a);
    return ts::launch_status("reshape_and_cache_fp8");
  }
  constexpr int kRows = 1;  // two as fast for many rows and slower for few, four slower
  const int lanes = lpr == 4 ? 4 : lpr / 2;
  const int64_t per_cta = 256 / lanes * kRows, grid = (rows + per_cta - 1) / per_cta;
  switch (lpr) {
    case 4: append_fp8_kernel<T, 4, 1, kRows><<<unsigned(grid), 256, 0, s>>>(a); break;
    case 8: append_fp8_kernel<T, 4, 2, kRows><<<unsigned(grid), 256, 0, s>>>(a); break;
    case 16: append_fp8_kernel<T, 8, 2, kRows><<<unsigned(grid), 256, 0, s>>>(a); break;
    default: append_fp8_kernel<T, 16, 2, kRows><<<unsigned(grid), 256, 0, s>>>(a); break;
  }
  return ts::launch_status("reshape_and_cache_fp8");
}

// ------------------------------------------------------------------------------ rotary + append

struct RotaryArgs {
  const void* qkv;
  int64_t qkv_stride;  // elements
  void* q_out;
  void* key_pool;
  void* value_pool;
  float* key_scales;  // nullptr: the pools hold T
  float* value_scales;
  const int64_t* slots;
  const int64_t* positions;
  const float* inv_freq;
  int hq, hkv, d, rd, block_size, block_shift;
  float mscale;
  int64_t num_slots;
  int32_t* error_flag;
};

// cos and sin of pos * f, times mscale. The turn count pos * f / 2 pi is taken in 64 bits, where
// its fraction is exact to 2^-30 even at position 2^22 (a 32-bit product is off by 2^-24 of an
// angle that reaches 10^5 radians); only the fraction is rounded to 32 bits.
__device__ __forceinline__ float2 cos_sin(int64_t pos, float f, float mscale) {
  const double turns = double(pos) * (double(f) * 0.15915494309189535);
  float s, c;
  sincospif(2.f * float(turns - rint(turns)), &s, &c);
  return make_float2(c * mscale, s * mscale);
}

// One CTA per token. A thread always has the same dims (c) of its rows: the first kInFlight rows
// are on their way while the token's cos and sin are computed (in shared memory, once), which it
// then keeps in registers for all its rows. Requires rd % (2 E) == 0 (half layout: a lane's partner
// values sit in one other lane), rows of LPR * 16 bytes, 16-byte aligned.
//
// 64 threads keep a token's set-up small beside its rows when there are many tokens (8,192 tokens of
// 32/8 heads: 39 us, 44 with 128); with few tokens 128 shorten it (256 tokens: 4.0 us, 5.2 with 64). The
// two cross between 1,024 and 1,536 tokens with 32/8, 64/8 and 16/16 heads, near 300 with 8/1, where
// the difference up to 1,024 tokens is 0.7 us.
constexpr int kRotaryThreads = 128, kRotaryThreadsMany = 64, kRotaryManyTokens = 1024;
template <typename T, int LPR, bool INTERLEAVED, bool FP8>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryArgs a) {
  ts::allow_dependents();
  constexpr int E = Vec<T>::E, D = LPR * E;
  const int RPC = blockDim.x / LPR;
  const int64_t t = blockIdx.x;
  const int c = threadIdx.x % LPR, rows = a.hq + 2 * a.hkv, half = a.rd / 2;
  const T* in = static_cast<const T*>(a.qkv) + t * a.qkv_stride + c * E;
  const int64_t pos = __ldg(a.positions + t), slot_raw = __ldg(a.slots + t);
  const int64_t slot = slot_raw < a.num_slots ? slot_raw : -1;
  Vec<T> v[kInFlight];
  auto live_row = [&](int r) { return r < rows && (r < a.hq || slot >= 0); };
  auto load = [&](int r0) {
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int r = r0 + i * RPC;
      if (r < rows) {
        v[i] = *reinterpret_cast<const Vec<T>*>(in + r * D);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[i].v[e] = ts::from_float<T>(0.f);
      }
    }
  };
  load(threadIdx.x / LPR);
  __shared__ alignas(16) float2 cs[D / 2];
  for (int i = threadIdx.x; i < half; i += blockDim.x)
    cs[i] = cos_sin(pos, __ldg(a.inv_freq + i), a.mscale);
  if (slot_raw >= a.num_slots && threadIdx.x == 0) flag(a.error_flag);
  const Place at(slot >= 0 ? slot : 0, a.block_size, a.block_shift);
  __syncthreads();
  const int i0 = c * E;          // this lane's first dimension
  const int hl = half / E;       // half layout: lanes with the first halves of the pairs
  const bool first = c < hl, turned = i0 < a.rd;
  // cos and sin for each of the lane's dims; with the sign of the partner's product.
  uint64_t wc[E / 2], ws[E / 2];
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    float2 u = make_float2(1.f, 0.f), v2 = u;
    if (turned && INTERLEAVED) {
      u = v2 = cs[(i0 + e) / 2];
      u.y = -u.y;
    } else if (turned) {
      const int j = (first ? i0 : i0 - half) + e;
      u = cs[j];
      v2 = cs[j + 1];
      if (first) u.y = -u.y, v2.y = -v2.y;
    }
    wc[e / 2] = ts::two(u.x, v2.x);
    ws[e / 2] = ts::two(u.y, v2.y);
  }
  const int partner = ((threadIdx.x % 32) + (first ? hl : (turned ? -hl : 0))) & 31;
  // Where the token's rows go: head h at base + h * step.
  T* const q_row = static_cast<T*>(a.q_out) + t * a.hq * D + c * E;
  const int64_t first_row = at.block * a.hkv * a.block_size + at.off;
#pragma unroll 1
  for (int r0 = threadIdx.x / LPR; r0 - int(threadIdx.x) / LPR < rows; r0 += kInFlight * RPC) {
    if (r0 >= kInFlight * RPC) load(r0);
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      if (r0 - int(threadIdx.x) / LPR + i * RPC >= rows) break;  // for the whole CTA
      const int r = r0 + i * RPC;
      const bool is_q = r < a.hq, is_v = r >= a.hq + a.hkv, live = live_row(r);
      Vec<T> o = v[i];
      if (!INTERLEAVED) {
        const uint32_t* raw = reinterpret_cast<const uint32_t*>(&v[i]);
        uint32_t* oraw = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
        for (int k = 0; k < 4; ++k) oraw[k] = __shfl_sync(0xffffffffu, raw[k], partner);
      }
      float x[E];
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float x0 = ts::to_float(v[i].v[e]), x1 = ts::to_float(v[i].v[e + 1]);
        const float y0 = ts::to_float(o.v[INTERLEAVED ? e + 1 : e]);
        const float y1 = ts::to_float(o.v[INTERLEAVED ? e : e + 1]);
        const float2 z = ts::halves(
            ts::fma2(ts::two(y0, y1), ws[e / 2], ts::mul2(ts::two(x0, x1), wc[e / 2])));
        x[e] = is_v || !turned ? x0 : z.x;
        x[e + 1] = is_v || !turned ? x1 : z.y;
      }
      const int h = is_q ? r : (is_v ? r - a.hq - a.hkv : r - a.hq);
      const int64_t prow = first_row + h * a.block_size;
      if (FP8) {
        // Rows of q only in the CTA's step: nothing to quantise.
        if (r0 - int(threadIdx.x) / LPR + (i + 1) * RPC > a.hq)
          store_row_fp8<E, LPR, 1, false>(x, c, live && !is_q,
                                static_cast<uint8_t*>(is_v ? a.value_pool : a.key_pool) + prow * D,
                                (is_v ? a.value_scales : a.key_scales) + prow);
      }
      if (live && (is_q || !FP8)) {
        T* dst = is_q ? q_row + r * D
                      : static_cast<T*>(is_v ? a.value_pool : a.key_pool) + prow * D + c * E;
        Vec<T> y;
#pragma unroll
        for (int e = 0; e < E; ++e) y.v[e] = ts::from_float<T>(x[e]);
        *reinterpret_cast<Vec<T>*>(dst) = y;
      }
    }
  }
}

// Any sizes and alignment: one warp per head row, the angles computed where they are used.
template <typename T>
__global__ void __launch_bounds__(256) rotary_any_kernel(const RotaryArgs a, int64_t num_tokens,
                                                         bool interleaved) {
  const int lane = threadIdx.x % 32;
  const int rows_per_tok = a.hq + 2 * a.hkv;
  const int64_t rows = num_tokens * rows_per_tok;
  const int half = a.rd / 2;
  for (int64_t row = (int64_t(blockIdx.x) * 256 + threadIdx.x) / 32; row < rows;
       row += int64_t(gridDim.x) * 8) {
    const int64_t t = row / rows_per_tok;
    const int r = int(row - t * rows_per_tok);
    const bool is_q = r < a.hq, is_v = r >= a.hq + a.hkv;
    const int h = is_q ? r : (is_v ? r - a.hq - a.hkv : r - a.hq);
    const int64_t slot_raw = __ldg(a.slots + t), pos = __ldg(a.positions + t);
    if (slot_raw >= a.num_slots && r == 0 && lane == 0) flag(a.error_flag);
    const bool live = slot_raw >= 0 && slot_raw < a.num_slots;
    if (!is_q && !live) continue;
    const T* src = static_cast<const T*>(a.qkv) + t * a.qkv_stride + int64_t(r) * a.d;
    auto value = [&](int i) -> float {
      const float x = ts::to_float(src[i]);
      if (is_v || i >= a.rd) return x;
      const int pair = interleaved ? i / 2 : i % half;
      const bool first = interleaved ? i % 2 == 0 : i < half;
      const int other = interleaved ? i ^ 1 : (first ? i + half : i - half);
      const float2 w = cos_sin(pos, __ldg(a.inv_freq + pair), a.mscale);
      const float y = ts::to_float(src[other]);
      return first ? x * w.x - y * w.y : x * w.x + y * w.y;
    };
    const int64_t blk = live ? slot_raw / a.block_size : 0;
    const int64_t prow = (blk * a.hkv + h) * a.block_size + (live ? slot_raw - blk * a.block_size : 0);
    if (is_q || a.key_scales == nullptr) {
      T* dst = is_q ? static_cast<T*>(a.q_out) + (t * a.hq + h) * a.d
                    : static_cast<T*>(is_v ? a.value_pool : a.key_pool) + prow * a.d;
      for (int i = lane; i < a.d; i += 32) dst[i] = ts::from_float<T>(value(i));
      continue;
    }
    uint32_t m = 0;
    for (int i = lane; i < a.d; i += 32) m = max(m, ts::abs_bits(value(i)));
    const float sc = ts::fp8_row_scale(row_max<32>(m));
    const ts::Fp8Divide by(sc);
    uint8_t* dst = static_cast<uint8_t*>(is_v ? a.value_pool : a.key_pool) + prow * a.d;
    for (int i = lane; i < a.d; i += 32) dst[i] = by.one(value(i));
    if (lane == 0) (is_v ? a.value_scales : a.key_scales)[prow] = sc;
  }
}

template <typename T, int LPR>
void launch_rotary_vec(const RotaryArgs& a, int64_t tokens, bool interleaved, cudaStream_t s) {
  const unsigned g = unsigned(tokens);
  const int threads = tokens < kRotaryManyTokens ? kRotaryThreads : kRotaryThreadsMany;
  const bool fp8 = a.key_scales != nullptr;
  if (interleaved)
    fp8 ? rotary_kernel<T, LPR, true, true><<<g, threads, 0, s>>>(a)
        : rotary_kernel<T, LPR, true, false><<<g, threads, 0, s>>>(a);
  else
    fp8 ? rotary_kernel<T, LPR, false, true><<<g, threads, 0, s>>>(a)
        : rotary_kernel<T, LPR, false, false><<<g, threads, 0, s>>>(a);
}

template <typename T>
int launch_rotary(const RotaryArgs& a, int64_t tokens, bool interleaved, cudaStream_t s) {
  constexpr int es = sizeof(T), E = Vec<T>::E;
  int lpr = row_lanes(a.d, es);
  const uintptr_t pool_align = a.key_scales != nullptr ? E : 16;
  if (a.rd % (2 * E) || !aligned(a.qkv, 16) || (a.qkv_stride * es) % 16 || !aligned(a.q_out, 16) ||
      !aligned(a.key_pool, pool_align) || !aligned(a.value_pool, pool_align))
    lpr = 0;
  switch (lpr) {
    case 4: launch_rotary_vec<T, 4>(a, tokens, interleaved, s); break;
    case 8: launch_rotary_vec<T, 8>(a, tokens, interleaved, s); break;
    case 16: launch_rotary_vec<T, 16>(a, tokens, interleaved, s); break;
    case 32: launch_rotary_vec<T, 32>(a, tokens, interleaved, s); break;
    default: {
      const int64_t g = (tokens * (a.hq + 2 * a.hkv) + 7) / 8;
      rotary_any_kernel<T><<<unsigned(g < 65536 ? g : 65536), 256, 0, s>>>(a, tokens, interleaved);
    }
  }
  return ts::launch_status("rotary_and_cache");
}

// ------------------------------------------------------------------------------ read back

struct ReadArgs {
  void* key_out;
  void* value_out;
  const uint8_t* key_pool;
  const uint8_t* value_pool;
  const float* key_scales;
  const float* value_scales;
  const int32_t* tables;
  const int32_t* loc;
  int num_seqs, max_blocks, heads, d, block_size, block_shift;
  int64_t num_blocks, num_tokens;
  int32_t* error_flag;
};

constexpr int kReadTokens = 16;  // tokens per CTA

// Warp 0 of a CTA finds the pool rows (of head 0) of output rows t0 .. t0 + kReadTokens - 1, one a
// lane. -1: the row belongs to no sequence (left as it was); -2: its block is not in the pool, or
// past the table (zeros). The sequence of t0 is narrowed down 32 ways a step; a later row moves on
// from there.
__device__ __forceinline__ void find_rows(const ReadArgs& a, int64_t t0, int64_t* src) {
  const int lane = threadIdx.x;
  int lo = 0, hi = a.num_seqs;  // loc[lo] <= t0 < loc[hi], or t0 is outside
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int probe = min(hi, lo + (lane + 1) * step);
    // Ascending: the probes at or below t0 are the first ones.
    const int below = __popc(__ballot_sync(0xffffffffu, probe < hi && __ldg(a.loc + probe) <= t0));
    hi = min(hi, lo + (below + 1) * step);
    lo += below * step;
  }
  const int64_t t = t0 + lane;
  if (lane >= kReadTokens) return;
  int64_t s = -1;
  if (t < a.num_tokens && t >= __ldg(a.loc) && t < __ldg(a.loc + a.num_seqs)) {
    while (__ldg(a.loc + lo + 1) <= t) ++lo;  // ends: t < loc[num_seqs]
    const Place at(t - __ldg(a.loc + lo), a.block_size, a.block_shift);
    s = -2;
    if (at.block >= 0 && at.block < a.max_blocks) {  // negative: token_start_loc not ascending
      const int64_t blk = __ldg(a.tables + int64_t(lo) * a.max_blocks + at.block);
      if (blk >= 0 && blk < a.num_blocks) s = blk * a.heads * a.block_size + at.off;
    }
  }
  if (s == -2) flag(a.error_flag);
  src[lane] = s;
}

// CTA = kReadTokens output tokens: their pool rows are looked up once, then every thread turns
// 16 codes of a (token, K|V, head) row into 16 values, kInFlight rows at a time. LPR = D / 16.
template <typename T, int LPR>
__global__ void __launch_bounds__(256) read_fp8_kernel(const ReadArgs a) {
  constexpr int D = LPR * 16, RPC = 256 / LPR, E = Vec<T>::E;
  __shared__ int64_t src[kReadTokens];
  const int64_t t0 = int64_t(blockIdx.x) * kReadTokens;
  if (threadIdx.x < 32) find_rows(a, t0, src);
  __syncthreads();
  const int c = threadIdx.x % LPR;
  const int per_tok = 2 * a.heads, rows = kReadTokens * per_tok;
  for (int r0 = threadIdx.x / LPR; r0 < rows; r0 += kInFlight * RPC) {
    uint4 code[kInFlight];
    float sc[kInFlight];
    int tok[kInFlight], k[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int r = r0 + i * RPC;
      tok[i] = r / per_tok;
      k[i] = r - tok[i] * per_tok;
      const int64_t s = r < rows ? src[tok[i]] : -1;
      code[i] = make_uint4(0, 0, 0, 0);
      sc[i] = 0.f;
      if (s >= 0) {
        const bool is_v = k[i] >= a.heads;
        const int64_t prow = s + int64_t(is_v ? k[i] - a.heads : k[i]) * a.block_size;
        code[i] = __ldg(reinterpret_cast<const uint4*>((is_v ? a.value_pool : a.key_pool) + prow * D) + c);
        sc[i] = __ldg((is_v ? a.value_scales : a.key_scales) + prow);
      }
      if (s == -1) tok[i] = -1;
    }
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      if (tok[i] < 0) continue;
      const bool is_v = k[i] >= a.heads;
      T* dst = static_cast<T*>(is_v ? a.value_out : a.key_out) +
               ((t0 + tok[i]) * a.heads + (is_v ? k[i] - a.heads : k[i])) * D + c * 16;
      const uint32_t word[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
      float f[16];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float2 p = __half22float2(ts::fp8_half2(word[q / 2] >> (16 * (q & 1))));
        f[2 * q] = p.x * sc[i];
        f[2 * q + 1] = p.y * sc[i];
      }
#pragma unroll
      for (int q = 0; q < 16 / E; ++q) {
        Vec<T> y;
#pragma unroll
        for (int e = 0; e < E; ++e) y.v[e] = ts::from_float<T>(f[q * E + e]);
        *reinterpret_cast<Vec<T>*>(dst + q * E) = y;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) read_fp8_any_kernel(const ReadArgs a) {
  __shared__ int64_t src[kReadTokens];
  const int64_t t0 = int64_t(blockIdx.x) * kReadTokens;
  if (threadIdx.x < 32) find_rows(a, t0, src);
  __syncthreads();
  const int64_t per_tok = 2 * int64_t(a.heads) * a.d;
  for (int64_t e = threadIdx.x; e < kReadTokens * per_tok; e += 256) {
    const int tl = int(e / per_tok);
    int64_t k = e - tl * per_tok;
    const bool is_v = k >= int64_t(a.heads) * a.d;
    if (is_v) k -= int64_t(a.heads) * a.d;
    const int h = int(k / a.d), i = int(k - int64_t(h) * a.d);
    const int64_t s = src[tl];
    if (s == -1) continue;
    float x = 0.f;
    if (s >= 0) {
      const int64_t prow = s + int64_t(h) * a.block_size;
      x = ts::fp8_float((is_v ? a.value_pool : a.key_pool)[prow * a.d + i]) *
          (is_v ? a.value_scales : a.key_scales)[prow];
    }
    static_cast<T*>(is_v ? a.value_out : a.key_out)[((t0 + tl) * a.heads + h) * a.d + i] =
        ts::from_float<T>(x);
  }
}

template <typename T>
int launch_read(const ReadArgs& a, cudaStream_t s) {
  const unsigned g = unsigned((a.num_tokens + kReadTokens - 1) / kReadTokens);
  const bool vec = aligned(a.key_out, 16) && aligned(a.value_out, 16) && aligned(a.key_pool, 16) &&
                   aligned(a.value_pool, 16);
  if (vec && a.d == 64)
    read_fp8_kernel<T, 4><<<g, 256, 0, s>>>(a);
  else if (vec && a.d == 128)
    read_fp8_kernel<T, 8><<<g, 256, 0, s>>>(a);
  else if (vec && a.d == 256)
    read_fp8_kernel<T, 16><<<g, 256, 0, s>>>(a);
  else
    read_fp8_any_kernel<T><<<g, 256, 0, s>>>(a);
  return ts::launch_status("read_cache_fp8");
}

}  // namespace

extern "C" int ts_reshape_and_cache_fp8(const void* key, const void* value,
                                        int64_t key_token_stride, int64_t value_token_stride,
                                        void* key_pool, void* value_pool, float* key_scales,
                                        float* value_scales, const int64_t* slot_mapping,
                                        int64_t num_tokens, int32_t num_kv_heads, int32_t head_dim,
                                        int32_t block_size, int64_t num_blocks, int32_t dtype,
                                        const int32_t* token_tags, int32_t* tag_pool,
                                        int32_t* error_flag, void* stream) {
  if (ts::dtype_size(dtype) == 0)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT, "reshape_and_cache_fp8: bad dtype %d", dtype);
  if (num_tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_blocks <= 0)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT,
                         "reshape_and_cache_fp8: bad sizes (tokens %lld, heads %d, head_dim %d, "
                         "block_size %d, blocks %lld)",
                         (long long)num_tokens, num_kv_heads, head_dim, block_size,
                         (long long)num_blocks);
  if (num_tokens == 0) return ts::ok();
  if (!key || !value || !key_pool || !value_pool || !key_scales || !value_scales || !slot_mapping)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT, "reshape_and_cache_fp8: null pointer");
  if ((token_tags == nullptr) != (tag_pool == nullptr))
    return ts::set_error(TS_ERR_INVALID_ARGUMENT,
                         "reshape_and_cache_fp8: token_tags and tag_pool go together");
  if (key_token_stride < int64_t(num_kv_heads) * head_dim ||
      value_token_stride < int64_t(num_kv_heads) * head_dim)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT,
                         "reshape_and_cache_fp8: token stride smaller than heads * head_dim");
  if (!aligned(key, ts::dtype_size(dtype)) || !aligned(value, ts::dtype_size(dtype)) ||
      !aligned(key_scales, 4) || !aligned(value_scales, 4))
    return ts::set_error(TS_ERR_MISALIGNED,
                         "reshape_and_cache_fp8: pointers not element-aligned");
  const AppendArgs a{key, value, key_token_stride, value_token_stride,
                     static_cast<uint8_t*>(key_pool), static_cast<uint8_t*>(value_pool),
                     key_scales, value_scales, slot_mapping, num_tokens, num_kv_heads, head_dim,
                     block_size, log2_or_minus_one(block_size),
                     log2_or_minus_one(2 * num_kv_heads), num_blocks * block_size, token_tags,
                     tag_pool, error_flag};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TS_FLOAT32) return launch_append<float>(a, s);
  if (dtype == TS_FLOAT16) return launch_append<__half>(a, s);
  return launch_append<__nv_bfloat16>(a, s);
}

extern "C" int ts_rotary_and_cache(const void* qkv, int64_t qkv_token_stride, void* q_out,
                                   void* key_pool, void* value_pool, float* key_scales,
                                   float* value_scales, const int64_t* slot_mapping,
                                   const int64_t* positions, const float* inv_freq,
                                   int64_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads,
                                   int32_t head_dim, int32_t rotary_dim, int32_t interleaved,
                                   float attention_scaling, int32_t block_size,
                                   int64_t num_blocks, int32_t dtype, int32_t* error_flag,
                                   void* stream) {
  if (ts::dtype_size(dtype) == 0)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT, "rotary_and_cache: bad dtype %d", dtype);
  if (num_tokens < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      block_size <= 0 || num_blocks <= 0)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT,
                         "rotary_and_cache: bad sizes (tokens %lld, heads %d/%d, head_dim %d, "
                         "block_size %d, blocks %lld)",
                         (long long)num_tokens, num_q_heads, num_kv_heads, head_dim, block_size,
                         (long long)num_blocks);
  if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 2)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT,
                         "rotary_and_cache: rotary_dim %d must be even and in 2..head_dim %d",
                         rotary_dim, head_dim);
  if (qkv_token_stride < (int64_t(num_q_heads) + 2 * int64_t(num_kv_heads)) * head_dim)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT, "rotary_and_cache: token stride too small");
  if ((key_scales == nullptr) != (value_scales == nullptr))
    return ts::set_error(TS_ERR_INVALID_ARGUMENT,
                         "rotary_and_cache: key_scales and value_scales go together");
  if (num_tokens == 0) return ts::ok();
  if (num_tokens > 2147483647)
    return ts::set_error(TS_ERR_UNSUPPORTED, "rotary_and_cache: too many tokens");
  if (!qkv || !q_out || !key_pool || !value_pool || !slot_mapping || !positions || !inv_freq)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT, "rotary_and_cache: null pointer");
  const uintptr_t es = ts::dtype_size(dtype), ps = key_scales != nullptr ? 1 : es;
  if (!aligned(qkv, es) || !aligned(q_out, es) || !aligned(key_pool, ps) ||
      !aligned(value_pool, ps) || !aligned(key_scales, 4) || !aligned(value_scales, 4))
    return ts::set_error(TS_ERR_MISALIGNED, "rotary_and_cache: pointers not element-aligned");
  const RotaryArgs a{qkv, qkv_token_stride, q_out, key_pool, value_pool, key_scales, value_scales,
                     slot_mapping, positions, inv_freq, num_q_heads, num_kv_heads, head_dim,
                     rotary_dim, block_size, log2_or_minus_one(block_size), attention_scaling,
                     num_blocks * block_size, error_flag};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TS_FLOAT32) return launch_rotary<float>(a, num_tokens, interleaved != 0, s);
  if (dtype == TS_FLOAT16) return launch_rotary<__half>(a, num_tokens, interleaved != 0, s);
  return launch_rotary<__nv_bfloat16>(a, num_tokens, interleaved != 0, s);
}

extern "C" int ts_read_cache_fp8(void* key_out, void* value_out, const void* key_pool,
                                 const void* value_pool, const float* key_scales,
                                 const float* value_scales, const int32_t* block_tables,
                                 int32_t max_blocks_per_seq, const int32_t* token_start_loc,
                                 int32_t num_seqs, int64_t num_tokens, int32_t num_kv_heads,
                                 int32_t head_dim, int32_t block_size, int64_t num_blocks,
                                 int32_t dtype, int32_t* error_flag, void* stream) {
  if (ts::dtype_size(dtype) == 0)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT, "read_cache_fp8: bad dtype %d", dtype);
  if (num_seqs < 0 || num_tokens < 0 || max_blocks_per_seq <= 0 || num_kv_heads <= 0 ||
      head_dim <= 0 || block_size <= 0 || num_blocks <= 0)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT,
                         "read_cache_fp8: bad sizes (seqs %d, tokens %lld, heads %d, head_dim %d, "
                         "block_size %d, blocks %lld, max_blocks %d)",
                         num_seqs, (long long)num_tokens, num_kv_heads, head_dim, block_size,
                         (long long)num_blocks, max_blocks_per_seq);
  if (num_seqs == 0 || num_tokens == 0) return ts::ok();
  if (num_tokens > 2147483647)
    return ts::set_error(TS_ERR_UNSUPPORTED, "read_cache_fp8: too many tokens");
  if (!key_out || !value_out || !key_pool || !value_pool || !key_scales || !value_scales ||
      !block_tables || !token_start_loc)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT, "read_cache_fp8: null pointer");
  const uintptr_t es = ts::dtype_size(dtype);
  if (!aligned(key_out, es) || !aligned(value_out, es) || !aligned(key_scales, 4) ||
      !aligned(value_scales, 4))
    return ts::set_error(TS_ERR_MISALIGNED, "read_cache_fp8: pointers not element-aligned");
  const ReadArgs a{key_out, value_out, static_cast<const uint8_t*>(key_pool),
                   static_cast<const uint8_t*>(value_pool), key_scales, value_scales, block_tables,
                   token_start_loc, num_seqs, max_blocks_per_seq, num_kv_heads, head_dim,
                   block_size, log2_or_minus_one(block_size), num_blocks, num_tokens, error_flag};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TS_FLOAT32) return launch_read<float>(a, s);
  if (dtype == TS_FLOAT16) return launch_read<__half>(a, s);
  return launch_read<__nv_bfloat16>(a, s);
}
