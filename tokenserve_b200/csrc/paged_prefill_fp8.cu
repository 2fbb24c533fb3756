// Chunked-prefill attention (causal) over the 8-bit paged cache (fp8.cuh).
//
// Query row j of a sequence whose step ends at context_lens[s] sits at position
// context_lens[s] - q_len + j and sees positions 0..that one; out = softmax(q k^T scale) v.
//
// bf16/fp16 queries, head_dim 64 or 128, block 16: tcgen05 kernel. It is bound by the tensor cores
// and by the exponentials (one per score), so the cache's 8 bits must cost neither of them:
//   * CTA = (sequence, KV head, pair of query tiles); a tile's 128 rows are 128/G tokens x the G
//     query heads of the KV head, so a converted K/V tile serves 256 rows.
//   * warp 12 (scout) runs up to four spans of 128 tokens ahead: block table, the span's scales and
//     references, left in shared memory.
//   * warps 8-11, 14, 15 (converters) take the blocks of 64-token tiles (4 of K, 4 of V) in turn:
//     codes from global memory two blocks ahead into registers, as fp16 (exact) into the swizzled
//     layout the MMAs read.
//   * warps 0-3 / 4-7 (softmax, one warpgroup per query tile, thread = row): q's row is scaled by a
//     power of two into fp16's range and written to shared memory; then per tile, 32 columns at a
//     time: s = S times K's scale, u = 2^(s + n - mt), P = u times V's scale over 2^n, rounded to
//     fp16 (11 bits), back to TMEM over S. 2^n is the largest V scale of the 32 tokens, mt the maximum
//     of s + log2(V's scale) over the row's first tile, kept while 32 columns' u add up to 2^14 at
//     most, so the exponentials wait for no maximum; a warp with a row past that takes the columns,
//     and all before them, to the new maximum. The softmax's sum, of 2^(s - m) with a maximum m of s, is that
//     of u times one factor per 32 columns, in fp32. The output is O 2^(mt - m) / sum. So a key of any
//     magnitude takes no bits from the others unless its weight does: P is off by 2^-11 of itself,
//     or by 2^-25 of the largest P below 2^-14 of that. Columns no row of a warp sees are skipped.
//     Everything is in loops over few columns: unrolled over a whole row, the roles' code outgrew
//     the instruction caches (a quarter of the stalls).
//   * warp 13: tcgen05.mma, S_x = Q_x K^T and O_x += P_x V, in the order PV_A(j), QK_A(j+2),
//     PV_B(j), QK_B(j+2): each query tile has two S buffers of 64 columns, so its softmax finds the
//     next tile's scores ready and waits for no MMA (with one buffer of 128 columns a tile's
//     softmax, PV and QK took turns: 5,000 clocks per 128 tokens).
// 64 sequences of 257-512 new tokens over 900-1,600 cached ones, 32/8 heads of 128: 844 us, 680 TFLOP/s
// (0.42 of cuBLAS bf16), fp16 841 us: what binds is the way of a tile's scores through softmax and
// MMAs and back. Codes times scales in fp16 tiles (one rounding of K and V each) took 841 us and left
// fp16 outputs 4.6e-4 off 64 bits instead of 2.9e-4 (2.1e-4 is their own rounding).
// A page outside the pool is skipped (its columns are masked). A V row with a NaN scale is stored
// as zeros and rows that see it become NaN, so rows before it in the chunk stay clean. V's rows past
// the last visible key are stored as zeros: their slots may hold anything. Other shapes and fp32
// queries run on CUDA cores (attention_portable.cu).
#include <cstddef>

#include "fp8.cuh"
#include "tcgen05.cuh"

namespace ts {
int paged_attention_portable(void* out, const void* query, int64_t q_stride, const void* kp,
                             const void* vp, const int32_t* bt, int max_blocks,
                             const int32_t* qsl, const int32_t* cl, int num_seqs, int num_rows,
                             int hq, int hkv, int hd, int bs, int64_t nb, float scale, int dtype,
                             cudaStream_t s, const float* k_scales, const float* v_scales);
}

namespace {

constexpr int kRows = 128;    // query rows per tile (M)
constexpr int kKvTile = 64;   // KV tokens per tile (N of QK, K of PV)
constexpr int kSpan = 128;    // KV tokens the scout describes at a time
constexpr int kBlock = 16;    // tokens per KV block
constexpr int kQHalf = kRows * 128;     // bytes of 64 fp16 columns of a query tile
constexpr int kKvHalf = kKvTile * 128;  // and of a KV tile
constexpr int kQTiles = 2;
constexpr int kStages = 4;  // K ring, and V ring
constexpr int kTilesPerSpan = kSpan / kKvTile;
// Span descriptions. The scout writes span t once the converters are done with t - kAhead, when
// the MMAs, and so the softmaxes, are done with kStages tiles before that.
constexpr int kInfos = 8, kAhead = 4;
static_assert(kAhead + kStages / kTilesPerSpan < kInfos, "a description outlives its readers");
constexpr int kConverters = 6;  // converter warps
constexpr int kUnits = 2 * kKvTile / kBlock;  // blocks of a tile, K then V
constexpr int kThreads = 512;
constexpr int kMaxTries = 1 << 22, kMaxNaps = 1 << 22;  // of a bounded wait
constexpr float kLog2e = 1.4426950408889634f;
// A stale maximum is kept while 32 columns' u add up to 2^14 at most: P, below 2 u, stays below fp16's
// 2^16, and weights near the true maximum, at least 1, are well inside its normal range.
constexpr float kMostSumU = 0x1p14f;
// S_A [0,128) and S_B [128,256), two buffers each, O_A [256,384), O_B [384,512).
constexpr uint32_t kTmemCols = 512;
// A group's n stays within this of the context's largest so far: u is then above fp32's 2^-126
// wherever 2^(s - m) is above 2^-64. (V rows below 2^-60 of the largest scale so far may lose bits.)
constexpr int kRefSpread = 60;
// log2(V's scale / 2^n) counts as this at least in mt, so that rows of zeros leave u, up to 2^100 then,
// and its sums finite.
constexpr float kLeastLog = -100.f;
constexpr float kMostSum = 0x1p60f;  // of a group's 2^(s - m), before m has to move

struct Args {
  void* out;
  const void* query;
  int64_t q_stride;
  const uint8_t* key_pool;
  const uint8_t* value_pool;
  const float* key_scales;
  const float* value_scales;
  const int32_t* block_tables;
  const int32_t* qsl;
  const int32_t* context_lens;
  int max_blocks, num_q_heads, num_kv_heads, group;
  int num_tokens;  // query rows: none past them is read or written
  int tq;       // query tokens per tile
  int q_tiles;  // query tiles per CTA, 1 or 2
  int64_t num_blocks;
  float scale_log2;
};

// A span as the scout leaves it: log2 of V's reference, n, for each 32 rows; the columns to mask (page
// outside the pool) or to spoil (V row NaN), if any; the blocks (negative: none); K's scale of each
// row and V's over 2^n, 0 for rows whose codes are not used (past the last key, or NaN).
struct alignas(16) TileInfo {
  float log_v[4];
  uint32_t skip[4], spoil[4];
  int block[kSpan / kBlock];
  float scale[2][kSpan];
  uint32_t any, dropped;  // dropped: V has rows that are not used
};
static_assert(offsetof(TileInfo, scale) % 16 == 0 && sizeof(TileInfo) % 16 == 0,
              "vector accesses of a description");

struct Shared {
  uint64_t q_full, k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[kQTiles][2], p_full[kQTiles][2], pv_done[kQTiles], o_full[kQTiles], drain;
  uint64_t info_full[kInfos], converted[kAhead];
  TileInfo info[kInfos];
  uint32_t tmem;
};

template <int D>
struct Geo {
  static constexpr int kQBytes = kRows * D * 2, kKvBytes = kKvTile * D * 2;
  static constexpr int kTiles = kQTiles * kQBytes + 2 * kStages * kKvBytes;
  static constexpr int kSmemBytes = kTiles + int(sizeof(Shared)) + 1024;
};

// Bounded wait (a try sleeps for some time, so the tries last about a second), false when it gives up:
// the waits of the roles that depend on this one give up in turn, and the rows become NaN. A loop of
// few instructions: there are many waits, and all roles share the caches.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t phase) {
  uint32_t ok;
  // Four tries a turn of the loop: two instructions a try instead of six.
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, %3;\n"
      "TRY:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "sub.u32 n, n, 1;\n\t"
      "setp.ne.u32 q, n, 0;\n\t"
      "@q bra TRY;\n"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(ts::smem_u32(bar)), "r"(phase), "n"(kMaxTries / 4)
      : "memory");
  return ok != 0;
}
// For the warps that run ahead: naps between tries leave the issue slots to the others.
__device__ __forceinline__ bool wait_ahead(uint64_t* bar, uint32_t phase) {
  bool ok = ts::mbar_try_wait(bar, phase);
#pragma unroll 1
  for (int i = 0; !ok && i < kMaxNaps; ++i) {
    __nanosleep(100);
    ok = ts::mbar_try_wait(bar, phase);
  }
  return __all_sync(0xffffffffu, ok);
}
// The same for a whole warp, with one answer.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t phase) {
  return __all_sync(0xffffffffu, wait_bar(bar, phase));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Bits of the largest finite value of four scales; scales are not negative and order like their bits.
__device__ __forceinline__ uint32_t top_bits(const float (&sc)[4]) {
  auto fin = [](float v) { return isfinite(v) ? v : 0.f; };
  const float m = fmaxf(fmaxf(fin(sc[0]), fin(sc[1])), fmaxf(fin(sc[2]), fin(sc[3])));
  return __float_as_uint(fmaxf(m, 0.f));
}

// The scout warp: describes the spans of a KV head's keys, n_kv of them visible. Lane l looks after
// tokens 4 l .. 4 l + 3 of each span, in block l / 4; their scales are loaded a span ahead.
struct Scout {
  const Args& a;
  const int32_t* table;
  int n_kv, lane;
  int64_t stride, mine;  // scales of a block over all heads; this lane's place among them
  int phys;              // this lane's block of the next span (-1 none, -2 not in the pool)
  float4 ks, vs;

  __device__ __forceinline__ Scout(const Args& args, int seq, int h, int keys, int l)
      : a(args), table(args.block_tables + int64_t(seq) * args.max_blocks), n_kv(keys), lane(l),
        stride(int64_t(args.num_kv_heads) * kBlock), mine(int64_t(h) * kBlock + l % 4 * 4) {}

  __device__ __forceinline__ int look_up(int t) const {
    const int b = t * (kSpan / kBlock) + lane / 4;
    if (b * kBlock >= n_kv) return -1;
    const int p = __ldg(table + b);
    return p >= 0 && int64_t(p) < a.num_blocks ? p : -2;
  }
  __device__ __forceinline__ void load(int block) {
    phys = block;
    ks = vs = make_float4(0.f, 0.f, 0.f, 0.f);
    if (phys >= 0) {
      ks = __ldg(reinterpret_cast<const float4*>(a.key_scales + phys * stride + mine));
      vs = __ldg(reinterpret_cast<const float4*>(a.value_scales + phys * stride + mine));
    }
  }

  __device__ __forceinline__ void run(Shared* sh) {
    const int spans = (n_kv + kSpan - 1) / kSpan;
    int run_n = -127;  // exponent of the largest V scale so far
#pragma unroll 1
    for (int t = 0; t < spans; ++t) {
      const int next = look_up(t + 1);
      const int reach = n_kv - t * kSpan - 4 * lane;  // of its tokens, those below n_kv
      float k[4] = {ks.x, ks.y, ks.z, ks.w}, v[4] = {vs.x, vs.y, vs.z, vs.w};
      uint32_t spoil = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= reach) k[i] = v[i] = 0.f;
        if (!isfinite(v[i])) spoil |= 1u << i;
      }
      if (t >= kAhead && !wait_ahead(&sh->converted[t % kAhead], ((t - kAhead) / kAhead) & 1))
        return;
      TileInfo* info = &sh->info[t % kInfos];
      // n of the lane's 32 tokens (8 lanes).
      int n = int(top_bits(v) >> 23) - 127;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) n = max(n, __shfl_xor_sync(0xffffffffu, n, o));
      run_n = max(run_n, __reduce_max_sync(0xffffffffu, n));
      n = min(max(n, max(run_n - kRefSpread, -126)), 126);
      const float inv_v = __uint_as_float(uint32_t(127 - n) << 23);
      // A NaN V row is stored as zeros (see the head of the file).
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = spoil >> i & 1 ? 0.f : v[i] * inv_v;
      *reinterpret_cast<float4*>(&info->scale[0][4 * lane]) = make_float4(k[0], k[1], k[2], k[3]);
      *reinterpret_cast<float4*>(&info->scale[1][4 * lane]) = make_float4(v[0], v[1], v[2], v[3]);
      if (lane % 4 == 0) info->block[lane / 4] = phys;
      if (lane % 8 == 0) info->log_v[lane / 8] = float(n);
      const bool any = __any_sync(0xffffffffu, spoil != 0 || phys == -2);
      const bool past = __any_sync(0xffffffffu, reach < 4);
      if (any) {
        uint32_t skip = (phys == -2 ? 0xfu : 0u) << lane % 8 * 4;
        spoil <<= lane % 8 * 4;
#pragma unroll 1
        for (int o = 1; o < 8; o <<= 1) {
          skip |= __shfl_xor_sync(0xffffffffu, skip, o);
          spoil |= __shfl_xor_sync(0xffffffffu, spoil, o);
        }
        if (lane % 8 == 0) {
          info->skip[lane / 8] = skip;
          info->spoil[lane / 8] = spoil;
        }
      } else if (lane < 4) {
        info->skip[lane] = info->spoil[lane] = 0;
      }
      if (lane == 0) {
        info->any = any;
        info->dropped = past || any;
      }
      __syncwarp();
      if (lane == 0) ts::mbar_arrive(&sh->info_full[t % kInfos]);
      load(next);
    }
  }
};

// One block of codes (16 rows of a KV head) in a converter warp's registers: a row in 8 lanes, each
// with 8 codes of every 64 columns, so a lane's values are one 16-byte chunk of each half tile.
template <int D>
struct Codes {
  static constexpr int kHalves = D / 64;
  static constexpr int kLoads = kBlock / 4;  // 4 rows per load instruction
  uint2 raw[kLoads][kHalves];

  __device__ __forceinline__ void load(const uint8_t* block, int lane) {  // nullptr: zeros
    const uint2* src = reinterpret_cast<const uint2*>(block) + lane / 8 * (D / 8) + lane % 8;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf)
        raw[i][hf] = block != nullptr ? __ldg(src + i * (D / 2) + hf * 8) : make_uint2(0, 0);
  }
  // Rows row0 .. row0 + 15 of the fp16 tile at `dst` (128-byte swizzled halves of 64 columns), with
  // `scale` (of those rows) only where it is not 0.
  __device__ __forceinline__ void store(uint8_t* dst, const float* scale, int row0, int lane) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = row0 + i * 4 + lane / 8;
      const bool used = scale == nullptr || scale[i * 4 + lane / 8] != 0.f;
      uint8_t* base = dst + row * 128 + (((lane & 7) ^ (row & 7)) << 4);
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf) {
        const uint2 w = used ? raw[i][hf] : make_uint2(0, 0);
        uint32_t v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const __half2 x = ts::fp8_half2((k < 2 ? w.x : w.y) >> (16 * (k & 1)));
          v[k] = *reinterpret_cast<const uint32_t*>(&x);
        }
        *reinterpret_cast<uint4*>(base + hf * kKvHalf) = make_uint4(v[0], v[1], v[2], v[3]);
      }
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) paged_prefill_fp8_kernel(const Args a) {
  using G = Geo<D>;
  using Mma = ts::MmaOp<T>;
  const int pair = blockIdx.x, h = blockIdx.y, seq = blockIdx.z;
  const int q0 = __shfl_sync(0xffffffffu, a.qsl[seq], 0);
  const int q_end = __shfl_sync(0xffffffffu, a.qsl[seq + 1], 0);
  if (q0 < 0 || q_end > a.num_tokens) return;  // not a chunk of this call's rows
  const int q_len = q_end - q0;
  const int tile0 = pair * a.q_tiles;
  if (tile0 * a.tq >= q_len) return;
  const int ctx = min(__shfl_sync(0xffffffffu, a.context_lens[seq], 0), a.max_blocks * kBlock);
  const int p0 = ctx - q_len;  // position of the first query row; negative rows see nothing
  int n_t[kQTiles];            // KV tiles each query tile needs
  int n_kv = 0;                // keys the CTA's last query row sees
#pragma unroll
  for (int x = 0; x < kQTiles; ++x) {
    const int first = (tile0 + x) * a.tq;
    const int n = x < a.q_tiles && first < q_len ? max(0, p0 + min(q_len, first + a.tq)) : 0;
    n_t[x] = (n + kKvTile - 1) / kKvTile;
    n_kv = max(n_kv, n);
  }
  const int n_max = (n_kv + kKvTile - 1) / kKvTile;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ts::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023) & ~1023u) - raw_addr);
  auto sQ = [&](int x) { return smem + x * G::kQBytes; };
  auto sK = [&](int st) { return smem + kQTiles * G::kQBytes + st * G::kKvBytes; };
  auto sV = [&](int st) { return sK(kStages + st); };
  Shared* sh = reinterpret_cast<Shared*>(smem + G::kTiles);

  // Through a shuffle, so that the compiler knows a role's control flow to be uniform.
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;

  // Token of a tile row, row / group: exact in fp32 for rows below 128.
  const float inv_group = 1.f / float(a.group);
  auto row_token = [&](int row) { return int((float(row) + 0.5f) * inv_group); };
  // The softmax warps' queries as they are, 16 bytes a lane and D / 8 lanes a row, on their way
  // while the barriers and tensor memory are set up.
  constexpr int kQLanes = D / 8, kQRows = 32 / kQLanes;
  auto q_place = [&](int w) {  // this lane's 16 bytes of row w of the warp's 32
    const int c = lane % kQLanes;
    return sQ(warp / 4 & 1) + (warp & 3) * 32 * 128 + (c >> 3) * kQHalf + w * 128 +
           (((c & 7) ^ (w & 7)) << 4);
  };
  if (warp < 4 * kQTiles) {
#pragma unroll 4
    for (int w = lane / kQLanes; w < 32; w += kQRows) {
      const int row = (warp & 3) * 32 + w, token = row_token(row);
      const int q = (tile0 + warp / 4) * a.tq + token;
      const bool in = token < a.tq && q < q_len;
      const T* src = static_cast<const T*>(a.query);
      if (in)
        src += int64_t(q0 + q) * a.q_stride + (h * a.group + row - token * a.group) * D +
               lane % kQLanes * 8;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ts::smem_u32(q_place(w))),
                   "l"(src), "r"(in ? 16 : 0)
                   : "memory");
    }
  }
  Scout scout(a, seq, h, n_kv, lane);
  if (warp == 12) scout.load(scout.look_up(0));
  if (warp == 14 && lane == 0) {
    ts::mbar_init(&sh->q_full, 4 * kQTiles);  // one arrival a warp, here and below
    for (int i = 0; i < kStages; ++i) {
      ts::mbar_init(&sh->k_full[i], kUnits / 2);
      ts::mbar_init(&sh->k_empty[i], 1);
      ts::mbar_init(&sh->v_full[i], kUnits / 2);
      ts::mbar_init(&sh->v_empty[i], 1);
    }
    for (int i = 0; i < kInfos; ++i) ts::mbar_init(&sh->info_full[i], 1);
    for (int i = 0; i < kAhead; ++i) ts::mbar_init(&sh->converted[i], kUnits * kTilesPerSpan);
    for (int x = 0; x < kQTiles; ++x) {
      for (int b = 0; b < 2; ++b) {
        ts::mbar_init(&sh->s_full[x][b], 1);
        ts::mbar_init(&sh->p_full[x][b], 4);
      }
      ts::mbar_init(&sh->pv_done[x], 1);
      ts::mbar_init(&sh->o_full[x], 1);
    }
    ts::mbar_init(&sh->drain, 1);
    ts::fence_mbar_init();
  }
  if (warp == 13) {
    ts::tc::tmem_alloc(&sh->tmem, kTmemCols);
    ts::tc::tmem_relinquish();
  }
  ts::tc::fence_before_sync();
  __syncthreads();
  ts::tc::fence_after_sync();
  constexpr uint32_t tmem = 0;  // all 512 columns: the allocation starts at the first

  if (warp >= 8) {
    if (warp == 12) {
      scout.run(sh);
    } else if (warp != 13) {
      // ---------------------------------------------------------- converters
      const int total = n_max * kUnits;
      const int64_t block_bytes = int64_t(a.num_kv_heads) * kBlock * D;
      Codes<D> codes[2];
      auto fetch = [&](Codes<D>& c, int u) -> bool {
        if (u >= total) return true;
        const int j = u / kUnits, k = u % kUnits, t = j / kTilesPerSpan;
        if (!wait_ahead(&sh->info_full[t % kInfos], (t / kInfos) & 1)) return false;
        const int phys =
            sh->info[t % kInfos].block[j % kTilesPerSpan * (kUnits / 2) + k % (kUnits / 2)];
        const uint8_t* pool = (k < kUnits / 2 ? a.key_pool : a.value_pool) + h * kBlock * D;
        c.load(phys >= 0 ? pool + phys * block_bytes : nullptr, lane);
        return true;
      };
      auto convert = [&](Codes<D>& c, int u) -> bool {
        const int j = u / kUnits, k = u % kUnits, st = j % kStages, t = j / kTilesPerSpan;
        const bool is_v = k >= kUnits / 2;
        if (j >= kStages && !wait_ahead(is_v ? &sh->v_empty[st] : &sh->k_empty[st],
                                       ((j - kStages) / kStages) & 1))
          return false;
        const TileInfo& info = sh->info[t % kInfos];
        const int row0 = k % (kUnits / 2) * kBlock;
        // K's rows past the last key make scores that are masked; V's are zeros.
        c.store(is_v ? sV(st) : sK(st),
                is_v && info.dropped ? info.scale[1] + j % kTilesPerSpan * kKvTile + row0 : nullptr,
                row0, lane);
        ts::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          ts::mbar_arrive(is_v ? &sh->v_full[st] : &sh->k_full[st]);
          ts::mbar_arrive(&sh->converted[t % kAhead]);
        }
        return true;
      };
      int u = warp < 12 ? warp - 8 : warp - 10;
      bool ok = fetch(codes[0], u) && fetch(codes[1], u + kConverters);
      while (ok && u < total) {
        ok = convert(codes[0], u) && fetch(codes[0], u + 2 * kConverters);
        u += kConverters;
        if (ok && u < total) ok = convert(codes[1], u) && fetch(codes[1], u + 2 * kConverters);
        u += kConverters;
      }
    } else if (n_max > 0) {
      // ---------------------------------------------------------- MMA issuer
      // The whole warp runs it, so addresses and descriptors stay in uniform registers, and one
      // elected lane issues.
      constexpr uint32_t idesc_qk = ts::tc::idesc_f16(false, kRows, kKvTile, false);
      constexpr uint32_t idesc_pv = ts::tc::idesc_f16(false, kRows, D, true);
      // Low words of the shared-memory descriptors: address / 16, and V's distance between halves.
      const uint32_t q_lo = ts::smem_u32(sQ(0)) >> 4 | 1u << 16;
      const uint32_t k_lo = ts::smem_u32(sK(0)) >> 4 | 1u << 16;
      const uint32_t v_lo = ts::smem_u32(sV(0)) >> 4 | uint32_t(kKvHalf >> 4) << 16;
      // The last query tile to use KV tile j releases its K (after QK) and V (after PV).
      auto last_user = [&](int j) { return j < n_t[1] ? 1 : 0; };
      bool ok = wait_warp(&sh->q_full, 0);
      // Step i: PV(i - 2) then QK(i), of each query tile in turn.
#pragma unroll 1
      for (int i = 0; ok && i < n_max + 2; ++i) {
        const int j = i - 2, b = i & 1, sk = i % kStages, sv = j & (kStages - 1);
#pragma unroll 1
        for (int x = 0; ok && x < kQTiles; ++x) {
          const int n_x = x ? n_t[1] : n_t[0];
          const uint32_t s_tmem = tmem + x * 128 + b * kKvTile;
          if (j >= 0 && j < n_x) {
            // The first query tile has waited for this V already (and below for this K): a wait
            // costs a hundred clocks even then.
            ok = ((x == 1 && j < n_t[0]) || wait_warp(&sh->v_full[sv], (j / kStages) & 1)) &&
                 wait_warp(&sh->p_full[x][b], (j / 2) & 1);
            if (!ok) break;
            ts::tc::fence_after_sync();
            const uint32_t dv = v_lo + sv * (G::kKvBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < kKvTile / 16; ++kk)
              ts::tc::mma_ts_elect(tmem + 256 + x * 128, s_tmem + kk * 8, dv + kk * 128, idesc_pv,
                                   j > 0 || kk > 0);
            ts::tc::commit_elect(j + 1 == n_x ? &sh->o_full[x] : &sh->pv_done[x]);
            if (x == last_user(j) && j + kStages < n_max) ts::tc::commit_elect(&sh->v_empty[sv]);
          }
          if (i < n_x) {
            ok = (x == 1 && i < n_t[0]) || wait_warp(&sh->k_full[sk], (i / kStages) & 1);
            if (!ok) break;
            ts::tc::fence_after_sync();
            const uint32_t dq = q_lo + x * (G::kQBytes >> 4);
            const uint32_t dk = k_lo + sk * (G::kKvBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              ts::tc::mma_ss_elect(s_tmem, dq + (((kk >> 2) * kQHalf + (kk & 3) * 32) >> 4),
                                   dk + (((kk >> 2) * kKvHalf + (kk & 3) * 32) >> 4), idesc_qk,
                                   kk > 0);
            ts::tc::commit_elect(&sh->s_full[x][b]);
            if (x == last_user(i) && i + kStages < n_max) ts::tc::commit_elect(&sh->k_empty[sk]);
          }
        }
      }
      if (!ok) {  // the MMAs in flight end before shared and tensor memory are released
        ts::tc::commit_elect(&sh->drain);
        ts::mbar_wait_bounded(&sh->drain, 0);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax / epilogue
    const int x = warp / 4;               // query tile of this warpgroup
    const int r = threadIdx.x - 128 * x;  // tile row == TMEM lane
    const int n_x = n_t[x];
    const int i = row_token(r);
    const int qi = (tile0 + x) * a.tq + i;
    const int pos = i < a.tq && qi < q_len ? p0 + qi : p0 + q_len - 1;  // rows of no query: anything
    const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t o_col = 256 + x * 128;

    // q's rows times 2^(14 - exponent of their amax), in fp16; `sl` undoes it (times the softmax
    // scale, whose sign goes with q). A warp loads its 32 rows 16 bytes a lane, D / 8 lanes a row.
    float sl = 0.f;
    {
      asm volatile("cp.async.wait_all;" ::: "memory");
      const float base = fabsf(a.scale_log2);
      constexpr int kBatch = 4;  // rows of a lane at a time
#pragma unroll 1
      for (int w0 = lane / kQLanes; w0 < 32; w0 += kBatch * kQRows) {
        uint4 v[kBatch];
        uint32_t m[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) v[b] = *reinterpret_cast<const uint4*>(q_place(w0 + b * kQRows));
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const uint32_t wds[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
          m[b] = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 u = Mma::unpack(wds[k]);
            m[b] = max(m[b], max(ts::abs_bits(u.x), ts::abs_bits(u.y)));
          }
        }
#pragma unroll
        for (int o = kQLanes / 2; o > 0; o >>= 1)
#pragma unroll
          for (int b = 0; b < kBatch; ++b) m[b] = max(m[b], __shfl_xor_sync(0xffffffffu, m[b], o));
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int e = max(int(m[b] >> 23), 27);  // biased exponent; tiny rows keep a finite factor
          const float up = copysignf(__uint_as_float(uint32_t(127 + 14 + 127 - e) << 23), a.scale_log2);
          const int my = __shfl_sync(0xffffffffu, e, lane % kQRows * kQLanes);
          if (lane / kQRows == w0 / kQRows + b) sl = base * __uint_as_float(uint32_t(my - 14) << 23);
          const uint32_t wds[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 u = Mma::unpack(wds[k]);
            o[k] = pack_half2(u.x * up, u.y * up);
          }
          *reinterpret_cast<uint4*>(q_place(w0 + b * kQRows)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
      ts::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ts::mbar_arrive(&sh->q_full);
    }

    const uint64_t sl2 = ts::two(sl, sl);
    const int pos_max = __reduce_max_sync(0xffffffffu, pos);
    const int pos_min = __reduce_min_sync(0xffffffffu, pos);
    // Maximum that the weights and O are relative to, the one of the sum, the sum.
    float t_run = -INFINITY, m_run = -INFINITY, l_run = 0.f;
    bool saw_nan = false;  // a V row that holds one; one of K is in the scores
    bool ok = true;
    for (int j = 0; j < n_x; ++j) {
      if (!wait_warp(&sh->s_full[x][j & 1], (j / 2) & 1)) {
        ok = false;
        break;
      }
      ts::tc::fence_after_sync();
      const uint32_t s_col = x * 128 + (j & 1) * kKvTile;
      uint32_t sa[32];
      ts::tc::tmem_ld32(lane_base + s_col, sa);
      constexpr int kGroups = kKvTile / 32;  // of 32 columns
      const volatile TileInfo* info = &sh->info[j / kTilesPerSpan % kInfos];
      const int word = j % kTilesPerSpan * kGroups;  // of the span's column masks
      const bool odd_columns = info->any != 0;
      float corr_o = 1.f;  // of O, when the weights' maximum moves
      const int limit = pos - j * kKvTile;  // columns c <= limit are visible
      // Column groups of 32 that some row of the warp sees, and those every row sees whole.
      const int n_some = min(kGroups, max(0, pos_max - j * kKvTile + 32) / 32);
      const int n_whole = odd_columns ? 0 : max(0, pos_min - j * kKvTile + 1) / 32;
      // K's (w = 0) scales, or V's over 2^n (1), of columns 32 c + 4 k .. 32 c + 4 k + 3.
      const uint32_t scale_at = ts::smem_u32(&sh->info[j / kTilesPerSpan % kInfos].scale[0][word * 32]);
      auto scales = [&](int w, int c, int k) {
        ulonglong2 v;
        asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];"
                     : "=l"(v.x), "=l"(v.y)
                     : "r"(scale_at + w * (kSpan * 4) + c * 128 + k * 16));
        return v;
      };
      // Scores of columns 32 c .. 32 c + 31, which `sa` holds raw, plus `plus`.
      auto scores = [&](int c, float plus, uint64_t (&e)[16]) {
        const uint64_t plus2 = ts::two(plus, plus);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const ulonglong2 ks = scales(0, c, k);
          e[2 * k] = ts::fma2(ts::two(sa[4 * k], sa[4 * k + 1]), ts::mul2(ks.x, sl2), plus2);
          e[2 * k + 1] = ts::fma2(ts::two(sa[4 * k + 2], sa[4 * k + 3]), ts::mul2(ks.y, sl2), plus2);
        }
      };
      // Maximum of scores, and of scores plus log2(V's scale / 2^n).
      auto maxima = [&](int c, const uint64_t (&e)[16], float& m, float& mt) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float2 v = ts::halves(e[k]);
          const ulonglong2 vs2 = scales(1, c, k / 2);
          const float2 vs = ts::halves(k % 2 ? vs2.y : vs2.x);
          m = ts::max3f(m, v.x, v.y);
          mt = ts::max3f(mt, v.x + fmaxf(__log2f(vs.x), kLeastLog),
                         v.y + fmaxf(__log2f(vs.y), kLeastLog));
        }
      };
      auto mask = [&](uint64_t (&e)[16], int c) {
        const int lim = limit - 32 * c;
        const uint32_t seen = lim >= 31 ? ~0u : lim < 0 ? 0u : (2u << lim) - 1;
        const uint32_t keep = seen & ~info->skip[word + c],
                       spoil = seen & info->spoil[word + c];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float2 v = ts::halves(e[k]);
          e[k] = ts::two(keep >> 2 * k & 1 ? v.x : -INFINITY, keep >> (2 * k + 1) & 1 ? v.y : -INFINITY);
        }
        saw_nan |= spoil != 0;
      };
      if (__any_sync(0xffffffffu, t_run == -INFINITY)) {  // a row that has seen nothing yet
        float m = -INFINITY, mt = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < n_some; ++c) {
          ts::tc::wait_ld(sa);
          uint64_t e[16];
          scores(c, 0.f, e);
          if (c >= n_whole) mask(e, c);
          float mg = -INFINITY;
          maxima(c, e, m, mg);
          mt = fmaxf(mt, mg + info->log_v[word + c]);
          ts::tc::tmem_ld32(lane_base + s_col + (c + 1 < n_some ? c + 1 : 0) * 32, sa);
        }
        if (t_run == -INFINITY) m_run = m, t_run = mt;
      }
      // P of columns 32 c .. 32 c + 31. Masked columns, and a warp whose maximum moves, run their own
      // copies of the code: where the paths met again, the registers of a whole row were copied.
      auto columns = [&](int c, auto masked) {
        const float log_v = info->log_v[word + c];
        const float less = t_run == -INFINITY ? 0.f : log_v - t_run;
        ts::tc::wait_ld(sa);
        uint64_t e[16], sum2 = ts::two(0.f, 0.f);  // log2 of P, two columns each; their sum
        scores(c, less, e);
        if (masked) mask(e, c);
        if (c + 1 < n_some) ts::tc::tmem_ld32(lane_base + s_col + (c + 1) * 32, sa);
        // From the weights' maximum and reference to the sum's; nothing seen: 0.
        const float to_sum = t_run == -INFINITY ? 0.f : ts::ex2(-less - m_run);
        uint32_t pw[16];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const ulonglong2 vs = scales(1, c, k);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float2 u = ts::halves(e[2 * k + i]);
            u = make_float2(ts::ex2(u.x), ts::ex2(u.y));
            sum2 = ts::add2(sum2, ts::two(u.x, u.y));
            u = ts::halves(ts::mul2(ts::two(u.x, u.y), i ? vs.y : vs.x));
            pw[2 * k + i] = pack_half2(u.x, u.y);
          }
        }
        const float2 s2 = ts::halves(sum2);
        const float sum_u = s2.x + s2.y, part = sum_u * to_sum;
        if (__all_sync(0xffffffffu, sum_u <= kMostSumU && part <= kMostSum)) {
          ts::tc::tmem_st16(lane_base + s_col + c * 16, pw);
          l_run += part;
          return;
        }
        // Once more, with the maxima that the columns need; the next columns' load is repeated.
        if (c + 1 < n_some) ts::tc::wait_ld(sa);
        ts::tc::tmem_ld32(lane_base + s_col + c * 32, sa);
        ts::tc::wait_ld(sa);
        scores(c, less, e);
        if (masked) mask(e, c);
        float m = -INFINITY, mt = -INFINITY;
        maxima(c, e, m, mt);
        m += -less;  // s
        const float up = fmaxf(mt, 0.f), f = ts::ex2(-up);
        if (m > m_run) {
          l_run *= ts::ex2(m_run - m);
          m_run = m;
        }
        t_run += up;
        corr_o *= f;
#pragma unroll 1
        for (int b = 0; b < c; ++b) {  // the tile's P so far
          uint32_t pw[16];
          ts::tc::wait_st();
          ts::tc::tmem_ld16(lane_base + s_col + b * 16, pw);
          ts::tc::wait_ld(pw);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&pw[k]));
            pw[k] = pack_half2(u.x * f, u.y * f);
          }
          ts::tc::tmem_st16(lane_base + s_col + b * 16, pw);
        }
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const ulonglong2 vs = scales(1, c, k);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float2 u = ts::halves(e[2 * k + i]);
            u = make_float2(ts::ex2(u.x - up), ts::ex2(u.y - up));
            sum += u.x + u.y;
            u = ts::halves(ts::mul2(ts::two(u.x, u.y), i ? vs.y : vs.x));
            pw[2 * k + i] = pack_half2(u.x, u.y);
          }
        }
        ts::tc::tmem_st16(lane_base + s_col + c * 16, pw);
        l_run += sum * (t_run == -INFINITY ? 0.f : ts::ex2(up - less - m_run));
        if (c + 1 < n_some) ts::tc::tmem_ld32(lane_base + s_col + (c + 1) * 32, sa);
      };
#pragma unroll 1
      for (int c = 0; c < min(n_whole, n_some); ++c) columns(c, std::false_type{});
#pragma unroll 1
      for (int c = min(n_whole, n_some); c < n_some; ++c) columns(c, std::true_type{});
      if (n_some == 0) ts::tc::wait_ld(sa);  // nothing above has waited for the load
#pragma unroll 1
      for (int c = n_some; c < kGroups; ++c) {
        uint32_t pw[16] = {};
        ts::tc::tmem_st16(lane_base + s_col + c * 16, pw);
      }
      if (j > 0 && __any_sync(0xffffffffu, corr_o != 1.f)) {
        // O holds the tiles up to j - 1 (up to j - 2 it does since S of tile j was ready).
        if (!wait_warp(&sh->pv_done[x], (j - 1) & 1)) {
          ok = false;
          break;
        }
        ts::tc::fence_after_sync();
#pragma unroll 1
        for (int c4 = 0; c4 < D / 32; ++c4) {
          uint32_t rr[32];
          ts::tc::tmem_ld32(lane_base + o_col + c4 * 32, rr);
          ts::tc::wait_ld(rr);
#pragma unroll
          for (int c = 0; c < 32; ++c) rr[c] = __float_as_uint(__uint_as_float(rr[c]) * corr_o);
          ts::tc::tmem_st32(lane_base + o_col + c4 * 32, rr);
        }
      }
      ts::tc::wait_st();
      ts::tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) ts::mbar_arrive(&sh->p_full[x][j & 1]);
    }
    if (ok && n_x > 0) ok = wait_warp(&sh->o_full[x], 0);
    if (!ok) m_run = INFINITY;  // a wait gave up: the rows become NaN below, whatever O holds
    ts::tc::fence_after_sync();
    if (x < a.q_tiles) {
      // A row that saw nothing has a sum of 0, and O = 0. An infinite score makes NaNs.
      float inv = l_run > 0.f ? ts::ex2(t_run - m_run) / l_run : l_run;
      if (saw_nan || m_run == INFINITY) inv = __uint_as_float(0x7fc00000u);
      // The row goes to the warp's part of its Q tile (no MMA reads it any more), 16 bytes at a
      // time in swizzled places, and from there to memory in whole rows.
      uint8_t* stage = sQ(x) + (warp & 3) * 32 * D * 2;
      constexpr int kChunks = D / 8;
#pragma unroll 1
      for (int c4 = 0; c4 < D / 32; ++c4) {
        uint32_t rr[32] = {};
        if (n_x > 0) {
          ts::tc::tmem_ld32(lane_base + o_col + c4 * 32, rr);
          ts::tc::wait_ld(rr);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            pk[k] = Mma::pack(__uint_as_float(rr[8 * c + 2 * k]) * inv,
                              __uint_as_float(rr[8 * c + 2 * k + 1]) * inv);
          *reinterpret_cast<uint4*>(stage + lane * D * 2 + ((c4 * 4 + c) ^ (lane & 7)) * 16) =
              make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
      }
      __syncwarp();
#pragma unroll 1
      for (int w0 = lane / kChunks; w0 < 32; w0 += 4 * kQRows) {
        uint4 v[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int w = w0 + b * kQRows;
          v[b] = *reinterpret_cast<const uint4*>(stage + w * D * 2 + (lane % kChunks ^ (w & 7)) * 16);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int row = (warp & 3) * 32 + w0 + b * kQRows, token = row_token(row);
          const int q = (tile0 + x) * a.tq + token;
          if (token < a.tq && q < q_len)
            *reinterpret_cast<uint4*>(
                static_cast<T*>(a.out) +
                (int64_t(q0 + q) * a.num_q_heads + h * a.group + row - token * a.group) * D +
                lane % kChunks * 8) = v[b];
        }
      }
    }
  }
  ts::tc::fence_before_sync();
  __syncthreads();
  if (warp == 13) {
    ts::tc::fence_after_sync();
    ts::tc::tmem_dealloc(sh->tmem, kTmemCols);
  }
}

bool tc_path(int group, int hkv, int hd, int bs, int dtype, const void* kp, const void* vp,
             const void* ks, const void* vs, const void* q, int64_t q_stride, const void* out, int num_seqs) {
  if (dtype != TS_BFLOAT16 && dtype != TS_FLOAT16) return false;
  if ((hd != 64 && hd != 128) || bs != kBlock || group > kRows) return false;
  if (num_seqs > 65535 || hkv > 65535) return false;
  if ((reinterpret_cast<uint64_t>(kp) | reinterpret_cast<uint64_t>(vp) |
       reinterpret_cast<uint64_t>(ks) | reinterpret_cast<uint64_t>(vs) |
       reinterpret_cast<uint64_t>(q) | reinterpret_cast<uint64_t>(out)) % 16)
    return false;
  return (q_stride * 2) % 16 == 0;
}

int sm_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cached[dev] == 0) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    cached[dev] = n > 0 ? n : 148;
  }
  return cached[dev];
}

template <typename T, int D>
int launch(const Args& a, dim3 grid, cudaStream_t s) {
  auto kern = paged_prefill_fp8_kernel<T, D>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             Geo<D>::kSmemBytes);
  if (e != cudaSuccess)
    return ts::set_error(static_cast<int>(e), "paged_prefill_fp8: %s", cudaGetErrorString(e));
  kern<<<grid, kThreads, Geo<D>::kSmemBytes, s>>>(a);
  return ts::launch_status("paged_prefill_fp8");
}

}  // namespace

extern "C" int ts_paged_prefill_fp8(void* out, const void* query, int64_t query_token_stride,
                                    const void* key_pool, const void* value_pool,
                                    const float* key_scales, const float* value_scales,
                                    const int32_t* block_tables, int32_t max_blocks_per_seq,
                                    const int32_t* query_start_loc, const int32_t* context_lens,
                                    int32_t num_seqs, int32_t num_query_tokens,
                                    int32_t max_query_len, int32_t num_q_heads,
                                    int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                    int64_t num_blocks, float scale, int32_t dtype, void* stream) {
  const int es = ts::dtype_size(dtype);
  if (es == 0)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT, "paged_prefill_fp8: bad dtype %d", dtype);
  if (num_seqs < 0 || num_query_tokens < 0 || max_query_len < 0 || num_q_heads <= 0 ||
      num_kv_heads <= 0 || num_q_heads % num_kv_heads || head_dim <= 0 || block_size <= 0 ||
      num_blocks <= 0 || max_blocks_per_seq <= 0)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT,
                         "paged_prefill_fp8: bad sizes (seqs %d, tokens %d, heads %d/%d, head_dim "
                         "%d, block_size %d)",
                         num_seqs, num_query_tokens, num_q_heads, num_kv_heads, head_dim,
                         block_size);
  if (query_token_stride < int64_t(num_q_heads) * head_dim)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT, "paged_prefill_fp8: query stride too small");
  if (num_seqs == 0 || num_query_tokens == 0 || max_query_len == 0) return ts::ok();
  if (!out || !query || !key_pool || !value_pool || !key_scales || !value_scales ||
      !block_tables || !query_start_loc || !context_lens)
    return ts::set_error(TS_ERR_INVALID_ARGUMENT, "paged_prefill_fp8: null pointer");
  if ((reinterpret_cast<uint64_t>(key_scales) | reinterpret_cast<uint64_t>(value_scales)) % 4 ||
      (reinterpret_cast<uint64_t>(query) | reinterpret_cast<uint64_t>(out)) % es)
    return ts::set_error(TS_ERR_MISALIGNED, "paged_prefill_fp8: pointers not element-aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int group = num_q_heads / num_kv_heads;
  if (!tc_path(group, num_kv_heads, head_dim, block_size, dtype, key_pool, value_pool,
               key_scales, value_scales, query, query_token_stride, out, num_seqs))
    return ts::paged_attention_portable(out, query, query_token_stride, key_pool, value_pool,
                                        block_tables, max_blocks_per_seq, query_start_loc,
                                        context_lens, num_seqs, num_query_tokens, num_q_heads,
                                        num_kv_heads, head_dim, block_size, num_blocks, scale,
                                        dtype, s, key_scales, value_scales);
  Args a;
  a.out = out;
  a.query = query;
  a.q_stride = query_token_stride;
  a.key_pool = static_cast<const uint8_t*>(key_pool);
  a.value_pool = static_cast<const uint8_t*>(value_pool);
  a.key_scales = key_scales;
  a.value_scales = value_scales;
  a.block_tables = block_tables;
  a.qsl = query_start_loc;
  a.context_lens = context_lens;
  a.max_blocks = max_blocks_per_seq;
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = group;
  a.num_tokens = num_query_tokens;
  a.tq = kRows / group;
  a.num_blocks = num_blocks;
  a.scale_log2 = scale * kLog2e;
  const int longest = max_query_len < num_query_tokens ? max_query_len : num_query_tokens;
  const int tiles = (longest + a.tq - 1) / a.tq;
  // Two query tiles a CTA share each converted K/V tile; one a CTA shortens a CTA's time when there
  // are too few pairs for the SMs (one 512-token chunk over 1,024 tokens: 32 us instead of 38).
  const int64_t pairs = int64_t((tiles + 1) / 2) * num_kv_heads * num_seqs;
  a.q_tiles = pairs < sm_count() ? 1 : kQTiles;
  const dim3 grid((tiles + a.q_tiles - 1) / a.q_tiles, num_kv_heads, num_seqs);
  if (dtype == TS_BFLOAT16)
    return head_dim == 128 ? launch<__nv_bfloat16, 128>(a, grid, s)
                           : launch<__nv_bfloat16, 64>(a, grid, s);
  return head_dim == 128 ? launch<__half, 128>(a, grid, s) : launch<__half, 64>(a, grid, s);
}
