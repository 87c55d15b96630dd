// The projection on 8-bit operands (float8.cuh): out[m][n] = sum_k x[m][k] w[n][k] (+ bias[n]), float32 sums, float32 or bf16 rows.
//
// tcgen05.mma of kind mxf8f6f4 multiplies 32 channels at a time and takes a power of two per row and 32 channels from tensor memory: the
// exponent bytes as they lie in the matrices, one byte for four instructions (a block of 128 channels).  No product is scaled by an
// instruction of ours, and partial sums of different blocks meet in one float32 accumulator.
//
// 147456 x 128 -> 512 in bf16: 30 us, bound by its 151 MB of writes (5.7 TB/s in all); 4096 x 4096 -> 4096: 53.4 us, 2570 TFLOP/s, bound by the tensor core
// and by the turns of its tiles.
#include <cuda.h>

#include "float8.cuh"
#include "tc05.cuh"
#include "tc_kernels.cuh"

namespace tc {

using namespace tc05;

lf_status make_map_bytes(lf_context* ctx, CUtensorMap* map, const void* base, uint64_t width, uint64_t rows, uint64_t pitch, uint32_t box_rows);
lf_status make_map_rows(lf_context* ctx, CUtensorMap* map, const void* base, bool f32, uint64_t width, uint64_t rows, uint32_t box_rows, bool narrow = false);
lf_status make_map_tiles(lf_context* ctx, CUtensorMap* map, const void* base, uint64_t tiles, uint32_t box_tiles);

void configure_float8_few();
bool float8_few_takes(int64_t rows, int k);
lf_status float8_few(lf_context* ctx, const void* source, int dtype, const f8::Matrix& x, const f8::Matrix& w, const float* bias, void* out, int out_dtype);

constexpr int F8_BM = 128, F8_BK = 128;      // a k step is a block of the format, and a row of it 128 bytes of shared memory
constexpr int F8_A_BYTES = F8_BM * F8_BK;
constexpr int F8_DEEP = 1024;                // channels from which the deeper ring pays (4096 x 4096 -> 4096: 57.3 -> 54.2 us)

// Places in tensor memory for a group's exponents, in turn.  A group writes its place when its first step's loads are here and its tile's accumulator is free; the products that
// read the place before it, F8_SLOTS groups back, have to be done then.  If they belong to a tile `accumulators` or more back, the accumulator's wait says so (a tile has
// at least one group).  Otherwise the groups between lie in at most two tiles, so that all but one of them have four steps, and the last of those products is
// 4 (F8_SLOTS - 2) + 2 steps back or more: the ring's wait for the step `stages` back says so.
constexpr int F8_SLOTS = 4;
__host__ __device__ constexpr bool slots_suffice(int stages, int accumulators) { return accumulators <= 2 && accumulators <= F8_SLOTS && stages <= 4 * (F8_SLOTS - 2) + 2; }

struct Float8Params {
  int m, n, k;
  int vector_out;              // rows start on 16-byte boundaries: they leave by TMA
  const float* bias;           // [n] or null
  const uint8_t *ex, *ew;      // exponents
  int64_t ex_tiles, ew_tiles;  // 128-row tiles of each
  int x_format;                // w is e4m3
  void* out;
  Status* status;
};

// kind::mxf8f6f4, scales 2^(byte - 127): formats of A and B (0 e4m3, 1 e5m2), both K-major; `id`: which byte of a scale word
__device__ __forceinline__ uint32_t make_idesc_f8(int M, int N, int a_format, int b_format, int id) {
  return ((uint32_t)id << 4) | ((uint32_t)a_format << 7) | ((uint32_t)b_format << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) |
         ((uint32_t)(M >> 4) << 24) | ((uint32_t)id << 29);
}
template <int CTAS>
__device__ __forceinline__ void umma_f8_scaled(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scale, uint32_t b_scale,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::%7.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scale), "r"(b_scale), "r"(accumulate), "n"(CTAS)
      : "memory");
}
// 32 rows of 16 bytes of shared memory -> four columns of tensor memory, the same for each quarter of the lanes
template <int CTAS>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::%2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc), "n"(CTAS) : "memory");
}

// Staging tiles of 32 rows: of 128 bytes (128-byte swizzle) or, NARROW, 64 (64-byte swizzle).
template <bool NARROW>
__device__ __forceinline__ uint32_t staged_at(int row, int piece) {
  return NARROW ? row * 64 + ((piece ^ (row >> 1 & 3)) << 4) : swizzle128_offset(row, piece);
}
// COUNT of a lane's columns of its row, with the bias, to the tile's pieces from `piece` on.
template <bool F32, bool NARROW, int COUNT>
__device__ __forceinline__ void stage_columns(uint8_t* stage, const float* bias, const uint32_t* r, int piece, int lane) {
  constexpr int kPiece = F32 ? 4 : 8;      // columns of 16 bytes
#pragma unroll
  for (int c = 0; c < COUNT; c += kPiece) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < kPiece; e += 4) {
      const float4 b = *reinterpret_cast<const float4*>(bias + c + e);
      const float2 x = add2(make_float2(__uint_as_float(r[c + e]), __uint_as_float(r[c + e + 1])), make_float2(b.x, b.y));
      const float2 y = add2(make_float2(__uint_as_float(r[c + e + 2]), __uint_as_float(r[c + e + 3])), make_float2(b.z, b.w));
      if (F32) { w[0] = __float_as_uint(x.x); w[1] = __float_as_uint(x.y); w[2] = __float_as_uint(y.x); w[3] = __float_as_uint(y.y); }
      else {
        const __nv_bfloat162 p0 = __floats2bfloat162_rn(x.x, x.y), p1 = __floats2bfloat162_rn(y.x, y.y);
        w[e / 2] = *reinterpret_cast<const uint32_t*>(&p0);
        w[e / 2 + 1] = *reinterpret_cast<const uint32_t*>(&p1);
      }
    }
    *reinterpret_cast<uint4*>(stage + staged_at<NARROW>(lane, piece + c / kPiece)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// The staged rows to columns from c0 on of rows from row0 on (the whole warp): by TMA, or, where no 16-byte access divides the rows, AHEAD at a time: the loads of
// that many, then their stores.  (Eight: 3001 x 449 x 1283 in float32 13.1 -> 12.1 us, its input's gradient 10.8 -> 10.1.  The kernels of 256 columns have no registers for it: eight
// there cost aligned rows, that never come here, 147456 x 128 x 512 43.1 -> 43.9 us.)
template <bool F32, bool NARROW, int AHEAD>
__device__ __forceinline__ void send_columns(const uint8_t* stage, const CUtensorMap* map, int vector_out, void* out, int c0, int row0, int m, int n, int lane) {
  constexpr int kColumns = (F32 ? 32 : 64) >> NARROW, kPiece = F32 ? 4 : 8;
  if (vector_out) {
    fence_async_smem();
    __syncwarp();
    if (lane == 0) { tma_store_3d(map, stage, c0, row0, 0); bulk_commit(); }
    return;
  }
  __syncwarp();
  const int rows = min(32, m - row0);
  for (int row = 0; row < rows; row += AHEAD) {
#pragma unroll
    for (int e = 0; e < kColumns; e += 32) {
      const int c = e + lane;
      const bool here = c < kColumns && c0 + c < n;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const uint8_t* from = stage + staged_at<NARROW>(row + k, c / kPiece);
        const int64_t at = (int64_t)(row0 + row + k) * n + c0 + c;
        if (here && row + k < rows) {
          if (F32) static_cast<float*>(out)[at] = *reinterpret_cast<const float*>(from + c % kPiece * 4);
          else static_cast<bf16*>(out)[at] = *reinterpret_cast<const bf16*>(from + c % kPiece * 2);
        }
      }
    }
  }
  __syncwarp();
}

// A warp's COLUMNS columns of 32 rows from (row0, col0) on, from registers, with the bias.
template <int COLUMNS, bool F32, bool NARROW, int AHEAD>
__device__ __forceinline__ void send_share(const uint32_t (&r)[COLUMNS / 32][32], uint8_t* stage, const float* bias, const CUtensorMap* map, const Float8Params& p, int col0,
                                           int row0, int lane) {
  constexpr int kSend = (F32 ? 32 : 64) >> NARROW, kStage = kSend < 32 ? kSend : 32;      // columns of a staging tile, and staged at a time
#pragma unroll
  for (int c = 0; c < COLUMNS; c += kStage) {
    const int within = c % kSend, c0 = col0 + c - within;
    if (c0 >= p.n) break;
    if (within == 0) {
      if (lane == 0) bulk_wait_read();      // the previous copy has read the staging rows
      __syncwarp();
    }
    stage_columns<F32, NARROW, kStage>(stage, bias + c, &r[c / 32][c % 32], within / (F32 ? 4 : 8), lane);
    if (within + kStage == kSend) send_columns<F32, NARROW, AHEAD>(stage, map, p.vector_out, p.out, c0, row0, p.m, p.n, lane);
  }
}

// One 128 x BN tile per work item, k stepped by 128 through a TMA ring.  A step that opens a group of four brings the group's exponent tiles
// with it; the MMA thread copies them to tensor memory (four slots in turn) in front of the step's products.  An accumulator
// of 256 columns has no second one beside it and the scales (512 columns in all): the epilogue's warps take their shares into registers with
// one wait and hand it back, so that the next tile's products run under the stores.  Narrower tiles have two.
// Warp roles: 0 = TMA producer, 1 = MMA issuer (owns TMEM), 2.. = epilogue, 64 columns of a lane quadrant each.
// DEEP (256 columns, many channels): three steps on their way leave the tensor core waiting a fifth of its time; a fourth takes the room of the wide staging
// tiles, and the epilogue, which then has a long main loop to hide under, has eight warps of 128 columns and tiles of 64-byte rows.
template <int BN, bool DEEP>
struct Float8Shape {
  static constexpr int stages = DEEP ? 4 : BN == 256 ? 3 : BN == 128 ? 5 : 6;
  static constexpr int b_bytes = BN * F8_BK, stage = F8_A_BYTES + b_bytes;
  static constexpr int b_tiles = (BN + 127) / 128, scales = 512 * (1 + b_tiles);
  static constexpr int accumulators = BN == 256 ? 1 : 2;
  static constexpr int share = DEEP ? 128 : 64, epi = 4 * (BN / share), staging = DEEP ? 2048 : 4096;
  static constexpr int threads = 64 + 32 * epi;
  static constexpr int smem = stages * (stage + scales) + epi * (staging + share * 4) + 256 + 1024;
  static_assert(slots_suffice(stages, accumulators), "");
};

template <int BN, bool F32, bool DEEP>
__global__ void __launch_bounds__(Float8Shape<BN, DEEP>::threads, 1)
float8_linear_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const __grid_constant__ CUtensorMap mapO,
                     const Float8Params p) {
  using S = Float8Shape<BN, DEEP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_shared(smem_raw);
  uint8_t* out_stage = smem + S::stages * S::stage;
  uint8_t* scale_s = out_stage + S::epi * S::staging;
  float* bias_s = reinterpret_cast<float*>(scale_s + S::stages * S::scales);
  uint64_t* bars = reinterpret_cast<uint64_t*>(bias_s + S::epi * S::share);
  uint64_t* full = bars;
  uint64_t* empty = full + S::stages;
  uint64_t* tmem_full = empty + S::stages;
  uint64_t* tmem_empty = tmem_full + S::accumulators;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + S::accumulators);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_m = (p.m + F8_BM - 1) / F8_BM, tiles_n = (p.n + BN - 1) / BN;
  const int total = tiles_m * tiles_n;
  const int kblocks = (p.k + F8_BK - 1) / F8_BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < S::accumulators; ++b) { mbar_init(&tmem_full[b], 1); mbar_init(&tmem_empty[b], S::epi); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  lf_chain();

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tensormap(&mapA);
      prefetch_tensormap(&mapB);
      int stage = 0; uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        const int mi = t / tiles_n, nj = t - mi * tiles_n;
        // exponent tiles of the second 128 columns may not exist
        const int b_tiles = min((int64_t)S::b_tiles, p.ew_tiles - (int64_t)nj * BN / 128);
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.status, 121)) { ok = false; break; }
          uint8_t* sA = smem + stage * S::stage;
          const bool opens = (kb & 3) == 0;
          mbar_expect_tx(&full[stage], S::stage + (opens ? 512 * (1 + b_tiles) : 0));
          tma_load_3d(sA, &mapA, &full[stage], kb * F8_BK, mi * F8_BM, 0);
          tma_load_3d(sA + F8_A_BYTES, &mapB, &full[stage], kb * F8_BK, nj * BN, 0);
          if (opens) {
            uint8_t* sc = scale_s + stage * S::scales;
            bulk_load(sc, p.ex + ((int64_t)(kb >> 2) * p.ex_tiles + mi) * 512, 512, &full[stage]);
            bulk_load(sc + 512, p.ew + ((int64_t)(kb >> 2) * p.ew_tiles + (int64_t)nj * BN / 128) * 512, 512 * b_tiles, &full[stage]);
          }
          if (++stage == S::stages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // The whole warp walks and waits and one lane issues, so that the instructions' operands stay in uniform registers (4096 x 4096 x 4096: 58 us, by one lane's
    // branch 64).
    const uint64_t a_first = make_smem_desc(smem_u32(smem), 16, 1024), b_first = make_smem_desc(smem_u32(smem) + F8_A_BYTES, 16, 1024);
    const uint64_t scale_first = make_smem_desc_plain(smem_u32(scale_s), 0, 128);
    int stage = 0; uint32_t phase = 0, it = 0, group = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x, ++it) {
      const int nj = t % tiles_n;
      const int left = p.n - nj * BN, columns = left >= BN ? BN : (left + 15) / 16 * 16;
      const uint32_t acc = it % S::accumulators;
      if (!__all_sync(0xffffffffu, mbar_wait(&tmem_empty[acc], ((it / S::accumulators) & 1) ^ 1, abort_flag, p.status, 122))) break;
      tc_fence_after();
      const uint32_t d = tmem_base + acc * BN;
      const uint32_t idesc = make_idesc_f8(F8_BM, columns, p.x_format, 0, 0);
      uint32_t scales = 0;
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, abort_flag, p.status, 123))) { ok = false; break; }      // (for all lanes alike)
        tc_fence_after();
        const uint64_t a = a_first + (uint32_t)(stage * S::stage >> 4), b = b_first + (uint32_t)(stage * S::stage >> 4);
        // Slots in turn (see F8_SLOTS): the slot's last reader, four groups back, is done.
        if ((kb & 3) == 0) scales = tmem_base + 256 + (group++ % F8_SLOTS) * 16;
        if (elect_one()) {
          if ((kb & 3) == 0) {
            const uint64_t sc = scale_first + (uint32_t)(stage * S::scales >> 4);
            tmem_copy_scales<1>(scales, sc);
            tmem_copy_scales<1>(scales + 8, sc + 32);
            if (BN == 256 && columns > 128) tmem_copy_scales<1>(scales + 12, sc + 64);
          }
#pragma unroll
          for (int kk = 0; kk < F8_BK / 32; ++kk)
            umma_f8_scaled<1>(d, a + kk * 2, b + kk * 2, idesc | (kb & 3) << 4 | (kb & 3) << 29, scales, scales + 8 + (BN == 64 ? 2u * (nj & 1) : 0u),
                           (kb | kk) != 0 ? 1u : 0u);
          umma_commit(&empty[stage]);
          if (kb + 1 == kblocks) umma_commit(&tmem_full[acc]);
        }
        __syncwarp();
        if (++stage == S::stages) { stage = 0; phase ^= 1; }
      }
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;      // TMEM lane quadrant, 64 of the tile's columns
    uint8_t* stage = out_stage + (warp - 2) * S::staging;
    float* bias = bias_s + (warp - 2) * S::share;
    uint32_t it = 0;
    int held = -1;      // first column of the bias share in shared memory
    if (lane == 0 && p.vector_out) prefetch_tensormap(&mapO);
    for (int t = blockIdx.x; t < total; t += gridDim.x, ++it) {
      const int mi = t / tiles_n, nj = t - mi * tiles_n;
      const int col0 = nj * BN + part * S::share, row0 = mi * F8_BM + q * 32;
      const bool mine = col0 < p.n && row0 < p.m;
      if (mine && held != col0) {
        held = col0;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < S::share; e += 32) bias[e + lane] = p.bias && col0 + e + lane < p.n ? p.bias[col0 + e + lane] : 0.f;
        __syncwarp();
      }
      const uint32_t acc = it % S::accumulators;
      if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], (it / S::accumulators) & 1, abort_flag, p.status, 124))) break;
      tc_fence_after();
      uint32_t r[S::share / 32][32];
      if (mine) {
        const uint32_t d = tmem_base + ((uint32_t)(q * 32) << 16) + acc * BN + part * S::share;
#pragma unroll
        for (int i = 0; i < S::share / 32; ++i) tmem_ld32(d + i * 32, r[i]);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < S::share / 32; ++i) tie32(r[i]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tmem_empty[acc]);      // the share is in registers: the accumulator may be overwritten
      if (!mine) continue;
      send_share<S::share, F32, DEEP, BN == 256 ? 1 : 8>(r, stage, bias, &mapO, p, col0, row0, lane);
    }
    if (lane == 0) bulk_wait_all();      // this thread's stores have landed
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_after_abort();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, 512); }
}

// Tiles of 256 x BN for two multiprocessors (a cluster of two CTAs), for products of many channels.  Of a pair each CTA loads its own 128 rows of x and half of the
// weights' rows, and the pair's MMA reads both halves: at 256 columns 32 KB a step instead of 48, and a step takes 0.33 us instead of 0.38.  192 columns, at 0.29, have two
// accumulators and divide what 256 do not: 5000 x 4096 -> 2048 takes 35 us (256: 41, 256 without pairs: 41), 12000 x 4096 -> 400 25 (29, 29).  4096 x 4096 -> 4096:
// 53.4 us at 256 (192: 55.2, without pairs 55.9), 2570 TFLOP/s, 256 tiles in four turns of 74 pairs.  A pair starts about 1 us later and its accumulator changes hands
// across two CTAs, so few channels have nothing of it.
// Each CTA's producer fills its own shared memory and the leader's barriers count both; the leader's MMA warp multiplies for both and its commits arrive in both.
// Exponents come by TMA like the rest: a CTA needs those of its own rows and of all the tile's outputs.
template <int BN>
struct PairShape {
  static constexpr int stages = 6, stage = F8_A_BYTES + BN / 2 * F8_BK, scales = 512 * 3;
  static constexpr int accumulators = BN == 256 ? 1 : 2, scale_columns = accumulators * BN;      // (and where the scales begin)
  static constexpr int share = BN == 256 ? 128 : 64, epi = 4 * (BN / share), staging = 2048, threads = 64 + 32 * epi;
  static constexpr int smem = stages * (stage + scales) + epi * (staging + share * 4) + 256 + 1024;
  static_assert(slots_suffice(stages, accumulators), "");
};

template <int BN, bool F32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairShape<BN>::threads, 1)
float8_pair_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const __grid_constant__ CUtensorMap mapEx,
                   const __grid_constant__ CUtensorMap mapEw, const __grid_constant__ CUtensorMap mapO, const Float8Params p) {
  using S = PairShape<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_shared(smem_raw);
  uint8_t* out_stage = smem + S::stages * S::stage;
  uint8_t* scale_s = out_stage + S::epi * S::staging;
  float* bias_s = reinterpret_cast<float*>(scale_s + S::stages * S::scales);
  uint64_t* full = reinterpret_cast<uint64_t*>(bias_s + S::epi * S::share);      // [stages] the leader's: both CTAs' loads are here
  uint64_t* empty = full + S::stages;            // [stages] multiplied
  uint64_t* tmem_full = empty + S::stages;
  uint64_t* tmem_empty = tmem_full + S::accumulators;          // the leader's: both CTAs' shares are in registers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + S::accumulators);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = pair_rank();
  const int tiles_m = (p.m + 255) / 256, tiles_n = (p.n + BN - 1) / BN, total = tiles_m * tiles_n;
  const int kblocks = (p.k + F8_BK - 1) / F8_BK;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (threadIdx.x == 32) { prefetch_tensormap(&mapA); prefetch_tensormap(&mapB); prefetch_tensormap(&mapEx); prefetch_tensormap(&mapEw); }
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < S::accumulators; ++b) { mbar_init(&tmem_full[b], 1); mbar_init(&tmem_empty[b], 2 * S::epi); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  pair_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  lf_chain();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0; uint32_t phase = 0;
      bool ok = true;
      for (int t = first; t < total && ok; t += step) {
        const int mi = t / tiles_n, nj = t - mi * tiles_n;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait_cluster(&empty[stage], phase ^ 1, abort_flag, p.status, 141)) { ok = false; break; }
          const bool opens = (kb & 3) == 0;
          if (rank == 0) mbar_expect_tx(&full[stage], 2 * (S::stage + (opens ? S::scales : 0)));
          const uint32_t bar = leader_bar(&full[stage]);
          uint8_t* sA = smem + stage * S::stage;
          tma_load_3d_pair(sA, &mapA, bar, kb * F8_BK, mi * 256 + (int)rank * 128, 0);
          tma_load_3d_pair(sA + F8_A_BYTES, &mapB, bar, kb * F8_BK, nj * BN + (int)rank * (BN / 2), 0);
          if (opens) {      // (tiles that do not exist: other rows' bytes or zeros, for rows and outputs that are not stored)
            uint8_t* sc = scale_s + stage * S::scales;
            tma_load_3d_pair(sc, &mapEx, bar, 0, (int)((kb >> 2) * p.ex_tiles) + mi * 2 + (int)rank, 0);
            tma_load_3d_pair(sc + 512, &mapEw, bar, 0, (int)((kb >> 2) * p.ew_tiles) + nj * BN / 128, 0);
          }
          if (++stage == S::stages) { stage = 0; phase ^= 1; }
        }
      }
      // the leader's arrivals have landed before this CTA may end
      for (int s = 0; s < S::stages && ok; ++s) {
        ok = mbar_wait_cluster(&empty[stage], phase ^ 1, abort_flag, p.status, 145);
        if (++stage == S::stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint64_t a_first = make_smem_desc(smem_u32(smem), 16, 1024), b_first = make_smem_desc(smem_u32(smem) + F8_A_BYTES, 16, 1024);
      const uint64_t scale_first = make_smem_desc_plain(smem_u32(scale_s), 0, 128);
      const uint32_t idesc = make_idesc_f8(256, BN, p.x_format, 0, 0);
      int stage = 0; uint32_t phase = 0, it = 0, group = 0;
      bool ok = true;
      for (int t = first; t < total && ok; t += step, ++it) {
        const uint32_t acc = it % S::accumulators, within = t % tiles_n * BN & 127;      // (the tile's first output in its 128 exponents)
        if (!__all_sync(0xffffffffu, mbar_wait_cluster(&tmem_empty[acc], ((it / S::accumulators) & 1) ^ 1, abort_flag, p.status, 142))) break;
        tc_fence_after();
        uint32_t scales = 0;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait_cluster(&full[stage], phase, abort_flag, p.status, 143))) { ok = false; break; }
          tc_fence_after();
          const uint64_t a = a_first + (uint32_t)(stage * S::stage >> 4), b = b_first + (uint32_t)(stage * S::stage >> 4);
          if ((kb & 3) == 0) scales = tmem_base + S::scale_columns + (group++ % F8_SLOTS) * 16;      // (as above)
          if (elect_one()) {
            if ((kb & 3) == 0) {
              const uint64_t sc = scale_first + (uint32_t)(stage * S::scales >> 4);
              tmem_copy_scales<2>(scales, sc);
              tmem_copy_scales<2>(scales + 8, sc + 32);
              tmem_copy_scales<2>(scales + 12, sc + 64);
            }
#pragma unroll
            for (int kk = 0; kk < F8_BK / 32; ++kk)
              umma_f8_scaled<2>(tmem_base + acc * BN, a + kk * 2, b + kk * 2, idesc | (kb & 3) << 4 | (kb & 3) << 29, scales, scales + 8 + within / 32,
                                (kb | kk) != 0 ? 1u : 0u);
            umma_commit_pair(&empty[stage]);
            if (kb + 1 == kblocks) umma_commit_pair(&tmem_full[acc]);
          }
          __syncwarp();
          if (++stage == S::stages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;      // TMEM lane quadrant, share of the tile's columns
    uint8_t* stage = out_stage + (warp - 2) * S::staging;
    float* bias = bias_s + (warp - 2) * S::share;
    uint32_t it = 0;
    int held = -1;      // first column of the bias share in shared memory
    if (lane == 0 && p.vector_out) prefetch_tensormap(&mapO);
    for (int t = first; t < total; t += step, ++it) {
      const int mi = t / tiles_n, nj = t - mi * tiles_n;
      const int col0 = nj * BN + part * S::share, row0 = mi * 256 + (int)rank * 128 + q * 32;
      const bool mine = col0 < p.n && row0 < p.m;
      if (mine && held != col0) {
        held = col0;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < S::share; e += 32) bias[e + lane] = p.bias && col0 + e + lane < p.n ? p.bias[col0 + e + lane] : 0.f;
        __syncwarp();
      }
      const uint32_t acc = it % S::accumulators;
      if (!__all_sync(0xffffffffu, mbar_wait_cluster(&tmem_full[acc], (it / S::accumulators) & 1, abort_flag, p.status, 144))) break;
      tc_fence_after();
      uint32_t r[S::share / 32][32];
      if (mine) {
        const uint32_t d = tmem_base + ((uint32_t)(q * 32) << 16) + acc * BN + part * S::share;
#pragma unroll
        for (int i = 0; i < S::share / 32; ++i) tmem_ld32(d + i * 32, r[i]);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < S::share / 32; ++i) tie32(r[i]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(leader_bar(&tmem_empty[acc]));
      if (mine) send_share<S::share, F32, true, 1>(r, stage, bias, &mapO, p, col0, row0, lane);
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_after_abort();
  __syncwarp();
  pair_sync();      // neither CTA's memory goes before both are through
  if (warp == 1) { tc_fence_after(); tmem_dealloc_pair(tmem_base, 512); }
}

// f(BN, F32, DEEP as types)
template <typename F>
static void linear_forms(int bn, bool deep, bool f32, F f) {
  auto with = [&](auto b) { if (f32) f(b, std::true_type{}, std::false_type{}); else f(b, std::false_type{}, std::false_type{}); };
  if (deep) { if (f32) f(std::integral_constant<int, 256>{}, std::true_type{}, std::true_type{}); else f(std::integral_constant<int, 256>{}, std::false_type{}, std::true_type{}); }
  else if (bn == 256) with(std::integral_constant<int, 256>{});
  else if (bn == 128) with(std::integral_constant<int, 128>{});
  else with(std::integral_constant<int, 64>{});
}

// f(BN, F32 as types)
template <typename F>
static void pair_forms(int bn, bool f32, F f) {
  auto with = [&](auto b) { if (f32) f(b, std::true_type{}); else f(b, std::false_type{}); };
  if (bn == 256) with(std::integral_constant<int, 256>{}); else with(std::integral_constant<int, 192>{});
}

void configure_float8_linear() {
  for (int i = 0; i < 8; ++i)
    linear_forms(64 << i % 4, i % 4 == 3, i / 4, [](auto bn, auto f32, auto deep) {
      constexpr int BN = decltype(bn)::value;
      constexpr bool D = decltype(deep)::value;
      cudaFuncSetAttribute(float8_linear_kernel<BN, decltype(f32)::value, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Float8Shape<BN, D>::smem);
    });
  for (int i = 0; i < 4; ++i)
    pair_forms(i & 1 ? 256 : 192, i >> 1, [](auto bn, auto f32) {
      constexpr int BN = decltype(bn)::value;
      cudaFuncSetAttribute(float8_pair_kernel<BN, decltype(f32)::value>, cudaFuncAttributeMaxDynamicSharedMemorySize, PairShape<BN>::smem);
    });
  configure_float8_few();
}

template <int BN, bool F32>
static lf_status launch_pair(lf_context* ctx, const f8::Matrix& x, const f8::Matrix& w, const Float8Params& p) {
  using S = PairShape<BN>;
  CUtensorMap ma, mb, mex, mew, mo{};
  LF_TRY(make_map_bytes(ctx, &ma, x.codes, x.channels, x.rows, x.pitch, 128));
  LF_TRY(make_map_bytes(ctx, &mb, w.codes, w.channels, w.rows, w.pitch, BN / 2));
  const int groups = (f8::blocks(p.k) + 3) / 4;
  LF_TRY(make_map_tiles(ctx, &mex, x.exponents, groups * x.tiles, 1));
  LF_TRY(make_map_tiles(ctx, &mew, w.exponents, groups * w.tiles, 2));
  if (p.vector_out) LF_TRY(make_map_rows(ctx, &mo, p.out, F32, p.n, p.m, 32, true));
  const int64_t tiles = (int64_t)((p.m + 255) / 256) * ((p.n + BN - 1) / BN), pairs = ctx->sm_count / 2;
  lf_prof_begin(ctx, LF_KERNEL_LN_GEMM);
  lf_launch(ctx, float8_pair_kernel<BN, F32>, 2 * (int)(tiles < pairs ? tiles : pairs), S::threads, S::smem, ma, mb, mex, mew, mo, p);
  lf_prof_end(ctx);
  ctx->launches++;
  return LF_OK;
}

template <int BN, bool F32, bool DEEP>
static lf_status launch_float8(lf_context* ctx, const f8::Matrix& x, const f8::Matrix& w, Float8Params p) {
  using S = Float8Shape<BN, DEEP>;
  CUtensorMap ma, mb, mo{};
  LF_TRY(make_map_bytes(ctx, &ma, x.codes, x.channels, x.rows, x.pitch, F8_BM));
  LF_TRY(make_map_bytes(ctx, &mb, w.codes, w.channels, w.rows, w.pitch, BN));
  if (p.vector_out) LF_TRY(make_map_rows(ctx, &mo, p.out, F32, p.n, p.m, 32, DEEP));
  const int64_t tiles = (int64_t)((p.m + F8_BM - 1) / F8_BM) * ((p.n + BN - 1) / BN);
  lf_prof_begin(ctx, LF_KERNEL_LN_GEMM);
  lf_launch(ctx, float8_linear_kernel<BN, F32, DEEP>, (int)(tiles < ctx->sm_count ? tiles : ctx->sm_count), S::threads, S::smem, ma, mb, mo, p);
  lf_prof_end(ctx);
  ctx->launches++;
  return LF_OK;
}

// What the forms take, in nanoseconds: at the start, for a turn, and for a step of a turn; a turn more where rows are float32, or odd (stored by threads).  Least squares over
// 172 products of 100 to 65536 rows, 40 to 4096 channels and 100 to 4096 outputs, each timed in every form: the form that they choose is 0.7 % slower than the
// fastest on average and 15 % at most.  (A rule on widths and turns alone was 7.7 % slower, 88 % at most; without pairs 3.6 %.)
struct FormCost { int ctas, bn; bool deep; int start, turn, step, turn_f32, odd_start, odd_turn; };
constexpr FormCost kForms[] = {
    {1, 64, false, 3100, 500, 264, 360, 0, 1100},    {1, 128, false, 3200, 630, 305, 570, 0, 1700},
    {1, 256, false, 4050, 1230, 349, 1120, 1100, 3230}, {1, 256, true, 3300, 1010, 362, 1940, 5000, 4300},      // DEEP: from F8_DEEP channels on
    {2, 192, false, 4000, 1720, 247, 1210, 2100, 2660}, {2, 256, false, 3900, 2230, 301, 1610, 3250, 4400},
};

}  // namespace tc

using namespace f8;

// Which kernel takes a product: few rows one launch that reads the weights at full width (4 x 1536 -> 384: 4.2 us; encoder and tiled product 2.2 + 6.7), else
// the encoder, then the tiled product.  (One kernel that encoded its rows on the way into the tiled product was slower than the two: with registers for 16
// encoding warps a multiprocessor hides too little of their latency, 147456 x 128 -> 512 took 40 us or more.)
extern "C" uint64_t lf_float8_linear_workspace(int64_t rows, int32_t channels) {
  if (rows <= 0 || channels <= 0 || tc::float8_few_takes(rows, channels)) return 0;
  return lf_float8_code_bytes(rows, channels) + lf_float8_exponent_bytes(rows, channels);
}

extern "C" lf_status lf_float8_linear_run(lf_context* ctx, const lf_float8_linear_desc* d, lf_result* r) {
  if (!ctx) return LF_ERR_ARGUMENT;
  if (!d || !d->out) return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 linear: null argument");
  const lf_float8_matrix &x = d->activations, &w = d->weights;
  LF_TRY(lf_float8_check_rows(ctx, "float8 linear", x.rows, x.channels, d->out_dtype));
  LF_TRY(lf_float8_check_rows(ctx, "float8 linear", w.rows, x.channels, d->out_dtype));
  LF_TRY(lf_float8_check(ctx, "float8 linear, weights", w, w.rows, x.channels));
  if (d->source && d->source_dtype != LF_DTYPE_F32 && d->source_dtype != LF_DTYPE_BF16) return lf_fail(ctx, LF_ERR_ARGUMENT, "unknown source dtype %d", d->source_dtype);
  if (w.format != LF_FLOAT8_E4M3) return lf_fail(ctx, LF_ERR_UNSUPPORTED, "float8 linear: weights are e4m3");
  if (w.rows > (1 << 24)) return lf_fail(ctx, LF_ERR_UNSUPPORTED, "float8 linear: %lld output channels are too many", (long long)w.rows);
  if (row_tiles(x.rows) * ((w.rows + 63) / 64) > 0x7fffffffll) return lf_fail(ctx, LF_ERR_UNSUPPORTED, "float8 linear: %lld x %lld outputs are too many", (long long)x.rows, (long long)w.rows);
  Matrix mx = matrix(x);
  const Matrix mw = matrix(w);
  const bool kept = x.codes != nullptr;
  if (kept || !d->source) LF_TRY(lf_float8_check(ctx, "float8 linear, activations", x, x.rows, x.channels));
  else if (x.format != LF_FLOAT8_E4M3 && x.format != LF_FLOAT8_E5M2) return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 linear: unknown 8-bit format %d", x.format);
  const uint64_t need = d->source && !kept ? lf_float8_linear_workspace(x.rows, x.channels) : 0;
  if (need && (!d->workspace || d->workspace_bytes < need || !lf_aligned16(d->workspace)))
    return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 linear: a workspace of %llu bytes on a 16-byte boundary is needed", (unsigned long long)need);
  const uint64_t out_bytes = (uint64_t)x.rows * w.rows * (d->out_dtype == LF_DTYPE_BF16 ? 2 : 4);
  if (d->source)
    LF_TRY(lf_float8_apart(ctx, "float8 linear", d->out, out_bytes, d->source, (uint64_t)x.rows * x.channels * (d->source_dtype == LF_DTYPE_BF16 ? 2 : 4)));
  LF_TRY(lf_float8_apart(ctx, "float8 linear", d->out, out_bytes, x));
  LF_TRY(lf_float8_apart(ctx, "float8 linear", d->out, out_bytes, w));
  if (d->bias) LF_TRY(lf_float8_apart(ctx, "float8 linear", d->out, out_bytes, d->bias, (uint64_t)w.rows * 4));
  if (need) LF_TRY(lf_float8_apart(ctx, "float8 linear", d->out, out_bytes, d->workspace, need));
  const lf_device_guard device(ctx);
  if (tc::float8_few_takes(x.rows, x.channels)) {
    LF_TRY(tc::float8_few(ctx, d->source, d->source ? d->source_dtype : LF_DTYPE_F32, mx, mw, d->bias, d->out, d->out_dtype));
    return lf_float8_done(ctx, r, 1);
  }
  const bool f32 = d->out_dtype == LF_DTYPE_F32;
  const int vector_out = lf_aligned16(d->out) && w.rows % (f32 ? 4 : 8) == 0;
  int launches = 1;
  if (d->source) {
    lf_float8_encode_desc e{};
    e.out = x; e.dtype = d->source_dtype; e.block_rows = 1; e.source = d->source;
    if (!kept) {
      e.out.codes = d->workspace;
      e.out.exponents = (char*)d->workspace + lf_float8_code_bytes(x.rows, x.channels);
    }
    LF_TRY(lf_float8_encode(ctx, &e, nullptr));
    mx = matrix(e.out);
    ++launches;
  }
  tc::Float8Params p{};
  p.m = (int)x.rows; p.n = (int)w.rows; p.k = x.channels;
  p.vector_out = vector_out;
  p.bias = d->bias; p.ex = mx.exponents; p.ew = mw.exponents; p.ex_tiles = mx.tiles; p.ew_tiles = mw.tiles;
  p.x_format = x.format;
  p.out = d->out;
  p.status = (tc05::Status*)ctx->tc_status;
  // The form that is done first.  Which that is depends on the turns (tiles over multiprocessors or pairs) and the steps of 128 channels.
  const int64_t steps = (p.k + tc::F8_BK - 1) / tc::F8_BK;
  const tc::FormCost* form = nullptr;
  int64_t best = 0;
  for (const tc::FormCost& f : tc::kForms) {
    if (f.bn == 256 && f.ctas == 1 && f.deep != (p.k >= tc::F8_DEEP)) continue;
    const int64_t tiles = (mx.tiles + f.ctas - 1) / f.ctas * ((p.n + f.bn - 1) / f.bn), at_once = ctx->sm_count / f.ctas, turns = (tiles + at_once - 1) / at_once;
    const int64_t cost = f.start + (vector_out ? 0 : f.odd_start) + turns * (f.turn + steps * f.step + (f32 ? f.turn_f32 : 0) + (vector_out ? 0 : f.odd_turn));
    if (!form || cost < best) { form = &f; best = cost; }
  }
  lf_status status = LF_OK;
  if (form->ctas == 2) tc::pair_forms(form->bn, f32, [&](auto b, auto o) { status = tc::launch_pair<decltype(b)::value, decltype(o)::value>(ctx, mx, mw, p); });
  else
    tc::linear_forms(form->bn, form->deep, f32, [&](auto b, auto o, auto deep) {
      status = tc::launch_float8<decltype(b)::value, decltype(o)::value, decltype(deep)::value>(ctx, mx, mw, p);
    });
  LF_TRY(status);
  return lf_float8_done(ctx, r, launches);
}
