// To and from the 8-bit form of a matrix (float8.cuh): activations with an exponent for every 128 channels of a row, weights with one
// for every 128 x 128 elements, both orientations in one pass.
//
// Each element is read and written once and needs a handful of instructions: memory bounds these kernels.  A lane has sixteen neighbouring
// channels, eight lanes a block of 128 (narrow rows: four lanes for at most 64 channels), so that the block's largest magnitude takes
// three shuffles and all accesses are 16 or 32 bytes; every lane keeps kUnits blocks in flight.  1 Mi x 128 in bf16: 61 us to codes, 60 back, 6.6 and 6.8 TB/s.
#include "float8.cuh"

namespace f8 {

constexpr int kThreads = 256, kUnits = 2;

template <typename T, int LANES, bool ELEMENTS>
__global__ void __launch_bounds__(kThreads)
encode_kernel(const T* x, const Matrix m, uint32_t units, uint32_t per_row, int how) {
  const int access = ELEMENTS ? (int)kElements : max(how, (int)kSixteen);
  const int lane = threadIdx.x % LANES;
  const uint32_t base = blockIdx.x * (uint32_t)(kThreads / LANES * kUnits) + threadIdx.x / LANES;
  __shared__ __align__(16) float rooms[ELEMENTS ? kThreads / 32 : 1][ELEMENTS ? kRoom : 4];
  float* room = rooms[ELEMENTS ? threadIdx.x >> 5 : 0];
  lf_chain();
  Raw<T> raw[kUnits];
  uint32_t row[kUnits], first[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const uint32_t unit = base + u * (kThreads / LANES);
    row[u] = per_row == 1 ? unit : unit / per_row;
    first[u] = (unit - row[u] * per_row) * kBlock + lane * kShare;
    load16<T, LANES>(raw[u], x + (int64_t)row[u] * m.channels + first[u], m.channels - (int)first[u], unit < units, access);
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    uint4 codes;
    const int s = encode16<LANES>(unpack<T, LANES>(raw[u], access, room), m.format, codes);
    if (base + u * (kThreads / LANES) < units) put16(m, row[u], first[u], codes, s);
  }
}

template <typename T, int LANES, bool ELEMENTS>
__global__ void __launch_bounds__(kThreads)
decode_kernel(const Matrix m, T* out, uint32_t units, uint32_t per_row, int how) {
  const int access = ELEMENTS ? (int)kElements : max(how, (int)kSixteen);
  const int lane = threadIdx.x % LANES;
  const uint32_t base = blockIdx.x * (uint32_t)(kThreads / LANES * kUnits) + threadIdx.x / LANES;
  __shared__ __align__(16) float rooms[ELEMENTS ? kThreads / 32 : 1][ELEMENTS ? kRoom : 4];
  float* room = rooms[ELEMENTS ? threadIdx.x >> 5 : 0];
  lf_chain();
  uint4 codes[kUnits];
  int s[kUnits];
  uint32_t row[kUnits], first[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const uint32_t unit = base + u * (kThreads / LANES);
    row[u] = per_row == 1 ? unit : unit / per_row;
    const uint32_t block = unit - row[u] * per_row;
    first[u] = block * kBlock + lane * kShare;
    codes[u] = make_uint4(0, 0, 0, 0);
    s[u] = 1;
    if (unit < units && first[u] < (uint32_t)m.channels) {
      codes[u] = *reinterpret_cast<const uint4*>(m.codes + row[u] * m.pitch + first[u]);
      s[u] = m.exponents[exponent_at(row[u], block, m.tiles)];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    Share v = decode16(codes[u], m.format);
    const float2 factor = both(up(s[u]));
#pragma unroll
    for (int i = 0; i < kShare / 2; ++i) v.v[i] = mul2(v.v[i], factor);
    store16<T, LANES>(out + (int64_t)row[u] * m.channels + first[u], m.channels - (int)first[u], base + u * (kThreads / LANES) < units, access, v, room);
  }
}

// One 128 x 128 block a block of threads: its largest magnitude, its codes in rows, and (t.codes set) the same codes with rows and
// channels exchanged - the exponent is the block's, so the transposed matrix stands for the same values.
// (1024 threads of sixteen elements: 512 x 128 took 5.8 us with 256 of 64.  Element by element 512, for what their rooms take of shared memory.)
__host__ __device__ constexpr int square_threads(bool elements) { return elements ? 512 : 1024; }
template <typename T, bool ELEMENTS>
__global__ void __launch_bounds__(square_threads(ELEMENTS))
encode_square_kernel(const T* x, const Matrix m, const Matrix t, int how) {
  constexpr int kSquareThreads = square_threads(ELEMENTS), kTurned = kBlock * kBlock, kRooms = ELEMENTS ? kSquareThreads / 32 * kRoom * 4 : 0;
  const int access = ELEMENTS ? (int)kElements : max(how, (int)kSixteen);
  __shared__ __align__(16) uint8_t shared_s[kTurned > kRooms ? kTurned : kRooms];      // the warps' rooms, then the codes on their way to the other orientation
  __shared__ float most_s[2][kSquareThreads / 32];
  // (channel ch's byte of row r; pieces of sixteen rows are exchanged by the channel, so that eight lanes' bytes lie in different banks)
  auto turned_at = [&](int ch, int r) { return shared_s + ch * kBlock + (r ^ (ch & 0x70)); };
  constexpr int kRows = kBlock * 8 / kSquareThreads;      // of a thread
  float* room = reinterpret_cast<float*>(shared_s) + (ELEMENTS ? threadIdx.x >> 5 : 0) * kRoom;
  const int lane = threadIdx.x & 7, strand = threadIdx.x >> 3;
  const int64_t row0 = (int64_t)blockIdx.y * kBlock;
  const int first = blockIdx.x * kBlock + lane * kShare;
  lf_chain();
  Raw<T> raw[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const int64_t row = row0 + strand + kSquareThreads / 8 * k;
    load16<T, 8>(raw[k], x + row * m.channels + first, m.channels - first, row < m.rows, access);
  }
  float most = 0.f, finite = 0.f;
  Share v[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    v[k] = unpack<T, 8>(raw[k], access, room);
    most = fmaxf(most, most_of(v[k]));
    finite = fmaxf(finite, most_finite_of(v[k]));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) { most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o)); finite = fmaxf(finite, __shfl_xor_sync(0xffffffffu, finite, o)); }
  if ((threadIdx.x & 31) == 0) { most_s[0][threadIdx.x >> 5] = most; most_s[1][threadIdx.x >> 5] = finite; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSquareThreads / 32; ++w) { most = fmaxf(most, most_s[0][w]); finite = fmaxf(finite, most_s[1][w]); }
  const int s = exponent_byte(__float_as_uint(finite), m.format);
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const int64_t row = row0 + strand + kSquareThreads / 8 * k;
    const uint4 codes = code16(v[k], s, m.format, most == kInfinity);
    if (row < m.rows && first < m.channels) *reinterpret_cast<uint4*>(m.codes + row * m.pitch + first) = codes;
    if (t.codes) {
      const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
      for (int i = 0; i < kShare; ++i) *turned_at(lane * kShare + i, strand + kSquareThreads / 8 * k) = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
  }
  if (threadIdx.x < kBlock) m.exponents[exponent_at(row0 + threadIdx.x, blockIdx.x, m.tiles)] = (uint8_t)s;
  if (!t.codes) return;
  __syncthreads();
  const int64_t trow0 = (int64_t)blockIdx.x * kBlock;
  const int tfirst = blockIdx.y * kBlock + lane * kShare;
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const int64_t row = trow0 + strand + kSquareThreads / 8 * k;
    if (row < t.rows && tfirst < t.channels)
      *reinterpret_cast<uint4*>(t.codes + row * t.pitch + tfirst) = *reinterpret_cast<const uint4*>(turned_at(strand + kSquareThreads / 8 * k, lane * kShare));
  }
  if (threadIdx.x < kBlock) t.exponents[exponent_at(trow0 + threadIdx.x, blockIdx.y, t.tiles)] = (uint8_t)s;
}

// f(T, LANES, ELEMENTS as types)
template <typename F>
static void row_forms(int dtype, int channels, int access, F f) {
  auto last = [&](auto t, auto lanes) { if (access == kElements) f(t, lanes, std::true_type{}); else f(t, lanes, std::false_type{}); };
  auto with = [&](auto t) { if (channels <= 64) last(t, std::integral_constant<int, 4>{}); else last(t, std::integral_constant<int, 8>{}); };
  if (dtype == LF_DTYPE_BF16) with(bf16{}); else with(float{});
}

}  // namespace f8

using namespace f8;

lf_status lf_float8_check_rows(lf_context* ctx, const char* what, int64_t rows, int channels, int dtype) {
  if (rows <= 0 || channels <= 0) return lf_fail(ctx, LF_ERR_SHAPE, "%s: rows and channels must be positive safe integers", what);
  if (rows > 0x7fffff00 || channels > (1 << 24) || (uint64_t)rows * blocks(channels) > 0x7fffffffull)
    return lf_fail(ctx, LF_ERR_UNSUPPORTED, "%s: %lld rows of %d channels are too many", what, (long long)rows, channels);
  if (dtype != LF_DTYPE_F32 && dtype != LF_DTYPE_BF16) return lf_fail(ctx, LF_ERR_ARGUMENT, "unknown activation dtype %d", dtype);
  return LF_OK;
}

lf_status lf_float8_check(lf_context* ctx, const char* what, const lf_float8_matrix& m, int64_t rows, int channels) {
  if (!m.codes || !m.exponents) return lf_fail(ctx, LF_ERR_ARGUMENT, "%s: null codes or exponents", what);
  if (m.rows != rows || m.channels != channels)
    return lf_fail(ctx, LF_ERR_SHAPE, "%s: an 8-bit matrix of %lld x %d; expected %lld x %d", what, (long long)m.rows, m.channels, (long long)rows, channels);
  if (m.format != LF_FLOAT8_E4M3 && m.format != LF_FLOAT8_E5M2) return lf_fail(ctx, LF_ERR_ARGUMENT, "%s: unknown 8-bit format %d", what, m.format);
  if (!lf_aligned16(m.codes) || !lf_aligned16(m.exponents))
    return lf_fail(ctx, LF_ERR_ARGUMENT, "%s: codes and exponents must start on 16-byte boundaries", what);
  return LF_OK;
}

lf_status lf_float8_apart(lf_context* ctx, const char* what, const void* out, uint64_t bytes, const void* operand, uint64_t operand_bytes) {
  const uintptr_t a = (uintptr_t)out, b = (uintptr_t)operand;
  if (a && b && a < b + operand_bytes && b < a + bytes) return lf_fail(ctx, LF_ERR_ARGUMENT, "%s: the output overlaps an operand", what);
  return LF_OK;
}
lf_status lf_float8_apart(lf_context* ctx, const char* what, const void* out, uint64_t bytes, const lf_float8_matrix& m) {
  if (!m.codes) return LF_OK;
  LF_TRY(lf_float8_apart(ctx, what, out, bytes, m.codes, lf_float8_code_bytes(m.rows, m.channels)));
  return lf_float8_apart(ctx, what, out, bytes, m.exponents, lf_float8_exponent_bytes(m.rows, m.channels));
}

lf_status lf_float8_done(lf_context* ctx, lf_result* r, int launches) {
  LF_CUDA(ctx, cudaGetLastError());
  if (r) { r->elapsed_ms = 0.f; r->peak_bytes = ctx->arena_peak; r->launches = (uint32_t)launches; }
  return LF_OK;
}

extern "C" {

uint64_t lf_float8_code_bytes(int64_t rows, int32_t channels) { return rows > 0 && channels > 0 ? (uint64_t)(rows * pitch(channels)) : 0; }
uint64_t lf_float8_exponent_bytes(int64_t rows, int32_t channels) { return rows > 0 && channels > 0 ? (uint64_t)exponent_bytes(rows, channels) : 0; }

lf_status lf_float8_encode(lf_context* ctx, const lf_float8_encode_desc* d, lf_result* r) {
  if (!ctx) return LF_ERR_ARGUMENT;
  if (!d || !d->source) return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 encode: null argument");
  const lf_float8_matrix& o = d->out;
  LF_TRY(lf_float8_check_rows(ctx, "float8 encode", o.rows, o.channels, d->dtype));
  LF_TRY(lf_float8_check(ctx, "float8 encode", o, o.rows, o.channels));
  if (d->block_rows != 1 && d->block_rows != kBlock) return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 encode: an exponent covers 1 or 128 rows; received %d", d->block_rows);
  const bool turned = d->transposed.codes != nullptr;
  if (turned && d->block_rows != kBlock) return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 encode: only blocks of 128 rows have a transposed form");
  if (turned) {
    if (o.rows > (1 << 24)) return lf_fail(ctx, LF_ERR_UNSUPPORTED, "float8 encode: %lld rows are too many for a transposed form", (long long)o.rows);
    LF_TRY(lf_float8_check(ctx, "float8 encode, transposed", d->transposed, o.channels, (int)o.rows));
    if (d->transposed.format != o.format) return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 encode: both forms have one format");
  }
  if (d->block_rows == kBlock && row_tiles(o.rows) > 65535) return lf_fail(ctx, LF_ERR_UNSUPPORTED, "float8 encode: %lld rows are too many for blocks of 128 rows", (long long)o.rows);
  const lf_device_guard device(ctx);
  const Matrix m = matrix(o);
  const int access = row_access(d->source, o.channels, d->dtype);
  lf_prof_begin(ctx, LF_KERNEL_ELEMENTWISE);
  if (d->block_rows == kBlock) {
    Matrix t8{};
    if (turned) t8 = matrix(d->transposed);
    const dim3 grid(blocks(o.channels), (unsigned)row_tiles(o.rows));
    auto run = [&](auto t, auto elements) {
      typedef decltype(t) T;
      constexpr bool E = decltype(elements)::value;
      lf_launch(ctx, encode_square_kernel<T, E>, grid, square_threads(E), 0, (const T*)d->source, m, t8, access);
    };
    auto typed = [&](auto t) { if (access == kElements) run(t, std::true_type{}); else run(t, std::false_type{}); };
    if (d->dtype == LF_DTYPE_BF16) typed(bf16{}); else typed(float{});
  } else {
    const uint32_t per_row = blocks(o.channels), units = (uint32_t)(o.rows * per_row);
    row_forms(d->dtype, o.channels, access, [&](auto t, auto lanes, auto elements) {
      typedef decltype(t) T;
      constexpr int L = decltype(lanes)::value;
      lf_launch(ctx, encode_kernel<T, L, decltype(elements)::value>, lf_ceil_div(units, kThreads / L * kUnits), kThreads, 0, (const T*)d->source, m, units, per_row, access);
    });
  }
  lf_prof_end(ctx);
  ctx->launches++;
  return lf_float8_done(ctx, r, 1);
}

lf_status lf_float8_decode(lf_context* ctx, const lf_float8_decode_desc* d, lf_result* r) {
  if (!ctx) return LF_ERR_ARGUMENT;
  if (!d || !d->out) return lf_fail(ctx, LF_ERR_ARGUMENT, "float8 decode: null argument");
  const lf_float8_matrix& o = d->source;
  LF_TRY(lf_float8_check_rows(ctx, "float8 decode", o.rows, o.channels, d->dtype));
  LF_TRY(lf_float8_check(ctx, "float8 decode", o, o.rows, o.channels));
  LF_TRY(lf_float8_apart(ctx, "float8 decode", d->out, (uint64_t)o.rows * o.channels * (d->dtype == LF_DTYPE_BF16 ? 2 : 4), o));
  const lf_device_guard device(ctx);
  const Matrix m = matrix(o);
  const int access = row_access(d->out, o.channels, d->dtype);
  const uint32_t per_row = blocks(o.channels), units = (uint32_t)(o.rows * per_row);
  lf_prof_begin(ctx, LF_KERNEL_ELEMENTWISE);
  row_forms(d->dtype, o.channels, access, [&](auto t, auto lanes, auto elements) {
    typedef decltype(t) T;
    constexpr int L = decltype(lanes)::value;
    lf_launch(ctx, decode_kernel<T, L, decltype(elements)::value>, lf_ceil_div(units, kThreads / L * kUnits), kThreads, 0, m, (T*)d->out, units, per_row, access);
  });
  lf_prof_end(ctx);
  ctx->launches++;
  return lf_float8_done(ctx, r, 1);
}

}  // extern "C"
