// Narrowing to e4m3 with a scale per block of 128 values of the contraction: 1 x 128 groups of a row (activations) or 128 x 128
// tiles (weights).
//
//   scale = max(max |x| / 448, 2^-126), 1 for a block of zeros, or that rounded up to a power of two;   q = e4m3(x * (1 / scale))
//
// the quotient, the reciprocal and the product rounded to nearest in f32.  NaN counts for nothing in the maximum and stays NaN; a
// block with an infinity has an infinite scale, and its infinities come out as NaN.  (2^-126 keeps the reciprocal finite.)
//
// One pass: a block is read once, kept in registers between its maximum and its narrowing, and written once, so that DRAM bounds both
// kernels.
#include "common.cuh"

namespace qb {

// 8 consecutive values as loaded: one 16-byte vector of bf16, two of f32.  kStream: they are read once and need no place in the caches.
template <bool F32, bool kStream = false>
struct Vec8 {
  uint4 w[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* base, size_t at) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + at * (F32 ? 4 : 2));
    w[0] = kStream ? __ldcs(p) : p[0];
    if (F32) w[F32 ? 1 : 0] = kStream ? __ldcs(p + 1) : p[1];
  }
  __device__ __forceinline__ void zero() {
    w[0] = make_uint4(0u, 0u, 0u, 0u);
    w[F32 ? 1 : 0] = w[0];
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    const uint32_t a[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
    if (F32) {
      const uint4& y = w[F32 ? 1 : 0];
      const uint32_t b[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = __uint_as_float(a[j]);
        v[4 + j] = __uint_as_float(b[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = bf16lo(a[j]);
        v[2 * j + 1] = bf16hi(a[j]);
      }
    }
  }
  __device__ __forceinline__ float top() const {
    float v[8];
    values(v);
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));  // (the operand that is not NaN)
    return m;
  }
  __device__ __forceinline__ uint2 narrow(float inv) const {
    float v[8];
    values(v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], inv);
    return make_uint2(pack_e4m3x4(v[0], v[1], v[2], v[3]), pack_e4m3x4(v[4], v[5], v[6], v[7]));
  }
};

// 1 x 128 groups: 8 lanes to a group, 16 values each, so that the scale is worked out by few lanes and a lane stores 16 bytes.  8192 x 8192
// bf16: 42.4 us with 16 lanes to a group and four groups to a thread, 33.4 with 8 and two, 31.7 - 32.5 (6.3 TB/s) with one; f32 49.2 (6.8 TB/s).
template <bool F32>
__global__ void __launch_bounds__(256) quantize_groups_kernel(const void* X, const int* row_index, uint8_t* out, float* scale_out, int units, int kb_total, int rows,
                                                               int src_rows, int cols, int pow2) {
  grid_dep_wait();
  grid_dep_launch();
  X = after_wait(X);
  const int l = threadIdx.x & 7, u = blockIdx.x * 32 + (threadIdx.x >> 3);
  const int row = u / kb_total, kb = u - row * kb_total, c = kb * 128 + l * 16;
  bool live = u < units;
  int from = row;
  if (live && row_index != nullptr) {
    from = after_wait(row_index)[row];
    live = from >= 0 && from < src_rows;
  }
  Vec8<F32> x[2];
  x[0].zero();
  x[1].zero();
  if (live && c < cols) {  // (a multiple of 16 columns)
    const size_t at = static_cast<size_t>(from) * cols + c;
    x[0].load(X, at);
    x[1].load(X, at + 8);
  }
  float top = fmaxf(x[0].top(), x[1].top());
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (!live) return;
  const float s = block_scale(top, pow2 != 0);
  if (l == 0) scale_out[static_cast<size_t>(kb) * rows + row] = s;
  if (c < cols) {
    const float inv = __frcp_rn(s);
    const uint2 a = x[0].narrow(inv), b = x[1].narrow(inv);
    *reinterpret_cast<uint4*>(out + static_cast<size_t>(row) * cols + c) = make_uint4(a.x, a.y, b.x, b.y);
  }
}

// 128 x 128 tiles: a CTA holds its tile in registers, 16 lanes to a row.  A CTA first reads, then writes, so four of them (two, f32) share an
// SM: 8192 x 8192 bf16 40.5 -> 34.4 us, and 32.9 (6.1 TB/s) past the caches, one launch behind the other; f32 49.8 (6.7 TB/s).
template <bool F32>
__global__ void __launch_bounds__(256, F32 ? 2 : 4) quantize_tiles_kernel(const void* X, uint8_t* out, float* scale_out, int kb_total, int rb_total, int rows, int cols, int pow2) {
  __shared__ float tops[8];
  grid_dep_wait();
  grid_dep_launch();
  X = after_wait(X);
  const int kb = blockIdx.x % kb_total, rb = blockIdx.x / kb_total;  // rb counts over the matrices of the batch
  const int r0 = rb % rb_total * 128, batch = rb / rb_total;
  const int c = kb * 128 + (threadIdx.x & 15) * 8, r = r0 + (threadIdx.x >> 4);
  const size_t at = (static_cast<size_t>(batch) * rows + r) * cols + c;
  Vec8<F32, true> x[8];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i].zero();
    if (r + 16 * i < rows && c < cols) x[i].load(X, at + static_cast<size_t>(16 * i) * cols);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i].top());
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = fmaxf(top, tops[w]);
  const float s = block_scale(top, pow2 != 0), inv = __frcp_rn(s);
  if (threadIdx.x == 0) scale_out[blockIdx.x] = s;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (r + 16 * i < rows && c < cols) __stcs(reinterpret_cast<uint2*>(out + at + static_cast<size_t>(16 * i) * cols), x[i].narrow(inv));
}

}  // namespace qb

using namespace qb;

extern "C" int32_t qb_quantize_e4m3_blocks(const void* X, const int32_t* row_index, void* out, float* scale_out, const qb_quant_blocks_params* p, void* stream) {
  QB_REQUIRE(p != nullptr, QB_ERR_INVALID_ARG, "quantize_e4m3_blocks: params are NULL");
  QB_REQUIRE(X && out && scale_out, QB_ERR_INVALID_ARG, "quantize_e4m3_blocks: NULL pointer");
  QB_REQUIRE(p->batch > 0 && p->rows > 0 && p->cols > 0, QB_ERR_INVALID_ARG, "quantize_e4m3_blocks: %d matrices of %d x %d", p->batch, p->rows, p->cols);
  constexpr int kMost = 0x7fffffff - 127;  // rounded up to whole blocks it is still an int
  QB_REQUIRE(p->cols <= kMost && (p->tile_rows == 1 || p->rows <= kMost), QB_ERR_INVALID_ARG, "quantize_e4m3_blocks: %d x %d is too large", p->rows, p->cols);
  QB_REQUIRE(p->cols % 16 == 0, QB_ERR_ALIGN, "quantize_e4m3_blocks: %d columns (must be a multiple of 16)", p->cols);
  QB_REQUIRE(p->src_dtype == QB_BF16 || p->src_dtype == QB_F32, QB_ERR_INVALID_ARG, "quantize_e4m3_blocks: source dtype %d", p->src_dtype);
  QB_REQUIRE(p->tile_rows == 1 || p->tile_rows == 128, QB_ERR_INVALID_ARG, "quantize_e4m3_blocks: tile_rows %d (1 or 128)", p->tile_rows);
  QB_REQUIRE(aligned16(X) && aligned16(out) && (reinterpret_cast<uintptr_t>(scale_out) & 3u) == 0 && (reinterpret_cast<uintptr_t>(row_index) & 3u) == 0, QB_ERR_ALIGN,
             "quantize_e4m3_blocks: X and out must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* o = static_cast<uint8_t*>(out);
  const bool f32 = p->src_dtype == QB_F32;
  const int kb = (p->cols + 127) / 128;
  if (p->tile_rows == 128) {
    QB_REQUIRE(row_index == nullptr, QB_ERR_UNSUPPORTED, "quantize_e4m3_blocks: a row index goes with 1 x 128 groups");
    const int rb = (p->rows + 127) / 128;
    const long long tiles = static_cast<long long>(p->batch) * rb * kb;
    QB_REQUIRE(tiles < (1ll << 31), QB_ERR_INVALID_ARG, "quantize_e4m3_blocks: %lld tiles", tiles);
    return launch_dep("quantize_e4m3_blocks", f32 ? quantize_tiles_kernel<true> : quantize_tiles_kernel<false>, dim3(static_cast<unsigned>(tiles)), dim3(256), 0, st, X, o,
                      scale_out, kb, rb, p->rows, p->cols, p->pow2 != 0);
  }
  QB_REQUIRE(p->batch == 1, QB_ERR_UNSUPPORTED, "quantize_e4m3_blocks: a batch goes with 128 x 128 tiles");
  QB_REQUIRE(p->src_rows > 0 && (row_index != nullptr || p->src_rows == p->rows), QB_ERR_INVALID_ARG, "quantize_e4m3_blocks: %d rows from %d", p->rows, p->src_rows);
  const long long units = static_cast<long long>(p->rows) * kb;
  QB_REQUIRE(units < (1ll << 31) - 1024, QB_ERR_INVALID_ARG, "quantize_e4m3_blocks: %lld groups", units);
  return launch_dep("quantize_e4m3_blocks", f32 ? quantize_groups_kernel<true> : quantize_groups_kernel<false>, dim3(static_cast<unsigned>((units + 31) / 32)), dim3(256), 0, st,
                    X, row_index, o, scale_out, static_cast<int>(units), kb, p->rows, p->src_rows, p->cols, p->pow2 != 0);
}
