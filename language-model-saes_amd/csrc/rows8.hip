// Activation rows held in 8 bits ("rows8"): writing, reading, transposing, and gradient rows formed from them.
//
// A row of d values is ceil(d / 32) blocks of 32.  The record of a row (sae_rows8_pitch(d) bytes):
//   int8  code[32 * blocks]   zeros behind the d-th
//   uint8 field[blocks]       exponent field of the block's step: step = 2^(field - 127); 0: step 0 (a block of zeros);
//                             255: the block held an infinity or a NaN
//   zeros up to a multiple of 16 bytes
// value = code * step.  A code has 7 magnitude bits and the step is a power of two between 2^-126 and 2^121, so every value
// is exact in bf16 and the product below is exact in fp32; field 255 is the float infinity, and 0 * inf makes every value of
// such a block NaN without a test.
#include "common.h"

namespace sae {

// field of a block whose largest magnitude has these bits: the smallest step that brings it to 127 after rounding, i.e.
// 2^(floor(log2 amax) - 6), and twice that where amax / step would round to 128 (mantissa from 127.5 / 64 on; the tie is
// even at 128).  In the last binade there is no larger step whose codes stay finite: codes stop at 127 there.
__device__ __forceinline__ uint32_t r8_field(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  if (amax_bits == 0u) return 0u;
  if (e == 255u) return 255u;
  if (e < 7u) return 1u;
  return e - 6u + ((e < 254u && (amax_bits & 0x7fffffu) >= 0x7f0000u) ? 1u : 0u);
}

// one float -> its code under a block's field
__device__ __forceinline__ int r8_code(float x, uint32_t field) {
  if (field == 0u || field == 255u) return 0;
  const float inv = __uint_as_float((254u - field) << 23);
  return (int)fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
}

template <int DT>
__device__ __forceinline__ float r8_load(const void *src, int64_t i) {
  if constexpr (DT == SAE_BF16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(src)[i]);
  else return reinterpret_cast<const float *>(src)[i];
}
template <int DT>
__device__ __forceinline__ void r8_store(void *dst, int64_t i, float x) {
  if constexpr (DT == SAE_BF16) reinterpret_cast<uint16_t *>(dst)[i] = f32_to_bf16_bits(x);
  else reinterpret_cast<float *>(dst)[i] = x;
}

// element j of a record
__device__ __forceinline__ float r8_value(const uint8_t *rec, int64_t codes, int64_t j) {
  const float step = __uint_as_float((uint32_t)rec[codes + (j >> 5)] << 23);
  return (float)(int8_t)rec[j] * step;
}

// One workgroup per row; half a wave owns a block, one value per lane.
template <int DT>
__global__ __launch_bounds__(256) void rows8_quantize_kernel(const void *__restrict__ src, int64_t stride, int64_t d, uint8_t *__restrict__ dst,
                                                             uint16_t *__restrict__ copy) {
  const int64_t row = blockIdx.x, nb = r8_blocks(d), codes = nb * R8_BLOCK, pitch = r8_pitch(d);
  uint8_t *rec = dst + row * pitch;
  for (int64_t j = threadIdx.x; j < codes; j += 256) {
    const float x = j < d ? r8_load<DT>(src, row * stride + j) : 0.f;
    uint32_t top = __float_as_uint(x) & 0x7fffffffu;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint32_t other = __shfl_xor(top, o, 64);
      top = other > top ? other : top;
    }
    const uint32_t field = r8_field(top);
    rec[j] = (uint8_t)(int8_t)r8_code(x, field);
    if ((j & 31) == 0) rec[codes + (j >> 5)] = (uint8_t)field;
    if (copy && j < d) copy[row * d + j] = f32_to_bf16_bits(x);
  }
  for (int64_t j = codes + nb + threadIdx.x; j < pitch; j += 256) rec[j] = 0;
}

// dst[i, :] = cast(scale * values of record row_idx[i]); a row index outside the buffer gives a row of NaN.
template <int DT>
__global__ __launch_bounds__(256) void rows8_gather_kernel(const uint8_t *__restrict__ rows, const int64_t *__restrict__ row_idx,
                                                           int64_t n_src, int64_t d, float scale, void *__restrict__ dst) {
  const int64_t i = blockIdx.x, r = row_idx ? row_idx[i] : i, codes = r8_blocks(d) * R8_BLOCK;
  const bool ok = r >= 0 && r < n_src;
  const uint8_t *rec = rows + (ok ? r : 0) * r8_pitch(d);
  for (int64_t j = threadIdx.x; j < d; j += 256) {
    const float x = ok ? r8_value(rec, codes, j) : __uint_as_float(0x7fc00000u);
    r8_store<DT>(dst, i * d + j, x * scale);
  }
}

// dst[c, r] = src[r, c] for r < rows, 0 for rows <= r < dst_pitch, through a 64 x 64 tile.
template <int SRC, int DT>
__global__ __launch_bounds__(256) void transpose_padded_kernel(const void *__restrict__ src, int64_t rows, int64_t cols, void *__restrict__ dst,
                                                               int64_t dst_pitch) {
  __shared__ float tile[64][65];
  const int64_t r0 = (int64_t)blockIdx.y * 64, c0 = (int64_t)blockIdx.x * 64;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  for (int i = ty; i < 64; i += 4) {
    const int64_t r = r0 + i, c = c0 + tx;
    float x = 0.f;
    if (r < rows && c < cols) {
      if constexpr (SRC == SAE_ROWS8) x = r8_value(reinterpret_cast<const uint8_t *>(src) + r * r8_pitch(cols), r8_blocks(cols) * R8_BLOCK, c);
      else x = r8_load<SRC>(src, r * cols + c);
    }
    tile[i][tx] = x;
  }
  __syncthreads();
  for (int i = ty; i < 64; i += 4) {
    const int64_t c = c0 + i, r = r0 + tx;
    if (c < cols && r < dst_pitch) r8_store<DT>(dst, c * dst_pitch + r, tile[tx][i]);
  }
}

// out[f, :] = sum over feature f's slots, in the index's order, of coef[slot] * values of record slot_tok[slot]
__global__ __launch_bounds__(256) void rows8_grad_rows_kernel(const int32_t *__restrict__ feat_ptr, const int32_t *__restrict__ feat_slot,
                                                              const int32_t *__restrict__ slot_tok, const float *__restrict__ coef,
                                                              const uint8_t *__restrict__ rows, float *__restrict__ out,
                                                              float *__restrict__ bias_out, int64_t d) {
  const int64_t f = blockIdx.x, codes = r8_blocks(d) * R8_BLOCK, pitch = r8_pitch(d);
  const int lo = feat_ptr[f], hi = feat_ptr[f + 1];
  if (bias_out && threadIdx.x < 64) {
    float s = 0.f;
    for (int i = lo + (int)threadIdx.x; i < hi; i += 64) s += coef[feat_slot[i]];
    s = wave_sum(s);
    if (threadIdx.x == 0) bias_out[f] = s;
  }
  for (int64_t j = threadIdx.x; j < d; j += 256) {
    float acc = 0.f;
    for (int i = lo; i < hi; ++i) {
      const int sl = feat_slot[i];
      acc = fmaf(coef[sl], r8_value(rows + (int64_t)slot_tok[sl] * pitch, codes, j), acc);
    }
    out[f * d + j] = acc;
  }
}

// called by sae_sparse_grad_rows (feature_index.hip) for a dense operand held as rows8
int rows8_grad_rows(const int32_t *feat_ptr, const int32_t *feat_slot, const int32_t *slot_tok, const float *coef, const void *dense,
                    float *out, float *bias_out, int64_t F, int64_t d, hipStream_t st) {
  hipLaunchKernelGGL(rows8_grad_rows_kernel, dim3((unsigned)F), dim3(256), 0, st, feat_ptr, feat_slot, slot_tok, coef,
                     reinterpret_cast<const uint8_t *>(dense), out, bias_out, d);
  return check_launch("sparse_grad_rows[rows8]");
}

}  // namespace sae

extern "C" int64_t sae_rows8_pitch(int64_t d) { return d > 0 ? sae::r8_pitch(d) : 0; }

extern "C" int sae_rows8_quantize(const void *src, int src_dtype, int64_t n, int64_t d, int64_t src_stride, void *rows, void *bf16_copy,
                                  void *stream) {
  using namespace sae;
  SAE_REQUIRE(src && rows, SAE_ERR_INVALID_ARG, "rows8_quantize: null pointer");
  SAE_REQUIRE(n > 0 && d > 0 && src_stride >= 0, SAE_ERR_INVALID_ARG, "rows8_quantize: bad sizes");
  SAE_REQUIRE(src_dtype == SAE_F32 || src_dtype == SAE_BF16, SAE_ERR_INVALID_ARG, "rows8_quantize: bad dtype %d", src_dtype);
  SAE_REQUIRE(n < (1LL << 31) && d < (1LL << 30), SAE_ERR_UNSUPPORTED, "rows8_quantize: size too large");
  SAE_REQUIRE(((uintptr_t)rows & 15) == 0, SAE_ERR_INVALID_ARG, "rows8_quantize: rows must be 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  uint8_t *out = reinterpret_cast<uint8_t *>(rows);
  uint16_t *copy = reinterpret_cast<uint16_t *>(bf16_copy);
  if (src_dtype == SAE_BF16)
    hipLaunchKernelGGL(rows8_quantize_kernel<SAE_BF16>, dim3((unsigned)n), dim3(256), 0, st, src, src_stride, d, out, copy);
  else
    hipLaunchKernelGGL(rows8_quantize_kernel<SAE_F32>, dim3((unsigned)n), dim3(256), 0, st, src, src_stride, d, out, copy);
  return check_launch("rows8_quantize");
}

extern "C" int sae_rows8_gather(const void *rows, const int64_t *row_idx, int64_t n_src_rows, int64_t n_rows, int64_t d, void *dst,
                                int dst_dtype, double scale, void *stream) {
  using namespace sae;
  SAE_REQUIRE(rows && dst, SAE_ERR_INVALID_ARG, "rows8_gather: null pointer");
  SAE_REQUIRE(n_rows > 0 && n_src_rows > 0 && d > 0, SAE_ERR_INVALID_ARG, "rows8_gather: bad sizes");
  SAE_REQUIRE(row_idx || n_rows <= n_src_rows, SAE_ERR_INVALID_ARG, "rows8_gather: more rows asked for than there are");
  SAE_REQUIRE(dst_dtype == SAE_F32 || dst_dtype == SAE_BF16, SAE_ERR_INVALID_ARG, "rows8_gather: bad dtype %d", dst_dtype);
  SAE_REQUIRE(n_rows < (1LL << 31) && d < (1LL << 30), SAE_ERR_UNSUPPORTED, "rows8_gather: size too large");
  SAE_REQUIRE(((uintptr_t)rows & 15) == 0, SAE_ERR_INVALID_ARG, "rows8_gather: rows must be 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  const uint8_t *in = reinterpret_cast<const uint8_t *>(rows);
  if (dst_dtype == SAE_BF16)
    hipLaunchKernelGGL(rows8_gather_kernel<SAE_BF16>, dim3((unsigned)n_rows), dim3(256), 0, st, in, row_idx, n_src_rows, d, (float)scale, dst);
  else
    hipLaunchKernelGGL(rows8_gather_kernel<SAE_F32>, dim3((unsigned)n_rows), dim3(256), 0, st, in, row_idx, n_src_rows, d, (float)scale, dst);
  return check_launch("rows8_gather");
}

extern "C" int sae_transpose_padded(const void *src, int src_dtype, int64_t rows, int64_t cols, void *dst, int dst_dtype, int64_t dst_pitch,
                                    void *stream) {
  using namespace sae;
  SAE_REQUIRE(src && dst, SAE_ERR_INVALID_ARG, "transpose_padded: null pointer");
  SAE_REQUIRE(rows > 0 && cols > 0 && dst_pitch >= rows, SAE_ERR_INVALID_ARG, "transpose_padded: bad sizes");
  SAE_REQUIRE(src_dtype == SAE_F32 || src_dtype == SAE_BF16 || src_dtype == SAE_ROWS8, SAE_ERR_INVALID_ARG, "transpose_padded: bad dtype %d", src_dtype);
  SAE_REQUIRE(dst_dtype == SAE_F32 || dst_dtype == SAE_BF16, SAE_ERR_INVALID_ARG, "transpose_padded: bad dtype %d", dst_dtype);
  const int64_t gy = (dst_pitch + 63) / 64, gx = (cols + 63) / 64;
  SAE_REQUIRE(gy <= 65535 && gx < (1LL << 31), SAE_ERR_UNSUPPORTED, "transpose_padded: %lld rows, at most %d", (long long)dst_pitch, 65535 * 64);
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)gx, (unsigned)gy);
#define SAE_TP(S, D) hipLaunchKernelGGL((transpose_padded_kernel<S, D>), grid, dim3(256), 0, st, src, rows, cols, dst, dst_pitch)
  if (dst_dtype == SAE_BF16) {
    if (src_dtype == SAE_ROWS8) SAE_TP(SAE_ROWS8, SAE_BF16);
    else if (src_dtype == SAE_BF16) SAE_TP(SAE_BF16, SAE_BF16);
    else SAE_TP(SAE_F32, SAE_BF16);
  } else {
    if (src_dtype == SAE_ROWS8) SAE_TP(SAE_ROWS8, SAE_F32);
    else if (src_dtype == SAE_BF16) SAE_TP(SAE_BF16, SAE_F32);
    else SAE_TP(SAE_F32, SAE_F32);
  }
#undef SAE_TP
  return check_launch("transpose_padded");
}
