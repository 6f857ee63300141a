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
#include <algorithm>

#include "common.h"

namespace sae {

// field of a block whose largest magnitude has these bits: the smallest step that brings it to 127 after rounding, i.e.
// 2^(floor(log2 amax) - 6), and twice that where amax / step would round to 128 (mantissa from 127.5 / 64 on, the tie going
// to the even 128: the addition carries into the exponent there).  In the last binade no larger step is left whose values
// stay finite: codes stop at 127 there.
__device__ __forceinline__ uint32_t r8_field(uint32_t amax_bits) {
  const uint32_t e = (amax_bits + 0x10000u) >> 23;
  uint32_t f = (e > 7u ? e : 7u) - 6u;
  f = f < 248u ? f : 248u;
  f = amax_bits == 0u ? 0u : f;
  return amax_bits >= 0x7f800000u ? 255u : f;
}

// Four floats -> their codes under a block's field, packed.  x / step is exact (a power of two); adding 1.5 * 2^23 rounds it to
// nearest even and leaves the code in the sum's low byte.
__device__ __forceinline__ uint32_t r8_codes(const float *x, uint32_t field) {
  const bool bad = field == 255u;   // an infinity or a NaN in the block: no codes
  const float inv = __uint_as_float((254u - field) << 23);   // field 0: all x are 0
  uint32_t b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    b[e] = __float_as_uint(__builtin_amdgcn_fmed3f((bad ? 0.f : x[e]) * (bad ? 0.f : inv), -127.f, 127.f) + 12582912.f);
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
  return lo | hi;
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

// Row and piece of a flat task number: tasks run over the pieces of one row, then the next.  t / per_row as a product with a
// 32-bit reciprocal, exact for t < 2^31 (multiplier = ceil(2^(31 + s) / per_row) with per_row <= 2^s).
struct R8Split {
  uint32_t per_row, mul;
  int shift;
  explicit R8Split(int64_t n) : per_row((uint32_t)n), mul(0), shift(0) {   // n >= 2
    while ((1LL << shift) < n) ++shift;
    mul = (uint32_t)(((1ULL << (31 + shift)) + (uint64_t)n - 1) / (uint64_t)n);
  }
  __device__ __forceinline__ uint32_t row(uint32_t t) const { return __umulhi(t, mul) >> (shift - 1); }
};

// 16 bytes at any element's address: rows may start anywhere, and the memory instructions take any alignment.  Float rows
// pass once, records stay: float rows are read and written past the caches (16384 x 4096 bf16 read 39 -> 30 us, 32768 x 2048
// gathered to fp32 71 -> 52 us).  Writing and reading are bound by HBM from a few thousand rows on: 16384 x 4096 bf16 written in
// 34 us (6.0 TB/s), read in 30 (6.7).
template <int ALIGN>
struct R8Bytes16;
template <>
struct R8Bytes16<2> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct R8Bytes16<4> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};
template <int ALIGN>
struct __attribute__((packed, aligned(ALIGN))) R8Bytes8 {
  uint32_t w[2];
};

// Pieces per thread, the same for writing and reading: a record is then read back on the XCD whose L2 it was written from.
// 5003 x 2049 bf16 written and read at once: 2 and 2 pieces 14.8 us, 4 and 4 15.7, 2 and 4 18.5, 4 and 2 19.1, 8 and 4 20.9.
// Alone: 20000 x 1037 bf16 read 10.8 / 13.4 / 15.4 us at 2 / 4 / 8 pieces, written 14.1 / 14.9 / 17.6; whole pieces, 32768 x 2048 gathered
// to fp32 62 / 50 / 51, 20000 x 2048 fp32 written 34.2 / 33.6 / 35.1.
__host__ __device__ constexpr int r8_pieces(bool whole) { return whole ? 4 : 2; }

// largest of the 4 (8) neighbouring lanes that hold a block: lane permutations inside the vector unit, no LDS
template <int LANES>
__device__ __forceinline__ uint32_t r8_block_max(uint32_t x) {
  auto with = [&](uint32_t y) { x = y > x ? y : x; };
  with(__builtin_amdgcn_update_dpp(0, x, 0xB1, 0xf, 0xf, false));   // quad_perm [1, 0, 3, 2]
  with(__builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, false));   // quad_perm [2, 3, 0, 1]
  if constexpr (LANES == 8) with(__builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, false));   // row_half_mirror
  return x;
}

// A thread takes pieces of 16 source bytes (8 bf16 or 4 fp32 values), 4 or 8 neighbouring lanes a block of 32.  All loads are
// requested before the first is used, and none stands behind a branch: a piece past the task list or the row's end reads one
// that is inside and drops it; one that crosses the row's end (not where WHOLE: d is a multiple of the piece) reads on into what
// lies behind the row and drops that; only where that would pass the source's last value, `extent` from its first, are
// values read one by one (5003 rows of 2049 bf16, 37 apart: 12.8 us with every row's last piece read so, 11.9 without).
template <int DT, bool WHOLE>
__global__ __launch_bounds__(256) void rows8_quantize_kernel(const void *__restrict__ src, int64_t stride, int64_t d, uint8_t *__restrict__ dst,
                                                             uint16_t *__restrict__ copy, R8Split split, uint32_t n_tasks,
                                                             int64_t extent) {
  constexpr int W = DT == SAE_BF16 ? 8 : 4, LANES = R8_BLOCK / W, U = r8_pieces(WHOLE), ES = DT == SAE_BF16 ? 2 : 4;
  const int64_t nb = r8_blocks(d), codes = nb * R8_BLOCK, pitch = r8_pitch(d);
  const uint32_t first = blockIdx.x * (256 * U) + threadIdx.x;
  const char *base = reinterpret_cast<const char *>(extent >= W ? src : dst);   // fewer values than a piece: any 16 bytes, dropped
  typename R8Bytes16<ES>::type q[U];
  int64_t start[U];
  uint32_t row[U], col[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t t = first + u * 256 < n_tasks ? first + u * 256 : n_tasks - 1;
    row[u] = split.row(t);
    col[u] = (t - row[u] * split.per_row) * W;
    start[u] = (int64_t)row[u] * stride + (col[u] < d ? col[u] : 0);
    const int64_t from = WHOLE || start[u] + W <= extent ? start[u] : 0;
    q[u] = __builtin_nontemporal_load(reinterpret_cast<const typename R8Bytes16<ES>::type *>(base + from * ES));
  }
#pragma unroll
  for (int u = 0; u < U; ++u) asm volatile("" : "+v"(q[u]));   // the loads stay up here, before the branches
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float x[W];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == SAE_BF16) {
        x[2 * e] = __uint_as_float(q[u][e] << 16);
        x[2 * e + 1] = __uint_as_float(q[u][e] & 0xffff0000u);
      } else {
        x[e] = __uint_as_float(q[u][e]);
      }
    }
    if (!WHOLE && start[u] + W > extent) {
#pragma unroll
      for (int e = 0; e < W; ++e) x[e] = col[u] + e < d ? r8_load<DT>(src, start[u] + e) : 0.f;
    }
    uint32_t top = 0u;
#pragma unroll
    for (int e = 0; e < W; ++e) {
      x[e] = (WHOLE ? col[u] : col[u] + e) < d ? x[e] : 0.f;
      const uint32_t m = __float_as_uint(x[e]) & 0x7fffffffu;
      top = m > top ? m : top;
    }
    const uint32_t field = r8_field(r8_block_max<LANES>(top));
    if (first + u * 256 >= n_tasks) continue;
    uint8_t *rec = dst + (int64_t)row[u] * pitch;
    uint32_t packed[W / 4];
#pragma unroll
    for (int e = 0; e < W; e += 4) packed[e / 4] = r8_codes(&x[e], field);
    if constexpr (W == 8) *reinterpret_cast<uint2 *>(rec + col[u]) = make_uint2(packed[0], packed[W / 4 - 1]);
    else *reinterpret_cast<uint32_t *>(rec + col[u]) = packed[0];
    const int in_block = (int)(col[u] & 31) / W;
    if (in_block == 0) rec[codes + (col[u] >> 5)] = (uint8_t)field;
    if (col[u] >= codes - R8_BLOCK)   // the last block's lanes fill the record up
      for (int64_t j = codes + nb + in_block; j < pitch; j += LANES) rec[j] = 0;
    if constexpr (DT == SAE_F32) {
      if (copy) {
        uint16_t *c = copy + (int64_t)row[u] * d + col[u];
        if (WHOLE ? col[u] < d : col[u] + 4 <= d) {
          R8Bytes8<2> o;
          o.w[0] = pack_bf16x2(x[0], x[1]);
          o.w[1] = pack_bf16x2(x[2], x[3]);
          *reinterpret_cast<R8Bytes8<2> *>(c) = o;
        } else if constexpr (!WHOLE) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col[u] + e < d) c[e] = f32_to_bf16_bits(x[e]);
        }
      }
    }
  }
}

// dst[i, :] = cast(scale * values of record row_idx[i]); a row index outside the buffer gives a row of NaN.  A thread takes
// pieces of 16 bytes of the output (8 bf16 or 4 fp32 values); loads as above (WHOLE, and nothing behind a branch: a thread
// past the task list reads the last piece again, an index outside the buffer reads row 0, and both drop what they read).
template <int DT, bool IDX, bool WHOLE>
__global__ __launch_bounds__(256) void rows8_gather_kernel(const uint8_t *__restrict__ rows, const int64_t *__restrict__ row_idx,
                                                           int64_t n_src, int64_t d, float scale, void *__restrict__ dst, R8Split split,
                                                           uint32_t n_tasks) {
  constexpr int W = DT == SAE_BF16 ? 8 : 4, U = r8_pieces(WHOLE), ES = DT == SAE_BF16 ? 2 : 4;
  const int64_t codes = r8_blocks(d) * R8_BLOCK, pitch = r8_pitch(d);
  const uint32_t first = blockIdx.x * (256 * U) + threadIdx.x;
  uint32_t row[U], col[U], packed[U][W / 4], field[U];
  int64_t r[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t t = first + u * 256 < n_tasks ? first + u * 256 : n_tasks - 1;
    row[u] = split.row(t);
    col[u] = (t - row[u] * split.per_row) * W;
    r[u] = IDX ? row_idx[row[u]] : (int64_t)row[u];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool inside = r[u] >= 0 && r[u] < n_src;
    const uint8_t *rec = rows + (inside ? r[u] : 0) * pitch;
    if constexpr (W == 8) {
      const uint2 q = *reinterpret_cast<const uint2 *>(rec + col[u]);
      packed[u][0] = inside ? q.x : 0u;
      packed[u][W / 4 - 1] = inside ? q.y : 0u;
    } else {
      const uint32_t q = *reinterpret_cast<const uint32_t *>(rec + col[u]);
      packed[u][0] = inside ? q : 0u;
    }
    const uint32_t q = rec[codes + (col[u] >> 5)];
    field[u] = inside ? q : 255u;   // 0 * inf: NaN
  }
#pragma unroll
  for (int u = 0; u < U; ++u) asm volatile("" : "+v"(packed[u][0]));   // the loads stay up here, before the branches
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (first + u * 256 >= n_tasks || col[u] >= d) continue;
    const float step = __uint_as_float(field[u] << 23);
    float x[W];
#pragma unroll
    for (int e = 0; e < W; ++e) x[e] = (float)(int8_t)(packed[u][e / 4] >> (8 * (e % 4))) * step * scale;
    char *at = reinterpret_cast<char *>(dst) + ((int64_t)row[u] * d + col[u]) * ES;
    if (WHOLE || col[u] + W <= d) {
      typename R8Bytes16<ES>::type o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (DT == SAE_BF16) o[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
        else o[e] = __float_as_uint(x[e]);
      }
      __builtin_nontemporal_store(o, reinterpret_cast<typename R8Bytes16<ES>::type *>(at));
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (col[u] + e < d) r8_store<DT>(at, e, x[e]);
    }
  }
}

// dst[c, r] = bf16(src[r, c]) for r < rows, 0 for rows <= r < dst_pitch: 128 rows x 64 columns per workgroup.  A thread takes 8
// columns of two rows at a time and writes them to LDS as pairs of rows, column by column (33-word columns: a wave's words
// fall on 64 banks), so that an output row leaves in whole 16-byte stores of 8 tokens.
template <int SRC>
__global__ __launch_bounds__(256) void transpose_padded_kernel(const void *__restrict__ src, int64_t rows, int64_t cols, uint16_t *__restrict__ dst,
                                                               int64_t dst_pitch, uint32_t col_blocks) {
  __shared__ uint32_t tile[2][64 * 33];
  const int64_t r0 = (int64_t)(blockIdx.x / col_blocks) * 128, c0 = (int64_t)(blockIdx.x % col_blocks) * 64;
  const int group = threadIdx.x & 7, pair = threadIdx.x >> 3;   // 8 columns, and 32 pairs of rows
  const int64_t col = c0 + group * 8, end = SRC == SAE_ROWS8 ? r8_blocks(cols) * R8_BLOCK : cols;
  const size_t pitch = dense_row_bytes<SRC>(cols);
  const uint8_t *base = reinterpret_cast<const uint8_t *>(src);
  u32x4 q[2][2];
  uint32_t field[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = r0 + h * 64 + pair * 2 + i;
      const uint8_t *row = base + (size_t)(r < rows ? r : rows - 1) * pitch;
      const bool in = r < rows && col < end;
      if constexpr (SRC == SAE_ROWS8) {
        const uint2 w = *reinterpret_cast<const uint2 *>(row + (col < end ? col : 0));
        field[h][i] = in ? (uint32_t)row[end + ((col < end ? col : 0) >> 5)] : 0u;
        q[h][i] = in ? u32x4{w.x, w.y, 0u, 0u} : u32x4{0u, 0u, 0u, 0u};
      } else {
        q[h][i] = u32x4{0u, 0u, 0u, 0u};
        if (in) {
          if (col + 8 <= cols) {
            const auto w = *reinterpret_cast<const typename R8Bytes16<2>::type *>(row + col * 2);
            q[h][i] = u32x4{w[0], w[1], w[2], w[3]};
          } else {
            uint32_t e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = col + j < cols ? (uint32_t)reinterpret_cast<const uint16_t *>(row)[col + j] : 0u;
            q[h][i] = u32x4{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
          }
        }
      }
    }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t even[4], odd[4];   // the two rows' 8 values as bf16 pairs of columns
    if constexpr (SRC == SAE_ROWS8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float step = __uint_as_float(field[h][i] << 23);
        const uint32_t w[2] = {q[h][i].x, q[h][i].y};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          (i ? odd : even)[j] = pack_bf16x2((float)(int8_t)(w[j >> 1] >> (16 * (j & 1))) * step, (float)(int8_t)(w[j >> 1] >> (16 * (j & 1) + 8)) * step);
      }
    } else {
      even[0] = q[h][0].x; even[1] = q[h][0].y; even[2] = q[h][0].z; even[3] = q[h][0].w;
      odd[0] = q[h][1].x; odd[1] = q[h][1].y; odd[2] = q[h][1].z; odd[3] = q[h][1].w;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      tile[h][(group * 8 + 2 * j) * 33 + pair] = (even[j] & 0xffffu) | (odd[j] << 16);
      tile[h][(group * 8 + 2 * j + 1) * 33 + pair] = (even[j] >> 16) | (odd[j] & 0xffff0000u);
    }
  }
  __syncthreads();
  const int part = threadIdx.x & 15, first = threadIdx.x >> 4;   // 16 threads write the 128 tokens of one column
  const int64_t r = r0 + part * 8;
  if (r >= dst_pitch) return;   // the pitch is a multiple of 8
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = first + 16 * k;
    if (c0 + c >= cols) break;
    const uint32_t *w = &tile[part >> 3][c * 33 + (part & 7) * 4];
    *reinterpret_cast<u32x4 *>(dst + (c0 + c) * dst_pitch + r) = u32x4{w[0], w[1], w[2], w[3]};
  }
}

// ---- gradient rows ---------------------------------------------------------------------------------------------------
// out[f, :] = sum over feature f's slots of coef * (values of the slot's record): a segmented sum over the feature index.
// Some features are kept by most tokens and most by few, so work is cut by position in feat_slot, not by feature: a wave
// owns a window of positions and 256 columns.  A segment that lies inside a window goes straight to its row; one that crosses
// leaves one partial row per window, joined in a fixed order by a third launch.
// (8192 tokens, 64 of 32768 features, d = 2048: 147 us; a workgroup per feature, as the first form here, took 33 ms there, the
// most frequent feature's 8192 records one after the other.  292 MB have to move, 42 us at the rate of a large fill.  The second
// launch is 121-132 us, 252 to 279 thousand cycles: its vector units issue for 225 thousand of them (13 instructions per record and
// four columns), the address units of its vector loads, two per record and chunk, are busy for 190.)
constexpr int R8_COLS = 256;   // columns of a chunk: four per lane (eight per lane: 196 us instead of 184, before the streaming
                               // stores)

// Positions per window.  Long windows leave fewer partial rows, short ones more waves: with few waves per CU a window's
// records, read one group after the other, are what takes the time.  us at 32 / 64 / 128 positions, by windows of 128 times
// chunks: 550 (1100 tokens, k = 32, d = 512) 16 / 18 / 24; 1536 (2048, 32, 768) 23 / 22 / 28; 3072 (4096, 32, 768) 33 / 29 / 31; 4096 (4096, 32,
// 1024) 37 / 34 / 34; 6144 (8192, 32, 768) 53 / 46 / 45; 8192 (16384, 32, 512) 89 / 74 / 69; 32768 (8192, 64, 2048) 192 / 158 / 146.
static int r8_window(int64_t n_slots, int64_t d) {
  const int64_t tasks = (n_slots + 127) / 128 * ((d + R8_COLS - 1) / R8_COLS);
  return tasks < 1024 ? 32 : tasks < 4096 ? 64 : 128;
}

// Positions in use, counted from the first feature's: the index may be a stretch of a longer one's features.  0 where they are
// more than the host was told: the launches behind the first then find nothing to do.
__device__ __forceinline__ int r8_used(const int32_t *__restrict__ feat_ptr, int64_t F, int n_slots) {
  const int used = feat_ptr[F] - feat_ptr[0];
  return used <= n_slots ? used : 0;
}

// The first launch.  Workgroups below feat_blocks, a wave per feature: the feature of each of its positions, a zero row where
// it has none, its coefficients' sum.  The others, a thread per position: token and coefficient in index order, so that the
// waves of the second launch, one per window and chunk of columns, read them in line (by slot they would touch a cache line
// per entry, once for every chunk).  Positions behind the last feature's, up to a whole window, get feature -1.  More positions in
// use than the host was told: rows and sums of NaN.
__global__ __launch_bounds__(256) void rows8_grad_prepare_kernel(const int32_t *__restrict__ feat_ptr, const int32_t *__restrict__ feat_slot,
                                                                 const int32_t *__restrict__ slot_tok, const float *__restrict__ coef,
                                                                 int32_t *__restrict__ pos_feat, int32_t *__restrict__ pos_tok,
                                                                 float *__restrict__ pos_coef, float *__restrict__ out,
                                                                 float *__restrict__ bias_out, int64_t F, int64_t d, uint32_t feat_blocks,
                                                                 int window, int n_slots) {
  const int first = feat_ptr[0];
  if (blockIdx.x >= feat_blocks) {
    const int64_t i = (int64_t)(blockIdx.x - feat_blocks) * 256 + threadIdx.x;
    const int total = r8_used(feat_ptr, F, n_slots);
    if (i < total) {
      const int slot = feat_slot[first + i];
      pos_tok[i] = slot_tok[slot];
      pos_coef[i] = coef[slot];
    } else if (i < ((int64_t)total + window - 1) / window * window) {
      pos_feat[i] = -1;
      pos_tok[i] = 0;
      pos_coef[i] = 0.f;
    }
    return;
  }
  const int64_t f = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (f >= F) return;
  const int lo = feat_ptr[f], hi = feat_ptr[f + 1];
  const bool fits = feat_ptr[F] - first <= n_slots;
  const float empty = fits ? 0.f : __uint_as_float(0x7fc00000u);
  if (fits)
    for (int i = lo + lane; i < hi; i += 64) pos_feat[i - first] = (int32_t)f;
  if (bias_out) {
    float s = empty;
#pragma unroll 4
    for (int i = lo + lane; i < hi; i += 64) s += coef[feat_slot[i]];
    s = wave_sum(s);
    if (lane == 0) bias_out[f] = s;
  }
  if (lo < hi && fits) return;
  float *row = out + f * d;
  if ((d & 3) == 0) {
    for (int64_t j = lane; j < (d >> 2); j += 64) store_stream(row, j, make_float4(empty, empty, empty, empty));
  } else {
    for (int64_t j = lane; j < d; j += 64) row[j] = empty;
  }
}

// The second launch: a wave per window and chunk.  What says which record is read is the same for the whole wave and stays in
// scalar registers.
template <int WINDOW>
__global__ __launch_bounds__(256) void rows8_grad_window_kernel(const int32_t *__restrict__ feat_ptr, const int32_t *__restrict__ pos_feat,
                                                                const int32_t *__restrict__ pos_tok, const float *__restrict__ pos_coef,
                                                                const uint8_t *__restrict__ rows, float *__restrict__ out,
                                                                float *__restrict__ part, int64_t F, int64_t d, int64_t n_windows,
                                                                int64_t n_tasks, int n_slots) {
  constexpr int G = 16;   // records requested together
  const int lane = threadIdx.x & 63;
  // tasks in chunk-major order, one contiguous eighth per XCD (workgroups go round the XCDs): what an XCD reads at a time
  // is one chunk of columns of all records, which its L2 holds
  const int64_t per_xcd = (n_tasks + 7) / 8;
  const int64_t local = (int64_t)(blockIdx.x >> 3) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t task = (int64_t)(blockIdx.x & 7) * per_xcd + local;
  if (local >= per_xcd || task >= n_tasks) return;
  const int64_t chunk = task / n_windows, window = task % n_windows;
  const int total = r8_used(feat_ptr, F, n_slots);
  const int w0 = (int)(window * WINDOW), w1 = w0 + WINDOW;
  if (w0 >= total) return;
  const int64_t codes = r8_blocks(d) * R8_BLOCK;
  const uint32_t pitch = (uint32_t)r8_pitch(d);
  const int64_t col = chunk * R8_COLS + lane * 4;
  const bool on = col < codes;
  const uint32_t code_off = on ? (uint32_t)col : 0u, field_off = (uint32_t)(codes + (on ? col >> 5 : 0));   // in a record
  const int before = w0 > 0 ? pos_feat[w0 - 1] : -1, after = w1 < total ? pos_feat[w1] : -1;

  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  int current = -1;   // the feature being summed
  auto flush = [&]() {
    if (on && current >= 0) {
      const float4 sum = make_float4(acc[0], acc[1], acc[2], acc[3]);
      const bool head = current == before, tail = current == after;
      if (head || tail) {
        *reinterpret_cast<float4 *>(part + (window * 2 + (head ? 0 : 1)) * codes + col) = sum;
      } else {
        float *dst = out + (int64_t)current * d + col;   // written once, read by no one here: it need not displace records
        if ((d & 3) == 0) {
          if (col < d) store_stream(dst, 0, sum);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < d) dst[e] = acc[e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = 0.f;
  };

  for (int p = w0; p < w1; p += G) {
    uint32_t codes4[G], field[G];
    int feat[G];
    float coef[G];
    // 32-bit offsets that the compiler cannot widen ahead of the loop: the loads then add them to a scalar base themselves
    uint32_t code_at = code_off, field_at = field_off;
    asm("" : "+v"(code_at), "+v"(field_at));
#pragma unroll
    for (int j = 0; j < G; ++j) {
      feat[j] = pos_feat[p + j];
      coef[j] = pos_coef[p + j];
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const uint8_t *rec = rows + (uint64_t)(uint32_t)pos_tok[p + j] * pitch;
      codes4[j] = *reinterpret_cast<const uint32_t *>(rec + code_at);
      field[j] = rec[field_at];
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
      if (feat[j] != current) {
        flush();
        current = feat[j];
      }
      const float step = __uint_as_float(field[j] << 23);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(coef[j], (float)(int8_t)(codes4[j] >> (8 * e)) * step, acc[e]);
    }
  }
  flush();
}

// The third launch: the segment that begins in this window and goes on behind it, 1024 columns per workgroup.  The first half of
// the threads adds the first, third, ... partial row, the second half the others, and the two sums are added: the most
// frequent feature's rows are a chain of half their number (8192 tokens, k = 8, d = 700: 29 -> 23 us for all three launches;
// four chains of 256 columns take 23 too, and 7 us more at 8192, 64, 2048, in workgroups that find nothing to do).  Workgroups of
// two waves for up to 256 columns: 38 instead of 44 us at 8192, 64, 64.
template <int LANES>
__global__ __launch_bounds__(2 * LANES) void rows8_grad_join_kernel(const int32_t *__restrict__ feat_ptr, const int32_t *__restrict__ pos_feat,
                                                              const float *__restrict__ part, float *__restrict__ out, int64_t F, int64_t d,
                                                             int length, int n_slots) {
  const int64_t window = blockIdx.x;
  const int total = r8_used(feat_ptr, F, n_slots);
  const int64_t w0 = window * length, w1 = w0 + length;
  const int f = pos_feat[w1 < (int64_t)gridDim.x * length ? w1 : w0], inside = pos_feat[w1 - 1], before = pos_feat[w0 > 0 ? w0 - 1 : 0];
  if (w1 >= total || f < 0 || inside != f || (w0 > 0 && before == f)) return;
  const int64_t last = (feat_ptr[f + 1] - feat_ptr[0] - 1) / length, codes = r8_blocks(d) * R8_BLOCK;
  __shared__ float4 sums[LANES];
  const int half = threadIdx.x / LANES, at = threadIdx.x % LANES;
  const int64_t j = ((int64_t)blockIdx.y * LANES + at) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (j < d) {
    if (half == 0) s = *reinterpret_cast<const float4 *>(part + (window * 2 + 1) * codes + j);
#pragma unroll 8
    for (int64_t w = window + 1 + half; w <= last; w += 2) {
      const float4 x = *reinterpret_cast<const float4 *>(part + w * 2 * codes + j);
      s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
  }
  if (half) sums[at] = s;
  __syncthreads();   // every thread of the workgroup is here: the returns above are the same for all
  if (half || j >= d) return;
  s.x += sums[at].x; s.y += sums[at].y; s.z += sums[at].z; s.w += sums[at].w;
  float *dst = out + (int64_t)f * d + j;
  if ((d & 3) == 0) {
    store_stream(dst, 0, s);
  } else {
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e < d) dst[e] = v[e];
  }
}

// Few slots: three launches take longer (17 us of host time) than their work.  Here a workgroup owns eight features and 256 columns;
// a wave looks a feature's slots up itself, one per lane, and adds their records in ascending order, 32 requested together.  A
// segment of more than 32 slots is cut into eighths, one per wave, whose sums are added in order.
// us as a call among others, this and the three launches: 64 tokens, k = 32, F = 6144, d = 768 10 and 17, 384 tokens of it 15 and 17, 512
// 17 and 17, 1024 25 and 19; 1024, 4, 512, 512 11 and 17; 64, 64, 32768, 2048 54 and 58, 256 tokens of it 73 and 62; features that
// nearly all tokens keep: 512, 16, 256, 768 14 and 17, 96, 64, 64, 512 18 and 17.
static bool r8_short(int64_t n_rows, int64_t n_slots, int64_t F, int64_t d) {
  return n_rows <= 1024 && n_slots * ((d + R8_COLS - 1) / R8_COLS) <= 40000 && n_slots <= 32 * F;
}

__global__ __launch_bounds__(512) void rows8_grad_short_kernel(const int32_t *__restrict__ feat_ptr, const int32_t *__restrict__ feat_slot,
                                                               const int32_t *__restrict__ slot_tok, const float *__restrict__ coef,
                                                               const uint8_t *__restrict__ rows, float *__restrict__ out,
                                                               float *__restrict__ bias_out, int64_t F, int64_t d) {
  constexpr int G = 32, PART = 8;   // records requested together, and in how many steps: a feature of few slots reads few
  constexpr int SHARED = 32;        // slots from which a segment is shared by the workgroup's waves
  __shared__ float4 part[8][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t f0 = (int64_t)blockIdx.x * 8, f = f0 + wave;
  const int bound = feat_ptr[f0 + lane < F ? f0 + lane : F];   // lanes 0 .. 8: where the workgroup's segments begin and end
  const int lo = __builtin_amdgcn_readlane(bound, wave), hi = __builtin_amdgcn_readlane(bound, wave + 1);
  const int64_t codes = r8_blocks(d) * R8_BLOCK, col = (int64_t)blockIdx.y * R8_COLS + lane * 4;
  const uint32_t pitch = (uint32_t)r8_pitch(d);
  const bool on = col < codes;
  const uint32_t code_at = on ? (uint32_t)col : 0u, field_at = (uint32_t)(codes + (on ? col >> 5 : 0));
  float acc[4];
  auto sum = [&](int first, int last) {   // of the records at positions first .. last - 1
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = 0.f;
    for (int p0 = first; p0 < last; p0 += 64) {
      const int n = last - p0 < 64 ? last - p0 : 64, slot = feat_slot[p0 + (lane < n ? lane : n - 1)];   // 64 slots, one per lane
      const int tok = slot_tok[slot];
      const float cf = coef[slot];
      for (int p = 0; p < n; p += G) {
        uint32_t codes4[G], field[G];
#pragma unroll
        for (int i = 0; i < G; i += PART) {
          if (p + i >= n) break;
#pragma unroll
          for (int j = i; j < i + PART; ++j) {
            const uint8_t *rec = rows + (uint64_t)(uint32_t)__builtin_amdgcn_readlane(tok, p + j) * pitch;   // past n: the last one again
            codes4[j] = *reinterpret_cast<const uint32_t *>(rec + code_at);
            field[j] = rec[field_at];
          }
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
          if (p + j >= n) break;
          const float c = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(cf), p + j)), step = __uint_as_float(field[j] << 23);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = fmaf(c, (float)(int8_t)(codes4[j] >> (8 * e)) * step, acc[e]);
        }
      }
    }
  };
  auto store = [&]() {
    float *dst = out + f * d + col;
    if ((d & 3) == 0) {
      if (col < d) store_stream(dst, 0, make_float4(acc[0], acc[1], acc[2], acc[3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < d) dst[e] = acc[e];
    }
  };
  if (f < F) {
    if (hi - lo <= SHARED) {
      sum(lo, hi);
      store();
    }
    if (bias_out && blockIdx.y == 0) {
      float s = 0.f;
      for (int i = lo + lane; i < hi; i += 64) s += coef[feat_slot[i]];
      s = wave_sum(s);
      if (lane == 0) bias_out[f] = s;
    }
  }
  const int next = __shfl_down(bound, 1, 64);   // every lane takes part: lane 7 reads lane 8
  // the same for every thread of the workgroup; past F all bounds are equal
  for (uint64_t shared = __ballot(lane < 8 && next - bound > SHARED); shared; shared &= shared - 1) {
    const int g = __builtin_ctzll(shared), first = __builtin_amdgcn_readlane(bound, g), n = __builtin_amdgcn_readlane(bound, g + 1) - first;
    const int each = (n + 63) / 64 * 8, a = first + (wave * each < n ? wave * each : n);   // an eighth for each wave, in whole PARTs
    sum(a, a + each < first + n ? a + each : first + n);
    part[wave][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (wave == g) {
      float4 s = part[0][lane];
#pragma unroll
      for (int w = 1; w < 8; ++w) {
        const float4 x = part[w][lane];
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
      }
      acc[0] = s.x; acc[1] = s.y; acc[2] = s.z; acc[3] = s.w;
      store();
    }
    __syncthreads();   // part is written again
  }
}

}  // namespace sae

extern "C" int64_t sae_rows8_pitch(int64_t d) { return d > 0 ? sae::r8_pitch(d) : 0; }

extern "C" int sae_rows8_quantize(const void *src, int src_dtype, int64_t n, int64_t d, int64_t src_stride, void *rows, void *bf16_copy,
                                  void *stream) {
  using namespace sae;
  SAE_REQUIRE(src && rows, SAE_ERR_INVALID_ARG, "rows8_quantize: null pointer");
  SAE_REQUIRE(n > 0 && d > 0 && src_stride >= 0, SAE_ERR_INVALID_ARG, "rows8_quantize: bad sizes");
  SAE_REQUIRE(src_dtype == SAE_F32 || src_dtype == SAE_BF16, SAE_ERR_INVALID_ARG, "rows8_quantize: bad dtype %d", src_dtype);
  SAE_REQUIRE(!bf16_copy || src_dtype == SAE_F32, SAE_ERR_INVALID_ARG, "rows8_quantize: a bf16 source is its own copy");
  SAE_REQUIRE(n < (1LL << 31) && d < (1LL << 30), SAE_ERR_UNSUPPORTED, "rows8_quantize: size too large");
  SAE_REQUIRE(((uintptr_t)rows & 15) == 0, SAE_ERR_INVALID_ARG, "rows8_quantize: rows must be 16-byte aligned");
  const int width = src_dtype == SAE_BF16 ? 8 : 4, size = src_dtype == SAE_BF16 ? 2 : 4;
  const R8Split split(r8_blocks(d) * (R8_BLOCK / width));
  const int64_t rows_per_launch = (1LL << 30) / split.per_row;   // task numbers stay below 2^31
  for (int64_t r0 = 0; r0 < n; r0 += rows_per_launch) {
    const int64_t m = n - r0 < rows_per_launch ? n - r0 : rows_per_launch, tasks = m * split.per_row;
    const int64_t per_block = 256 * r8_pieces(d % width == 0);
    const dim3 grid((unsigned)((tasks + per_block - 1) / per_block));
    const void *in = reinterpret_cast<const char *>(src) + r0 * src_stride * size;
    const int64_t extent = (m - 1) * src_stride + d;   // values from the first to the last that may be read
    uint8_t *out = reinterpret_cast<uint8_t *>(rows) + r0 * r8_pitch(d);
    uint16_t *copy = bf16_copy ? reinterpret_cast<uint16_t *>(bf16_copy) + r0 * d : nullptr;
#define SAE_R8_QUANTIZE(DT, WHOLE)                                                                                              \
  hipLaunchKernelGGL((rows8_quantize_kernel<DT, WHOLE>), grid, dim3(256), 0, (hipStream_t)stream, in, src_stride, d, out, copy, split, \
                     (uint32_t)tasks, extent)
    if (src_dtype == SAE_BF16) { if (d % width == 0) SAE_R8_QUANTIZE(SAE_BF16, true); else SAE_R8_QUANTIZE(SAE_BF16, false); }
    else { if (d % width == 0) SAE_R8_QUANTIZE(SAE_F32, true); else SAE_R8_QUANTIZE(SAE_F32, false); }
#undef SAE_R8_QUANTIZE
  }
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
  const int width = dst_dtype == SAE_BF16 ? 8 : 4, size = dst_dtype == SAE_BF16 ? 2 : 4;
  const R8Split split(r8_blocks(d) * (R8_BLOCK / width));
  const int64_t rows_per_launch = (1LL << 30) / split.per_row;   // task numbers stay below 2^31
  for (int64_t r0 = 0; r0 < n_rows; r0 += rows_per_launch) {
    const int64_t m = n_rows - r0 < rows_per_launch ? n_rows - r0 : rows_per_launch, tasks = m * split.per_row;
    const int64_t per_block = 256 * r8_pieces(d % width == 0);
    const dim3 grid((unsigned)((tasks + per_block - 1) / per_block));
    const uint8_t *in = reinterpret_cast<const uint8_t *>(rows) + (row_idx ? 0 : r0 * r8_pitch(d));
    const int64_t *idx = row_idx ? row_idx + r0 : nullptr;
    void *out = reinterpret_cast<char *>(dst) + r0 * d * size;
#define SAE_R8_GATHER(DT, IDX, WHOLE)                                                                                         \
  hipLaunchKernelGGL((rows8_gather_kernel<DT, IDX, WHOLE>), grid, dim3(256), 0, (hipStream_t)stream, in, idx, IDX ? n_src_rows : m, d, \
                     (float)scale, out, split, (uint32_t)tasks)
#define SAE_R8_GATHER_TYPE(DT)                                                                        \
  if (idx) { if (d % width == 0) SAE_R8_GATHER(DT, true, true); else SAE_R8_GATHER(DT, true, false); } \
  else { if (d % width == 0) SAE_R8_GATHER(DT, false, true); else SAE_R8_GATHER(DT, false, false); }
    if (dst_dtype == SAE_BF16) { SAE_R8_GATHER_TYPE(SAE_BF16) } else { SAE_R8_GATHER_TYPE(SAE_F32) }
#undef SAE_R8_GATHER_TYPE
#undef SAE_R8_GATHER
  }
  return check_launch("rows8_gather");
}

extern "C" int sae_transpose_padded(const void *src, int src_dtype, int64_t rows, int64_t cols, void *dst, int64_t dst_pitch, void *stream) {
  using namespace sae;
  SAE_REQUIRE(src && dst, SAE_ERR_INVALID_ARG, "transpose_padded: null pointer");
  SAE_REQUIRE(rows > 0 && cols > 0 && dst_pitch >= rows && dst_pitch % 8 == 0, SAE_ERR_INVALID_ARG, "transpose_padded: bad sizes");
  SAE_REQUIRE(src_dtype == SAE_BF16 || src_dtype == SAE_ROWS8, SAE_ERR_INVALID_ARG, "transpose_padded: bad dtype %d", src_dtype);
  SAE_REQUIRE(((uintptr_t)dst & 15) == 0 && (src_dtype != SAE_ROWS8 || ((uintptr_t)src & 15) == 0), SAE_ERR_INVALID_ARG,
              "transpose_padded: 16-byte alignment required");
  const int64_t gy = (dst_pitch + 127) / 128, gx = (cols + 63) / 64;
  // one grid axis of less than 2^32 threads: 2^24 workgroups write 256 GiB
  SAE_REQUIRE(dst_pitch < (1LL << 30) && cols < (1LL << 30) && gx * gy < (1LL << 24), SAE_ERR_UNSUPPORTED,
              "transpose_padded: %lld x %lld is too large", (long long)dst_pitch, (long long)cols);
  const dim3 grid((unsigned)(gx * gy));
  uint16_t *out = reinterpret_cast<uint16_t *>(dst);
  if (src_dtype == SAE_ROWS8)
    hipLaunchKernelGGL(transpose_padded_kernel<SAE_ROWS8>, grid, dim3(256), 0, (hipStream_t)stream, src, rows, cols, out, dst_pitch, (uint32_t)gx);
  else
    hipLaunchKernelGGL(transpose_padded_kernel<SAE_BF16>, grid, dim3(256), 0, (hipStream_t)stream, src, rows, cols, out, dst_pitch, (uint32_t)gx);
  return check_launch("transpose_padded");
}

extern "C" int64_t sae_rows8_grad_rows_workspace_bytes(int64_t n_rows, int64_t n_slots, int64_t F, int64_t d) {
  using namespace sae;
  if (n_rows <= 0 || n_slots <= 0 || F <= 0 || d <= 0 || r8_short(n_rows, n_slots, F, d)) return 0;
  const int64_t length = r8_window(n_slots, d), windows = (n_slots + length - 1) / length;
  // feature, token and coefficient of every position, and two partial rows per window
  return windows * length * 12 + windows * 2 * r8_blocks(d) * R8_BLOCK * 4;
}

extern "C" int sae_rows8_grad_rows(const int32_t *feat_ptr, const int32_t *feat_slot, const int32_t *slot_tok, const float *coef,
                                   const void *rows, int64_t n_rows, float *out, float *bias_out, int64_t F, int64_t d, int64_t n_slots,
                                   void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace sae;
  SAE_REQUIRE(feat_ptr && feat_slot && slot_tok && coef && rows && out, SAE_ERR_INVALID_ARG, "rows8_grad_rows: null pointer");
  SAE_REQUIRE(F > 0 && d > 0 && n_slots > 0 && n_rows > 0, SAE_ERR_INVALID_ARG, "rows8_grad_rows: bad sizes");
  SAE_REQUIRE(F < (1LL << 31) - 1 && d <= 65535LL * R8_COLS && n_slots < (1LL << 31) - 128, SAE_ERR_UNSUPPORTED, "rows8_grad_rows: size too large");
  SAE_REQUIRE((((uintptr_t)rows | (uintptr_t)workspace) & 15) == 0 && ((uintptr_t)out & (d % 4 == 0 ? 15 : 3)) == 0, SAE_ERR_INVALID_ARG,
              "rows8_grad_rows: 16-byte alignment required");
  const int64_t need = sae_rows8_grad_rows_workspace_bytes(n_rows, n_slots, F, d);
  SAE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), SAE_ERR_WORKSPACE, "rows8_grad_rows: workspace of %lld bytes needed",
              (long long)need);
  hipStream_t st = (hipStream_t)stream;
  const int length = r8_window(n_slots, d);
  const int64_t windows = (n_slots + length - 1) / length, positions = windows * length;
  int32_t *pos_feat = reinterpret_cast<int32_t *>(workspace), *pos_tok = pos_feat + positions;
  float *pos_coef = reinterpret_cast<float *>(pos_tok + positions), *part = pos_coef + positions;
  const uint8_t *rec = reinterpret_cast<const uint8_t *>(rows);
  const int64_t feat_blocks = (F + 3) / 4, chunks = (r8_blocks(d) * R8_BLOCK + R8_COLS - 1) / R8_COLS, tasks = windows * chunks;
  const int64_t per_xcd = (tasks + 7) / 8, blocks = (per_xcd + 3) / 4 * 8;
  // a grid's first axis counts less than 2^32 threads; every launch is checked before the first is made
  const int64_t short_blocks = (F + 7) / 8, prepare_blocks = feat_blocks + (positions + 255) / 256;
  const int64_t threads = need == 0 ? short_blocks * 512
                                    : std::max(std::max(prepare_blocks, blocks) * 256, windows * (d <= 256 ? 128 : 512));
  SAE_REQUIRE(threads < (1LL << 32), SAE_ERR_UNSUPPORTED, "rows8_grad_rows: %lld slots of %lld features are too many", (long long)n_slots,
              (long long)F);
  if (need == 0) {
    hipLaunchKernelGGL(rows8_grad_short_kernel, dim3((unsigned)short_blocks, (unsigned)chunks), dim3(512), 0, st, feat_ptr, feat_slot, slot_tok,
                       coef, rec, out, bias_out, F, d);
    return check_launch("rows8_grad_rows");
  }
  hipLaunchKernelGGL(rows8_grad_prepare_kernel, dim3((unsigned)prepare_blocks), dim3(256), 0, st, feat_ptr, feat_slot,
                     slot_tok, coef, pos_feat, pos_tok, pos_coef, out, bias_out, F, d, (uint32_t)feat_blocks, length, (int)n_slots);
#define SAE_R8_GRAD(W)                                                                                                              \
  hipLaunchKernelGGL(rows8_grad_window_kernel<W>, dim3((unsigned)blocks), dim3(256), 0, st, feat_ptr, pos_feat, pos_tok, pos_coef, rec, out, \
                     part, F, d, windows, tasks, (int)n_slots)
  if (length == 32) SAE_R8_GRAD(32);
  else if (length == 64) SAE_R8_GRAD(64);
  else SAE_R8_GRAD(128);
#undef SAE_R8_GRAD
  if (d <= 256)
    hipLaunchKernelGGL(rows8_grad_join_kernel<64>, dim3((unsigned)windows), dim3(128), 0, st, feat_ptr, pos_feat, part, out, F, d, length,
                       (int)n_slots);
  else
    hipLaunchKernelGGL(rows8_grad_join_kernel<256>, dim3((unsigned)windows, (unsigned)((d + 1023) / 1024)), dim3(512), 0, st, feat_ptr, pos_feat,
                       part, out, F, d, length, (int)n_slots);
  return check_launch("rows8_grad_rows");
}
