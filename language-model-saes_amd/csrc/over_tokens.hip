// out[m, n] = sum_t left[t, m] right[t, n]: a product over the token axis of operands that lie [tokens, columns], either of
// them possibly in 8-bit records.
//
// The 256 x 256 tiles of the GEMM kernel need many output tiles, operands whose widths and tokens fill its slabs, and
// floats: for a small or ragged product the copies that bring operands into that form take longer than the product, and a
// dozen tiles leave most of the card idle.  Here a workgroup of four waves owns 64 x 64 outputs (and, where there are few of
// those, a slice of the tokens: slices are joined in order by a second launch); operands are read as they lie, any width, any
// token count, records widened to bf16 (exactly) on their way into LDS.  A slab is multiplied while the next is written to LDS
// and two more are on their way in registers; nothing tests or moves what is still on its way, or the loads would be waited
// for at once (1000 x 1003 x 521 uncut 27 us then, 11 now; 4096 x 4096 x 768 70 and 59; fp32 4096 x 2048 x 2048 334 and 268).
// A small product is a chain: 1000 x 1003 x 521 is 3.9 us of start, first slab and store and 15 slabs of 0.46 us behind it.
//
// bf16 and 8-bit operands: slabs of 64 tokens, v_mfma_f32_16x16x32_bf16, whose fragments (8 consecutive tokens of one column)
// are read across the token rows with ds_read_b64_tr_b16 (see encoder_gemm.hip).  With an fp32 operand: slabs of 32 tokens as
// floats, v_mfma_f32_16x16x4_f32, whose fragments (one token of one column) are read as they lie.
#include "common.h"

namespace sae {

constexpr int OT_TILE = 64;
constexpr int64_t OT_COLUMNS = 1LL << 24;   // of an operand: 64 bf16 or 32 fp32 rows, a slab, stay within 32-bit offsets
constexpr int OT_AHEAD = 2;   // slabs on their way in registers (four: no less time)
typedef __attribute__((ext_vector_type(4))) float ot_f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 ot_bf16x8;
typedef __attribute__((ext_vector_type(4))) short ot_i16x4;
typedef __attribute__((ext_vector_type(8))) short ot_i16x8;
typedef __attribute__((address_space(3))) ot_i16x4 *ot_lds_i16x4;

template <int BYTES, int ALIGN>
struct __attribute__((packed, aligned(ALIGN))) OtBytes {
  uint32_t w[BYTES / 4];
};

// One operand's share of a slab: the slab is cut into chunks of 16 LDS bytes (8 bf16 or 4 fp32 columns of one token), two per
// thread.  fetch() requests them, chunk() widens one.
template <int SRC, bool WIDE>
struct OtOperand {
  static constexpr int W = WIDE ? 4 : 8, TOKENS = WIDE ? 32 : 64, PER_TOKEN = OT_TILE / W;
  static constexpr int BYTES = SRC == SAE_ROWS8 ? W : SRC == SAE_BF16 ? 2 * W : 4 * W;   // of a chunk in memory
  static constexpr int ALIGN = SRC == SAE_ROWS8 ? W : SRC == SAE_BF16 ? 2 : 4;
  const uint8_t *base;
  size_t pitch;
  int behind;         // rows that a chunk reaching past its row's end may touch: 0 where a row is a whole number of chunks
  int valid;          // columns of this thread's chunks that exist (0 .. W; a record's codes reach to a multiple of 32)
  uint32_t at, field_at;
  uint32_t first, first_field, half;   // offsets in a slab: this thread's first chunk, its field, and how far on the second lies
  struct Raw {
    uint32_t w[2][BYTES / 4];
    uint32_t field[2];
  };

  __device__ __forceinline__ void init(const void *p, int64_t cols, int64_t col0) {
    const int64_t col = col0 + (threadIdx.x % PER_TOKEN) * W;
    base = reinterpret_cast<const uint8_t *>(p);
    pitch = dense_row_bytes<SRC>(cols);
    const int64_t end = SRC == SAE_ROWS8 ? r8_blocks(cols) * R8_BLOCK : cols, left = end - col;
    valid = left >= W ? W : left > 0 ? (int)left : 0;
    const int64_t c = valid > 0 ? col : 0;
    at = (uint32_t)(c * (BYTES / W));
    field_at = (uint32_t)(end + (c >> 5));
    behind = SRC == SAE_ROWS8 || cols % W == 0 ? 0 : cols >= W ? 1 : (W - 2) / (int)cols + 1;
    const uint32_t row = (uint32_t)(threadIdx.x / PER_TOKEN) * (uint32_t)pitch;
    first = row + at;
    first_field = row + field_at;
    half = (uint32_t)(256 / PER_TOKEN) * (uint32_t)pitch;
  }
  // A slab all of whose rows exist, and `behind` rows more: a chunk that reaches past its row's end reads on into the rows
  // behind, for columns whose sums are not stored.  No branch and no test of what arrives: the loads stay in flight until
  // chunk() needs them.
  __device__ __forceinline__ void fetch(Raw &r, int64_t t0) const {
    const uint8_t *slab = base + (size_t)t0 * pitch;
    uint32_t where = first, field_where = first_field;
    asm("" : "+v"(where), "+v"(field_where));   // 32-bit offsets to a scalar base, not widened ahead of the loop
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const OtBytes<BYTES, ALIGN> q = *reinterpret_cast<const OtBytes<BYTES, ALIGN> *>(slab + (where + i * half));
#pragma unroll
      for (int e = 0; e < BYTES / 4; ++e) r.w[i][e] = q.w[e];
      if constexpr (SRC == SAE_ROWS8) r.field[i] = slab[field_where + i * half];
    }
  }
  // any slab: rows from n_tokens on and columns that do not exist are zeros
  __device__ __forceinline__ void fetch_ragged(Raw &r, int64_t t0, int64_t n_tokens) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t t = t0 + threadIdx.x / PER_TOKEN + i * (256 / PER_TOKEN);
      const uint8_t *row = base + (size_t)(t < n_tokens ? t : n_tokens - 1) * pitch;
      if (SRC == SAE_ROWS8 || valid == W) {
        const OtBytes<BYTES, ALIGN> q = *reinterpret_cast<const OtBytes<BYTES, ALIGN> *>(row + at);
#pragma unroll
        for (int e = 0; e < BYTES / 4; ++e) r.w[i][e] = q.w[e];
        if constexpr (SRC == SAE_ROWS8) r.field[i] = row[field_at];
      } else {
#pragma unroll
        for (int e = 0; e < BYTES / 4; ++e) {
          if constexpr (SRC == SAE_F32) {
            r.w[i][e] = e < valid ? reinterpret_cast<const uint32_t *>(row + at)[e] : 0u;
          } else {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(row + at) + 2 * e;
            r.w[i][e] = (2 * e < valid ? (uint32_t)h[0] : 0u) | (2 * e + 1 < valid ? (uint32_t)h[1] << 16 : 0u);
          }
        }
      }
      if (t >= n_tokens || valid == 0) {
#pragma unroll
        for (int e = 0; e < BYTES / 4; ++e) r.w[i][e] = 0u;
        r.field[i] = 0u;
      }
    }
  }
  __device__ __forceinline__ u32x4 chunk(const Raw &r, int i) const {
    if constexpr (SRC == SAE_ROWS8) {
      const float step = __uint_as_float(r.field[i] << 23);
      auto value = [&](int e) { return (float)(int8_t)(r.w[i][e / 4] >> (8 * (e % 4))) * step; };
      if constexpr (WIDE) {
        return u32x4{__float_as_uint(value(0)), __float_as_uint(value(1)), __float_as_uint(value(2)), __float_as_uint(value(3))};
      } else {
        return u32x4{pack_bf16x2(value(0), value(1)), pack_bf16x2(value(2), value(3)), pack_bf16x2(value(4), value(5)),
                     pack_bf16x2(value(6), value(7))};
      }
    } else if constexpr (SRC == SAE_BF16 && WIDE) {
      return u32x4{r.w[i][0] << 16, r.w[i][0] & 0xffff0000u, r.w[i][1] << 16, r.w[i][1] & 0xffff0000u};
    } else {
      return u32x4{r.w[i][0], r.w[i][1], r.w[i][2], r.w[i][3]};
    }
  }
};

// byte of chunk c (16 bytes) of token row r in a slab: bf16 rows are 128 bytes, and the chunk pairs are exchanged by the row
// so that the eight rows x 32 bytes which half a wave reads across at once are 256 distinct bytes; fp32 rows of 256 bytes lie
// 320 apart, so that four rows x 64 bytes are
template <bool WIDE>
__device__ __forceinline__ uint32_t ot_lds_at(uint32_t r, uint32_t c) {
  if constexpr (WIDE) return r * 320u + c * 16u;
  else return r * 128u + ((c ^ (((r >> 1) & 1u) | (((r >> 3) & 1u) << 1)) * 2u) * 16u);
}

// four neighbouring outputs from column col on, those that exist
template <int OUT>
__device__ __forceinline__ void ot_store(char *dst, int64_t at, ot_f32x4 v, int64_t col, int64_t n) {
  if constexpr (OUT == SAE_BF16) {
    uint16_t *o = reinterpret_cast<uint16_t *>(dst) + at;
    if (col + 4 <= n) {
      OtBytes<8, 2> q;
      q.w[0] = pack_bf16x2(v[0], v[1]);
      q.w[1] = pack_bf16x2(v[2], v[3]);
      *reinterpret_cast<OtBytes<8, 2> *>(o) = q;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < n) o[e] = f32_to_bf16_bits(v[e]);
    }
  } else {
    float *o = reinterpret_cast<float *>(dst) + at;
    if (col + 4 <= n) {
      OtBytes<16, 4> q;
#pragma unroll
      for (int e = 0; e < 4; ++e) q.w[e] = __float_as_uint(v[e]);
      *reinterpret_cast<OtBytes<16, 4> *>(o) = q;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < n) o[e] = v[e];
    }
  }
}

template <int SRC_L, int SRC_R, int OUT>
__global__ __launch_bounds__(256) void over_tokens_kernel(const void *__restrict__ left, const void *__restrict__ right, int64_t tokens,
                                                          int64_t m, int64_t n, int64_t tokens_per_slice, void *__restrict__ out) {
  constexpr bool WIDE = SRC_L == SAE_F32 || SRC_R == SAE_F32;
  constexpr int TOKENS = WIDE ? 32 : 64, SLAB = WIDE ? 32 * 320 : 64 * 128;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][2][SLAB];   // two slabs of each operand
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  const int64_t m0 = (int64_t)blockIdx.x * OT_TILE, n0 = (int64_t)blockIdx.y * OT_TILE;
  const int64_t t_first = (int64_t)blockIdx.z * tokens_per_slice;
  OtOperand<SRC_L, WIDE> L;
  OtOperand<SRC_R, WIDE> R;
  L.init(left, m, m0);
  R.init(right, n, n0);
  // slabs that fetch() may read; of the slice's others there is one, or two where the last tokens reach into a second
  const int64_t safe = tokens - (L.behind > R.behind ? L.behind : R.behind);
  const int64_t t_end = t_first + tokens_per_slice < safe ? t_first + tokens_per_slice : safe;
  const int steps = t_end > t_first ? (int)((t_end - t_first) / TOKENS) : 0;
  const int64_t t_stop = t_first + tokens_per_slice < tokens ? t_first + tokens_per_slice : tokens;
  auto t_slab = [&](int s) { return t_first + (int64_t)(s < steps ? s : steps - 1) * TOKENS; };   // past the end: the last one again, dropped
  typename OtOperand<SRC_L, WIDE>::Raw l[OT_AHEAD];
  typename OtOperand<SRC_R, WIDE>::Raw r[OT_AHEAD];
  ot_f32x4 acc[2][2];   // [16 columns of right][16 columns of left]
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[i][j][v] = 0.f;

  const int frow = lane & 15, fq = lane >> 4;
  auto stage = [&](int buf, const typename OtOperand<SRC_L, WIDE>::Raw &l, const typename OtOperand<SRC_R, WIDE>::Raw &r) {
    constexpr int P = OtOperand<SRC_L, WIDE>::PER_TOKEN;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t where = ot_lds_at<WIDE>(tid / P + i * (256 / P), tid % P);
      *reinterpret_cast<u32x4 *>(&lds[buf][0][where]) = L.chunk(l, i);
      *reinterpret_cast<u32x4 *>(&lds[buf][1][where]) = R.chunk(r, i);
    }
  };
  auto multiply = [&](int buf) {
    if constexpr (WIDE) {
      const float *ll = reinterpret_cast<const float *>(lds[buf][0]), *lr = reinterpret_cast<const float *>(lds[buf][1]);
#pragma unroll
      for (int k = 0; k < TOKENS; k += 4) {
        float a[2], b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          a[i] = lr[(k + fq) * 80 + wn * 32 + i * 16 + frow];
          b[i] = ll[(k + fq) * 80 + wm * 32 + i * 16 + frow];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[j], acc[i][j], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int k = 0; k < TOKENS; k += 32) {
        ot_bf16x8 a[2], b[2];
        const uint32_t row = k + 8 * fq + (frow >> 2);
        auto across = [&](const uint8_t *slab, uint32_t col) {   // 8 tokens of column col + frow
          const uint32_t c = (col + 4 * (frow & 3)) >> 3, byte = (frow & 1) * 8;
          const ot_i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ot_lds_i16x4)(slab + ot_lds_at<WIDE>(row, c) + byte));
          const ot_i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ot_lds_i16x4)(slab + ot_lds_at<WIDE>(row + 4, c) + byte));
          return __builtin_bit_cast(ot_bf16x8, (ot_i16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          a[i] = across(lds[buf][1], wn * 32 + i * 16);
          b[i] = across(lds[buf][0], wm * 32 + i * 16);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
      }
    }
  };

  // slab s is multiplied while s + 1 is written to LDS and the OT_AHEAD slabs behind it are on their way
  if (steps > 0) {
#pragma unroll
    for (int i = 0; i < OT_AHEAD; ++i) {
      L.fetch(l[i], t_slab(i));
      R.fetch(r[i], t_slab(i));
    }
    stage(0, l[0], r[0]);
    L.fetch(l[0], t_slab(OT_AHEAD));
    R.fetch(r[0], t_slab(OT_AHEAD));
    for (int s = 0; s < steps; s += OT_AHEAD) {
#pragma unroll
      for (int u = 0; u < OT_AHEAD; ++u) {
        if (s + u >= steps) break;   // the same for every thread
        constexpr int A = OT_AHEAD;
        __syncthreads();   // slab s + u is in LDS, and the other buffer has been read by all
        stage((u + 1) & 1, l[(u + 1) % A], r[(u + 1) % A]);
        L.fetch(l[(u + 1) % A], t_slab(s + u + 1 + A));
        R.fetch(r[(u + 1) % A], t_slab(s + u + 1 + A));
        multiply(u & 1);
      }
    }
  }
  for (int64_t t = t_first + (int64_t)steps * TOKENS; t < t_stop; t += TOKENS) {   // the same for every thread
    __syncthreads();
    L.fetch_ragged(l[0], t, tokens);
    R.fetch_ragged(r[0], t, tokens);
    stage(0, l[0], r[0]);
    __syncthreads();
    multiply(0);
  }

  // a lane holds four neighbouring columns of right for one column of left
  char *dst = reinterpret_cast<char *>(out) + (size_t)blockIdx.z * m * n * 4;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t row = m0 + wm * 32 + j * 16 + frow;
    if (row >= m) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t col = n0 + wn * 32 + i * 16 + 4 * fq;
      const ot_f32x4 v = acc[i][j];
      ot_store<OUT>(dst, row * n + col, v, col, n);
    }
  }
}

// out[i] = the slices' sums, added in token order
template <int OUT>
__global__ __launch_bounds__(256) void over_tokens_join_kernel(const float *__restrict__ part, int64_t count, int slices, void *__restrict__ out) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= count) return;
  const int width = count - i < 4 ? (int)(count - i) : 4;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int z = 0; z < slices; ++z) {
    const float *p = part + (int64_t)z * count + i;
    if (width == 4) {
      const OtBytes<16, 4> q = *reinterpret_cast<const OtBytes<16, 4> *>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += __uint_as_float(q.w[e]);
    } else {
      for (int e = 0; e < width; ++e) s[e] += p[e];
    }
  }
  for (int e = 0; e < width; ++e) {
    if constexpr (OUT == SAE_BF16) reinterpret_cast<uint16_t *>(out)[i + e] = f32_to_bf16_bits(s[e]);
    else reinterpret_cast<float *>(out)[i + e] = s[e];
  }
}

static void launch_join(const float *partials, int64_t count, int64_t slices, void *out, int out_dtype, hipStream_t st) {
  const dim3 grid((unsigned)((count + 1023) / 1024));
  if (out_dtype == SAE_BF16) hipLaunchKernelGGL(over_tokens_join_kernel<SAE_BF16>, grid, dim3(256), 0, st, partials, count, (int)slices, out);
  else hipLaunchKernelGGL(over_tokens_join_kernel<SAE_F32>, grid, dim3(256), 0, st, partials, count, (int)slices, out);
}

}  // namespace sae

extern "C" int sae_join_slices(const float *partials, int64_t n_slices, int64_t count, void *out, int out_dtype, void *stream) {
  using namespace sae;
  SAE_REQUIRE(partials && out, SAE_ERR_INVALID_ARG, "join_slices: null pointer");
  SAE_REQUIRE(n_slices > 0 && count > 0, SAE_ERR_INVALID_ARG, "join_slices: sizes must be positive");
  SAE_REQUIRE(out_dtype == SAE_F32 || out_dtype == SAE_BF16, SAE_ERR_INVALID_ARG, "join_slices: bad dtype %d", out_dtype);
  SAE_REQUIRE(n_slices < (1LL << 31) && (count + 1023) / 1024 < (1LL << 24), SAE_ERR_UNSUPPORTED, "join_slices: size too large");
  launch_join(partials, count, n_slices, out, out_dtype, (hipStream_t)stream);
  return check_launch("join_slices");
}

extern "C" int sae_gemm_over_tokens(const void *left, int left_dtype, const void *right, int right_dtype, int64_t tokens, int64_t m, int64_t n,
                                    void *out, int out_dtype, int64_t n_slices, float *partials, void *stream) {
  using namespace sae;
  auto known = [](int t) { return t == SAE_F32 || t == SAE_BF16 || t == SAE_ROWS8; };
  SAE_REQUIRE(left && right && out, SAE_ERR_INVALID_ARG, "gemm_over_tokens: null pointer");
  SAE_REQUIRE(tokens > 0 && m > 0 && n > 0 && n_slices > 0, SAE_ERR_INVALID_ARG, "gemm_over_tokens: sizes must be positive");
  SAE_REQUIRE(known(left_dtype) && known(right_dtype), SAE_ERR_INVALID_ARG, "gemm_over_tokens: bad dtype %d, %d", left_dtype, right_dtype);
  const bool wide = left_dtype == SAE_F32 || right_dtype == SAE_F32;
  SAE_REQUIRE(out_dtype == SAE_F32 || (out_dtype == SAE_BF16 && !wide), SAE_ERR_INVALID_ARG, "gemm_over_tokens: bad out_dtype %d", out_dtype);
  const int64_t slab = wide ? 32 : 64, slabs = (tokens + slab - 1) / slab;
  // left's tiles are the grid's x, right's its y, which ends at 65535
  SAE_REQUIRE(m <= OT_COLUMNS && n <= 65535LL * OT_TILE && slabs < (1LL << 30), SAE_ERR_UNSUPPORTED, "gemm_over_tokens: size too large");
  SAE_REQUIRE(n_slices == 1 || (m * n + 1023) / 1024 < (1LL << 24), SAE_ERR_UNSUPPORTED, "gemm_over_tokens: too many outputs for slices");
  SAE_REQUIRE(n_slices <= 65535 && n_slices <= slabs && (n_slices == 1 || partials), SAE_ERR_INVALID_ARG,
              "gemm_over_tokens: %lld slices of %lld slabs (with partial results for more than one)", (long long)n_slices, (long long)slabs);
  SAE_REQUIRE((left_dtype != SAE_ROWS8 || ((uintptr_t)left & 15) == 0) && (right_dtype != SAE_ROWS8 || ((uintptr_t)right & 15) == 0),
              SAE_ERR_INVALID_ARG, "gemm_over_tokens: records must be 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  const int64_t per_slice = (slabs + n_slices - 1) / n_slices * slab, slices = (tokens + per_slice - 1) / per_slice;
  const dim3 grid((unsigned)((m + OT_TILE - 1) / OT_TILE), (unsigned)((n + OT_TILE - 1) / OT_TILE), (unsigned)slices);
  void *to = slices > 1 ? partials : out;
  const bool low = out_dtype == SAE_BF16 && slices == 1;
#define SAE_OT(L, R, O) hipLaunchKernelGGL((over_tokens_kernel<L, R, O>), grid, dim3(256), 0, st, left, right, tokens, m, n, per_slice, to)
#define SAE_OT_LOW(L, R) \
  if (left_dtype == L && right_dtype == R) { if (low) SAE_OT(L, R, SAE_BF16); else SAE_OT(L, R, SAE_F32); }
#define SAE_OT_WIDE(L, R) \
  if (left_dtype == L && right_dtype == R) SAE_OT(L, R, SAE_F32);
  SAE_OT_LOW(SAE_BF16, SAE_BF16)
  SAE_OT_LOW(SAE_BF16, SAE_ROWS8)
  SAE_OT_LOW(SAE_ROWS8, SAE_BF16)
  SAE_OT_LOW(SAE_ROWS8, SAE_ROWS8)
  SAE_OT_WIDE(SAE_F32, SAE_F32)
  SAE_OT_WIDE(SAE_F32, SAE_BF16)
  SAE_OT_WIDE(SAE_F32, SAE_ROWS8)
  SAE_OT_WIDE(SAE_BF16, SAE_F32)
  SAE_OT_WIDE(SAE_ROWS8, SAE_F32)
#undef SAE_OT_WIDE
#undef SAE_OT_LOW
#undef SAE_OT
  if (slices > 1) launch_join(partials, m * n, slices, out, out_dtype, st);
  return check_launch("gemm_over_tokens");
}
