// Softmax attention without a stored probability matrix: shared pieces of the forward, gradient and single-token kernels (internal header).
//
//   s_ij = scale q_i . k_j   (seen: j < k_lens[b], and j <= q_start[b] + i when causal)      l_i = log sum_j exp s_ij
//   o_i  = sum_j p_ij v_j,  p_ij = exp(s_ij - l_i)
//   D_i  = do_i . o_i,  ds_ij = p_ij (do_i . v_j - D_i):   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// Every product runs on 32 x 32 matrix instructions, and every kernel arranges them the same way:
//   * the tile that a wave OWNS (32 queries, or 32 keys in the key gradient) is the COLUMN side: lane l holds column l & 31, so a softmax
//     statistic is one number per lane and a reduction over the other side is in-lane plus one exchange between the wave's halves;
//   * the tile that STREAMS through LDS is the row side, read in one of two ways: `row_frag` (a row's consecutive elements: products that
//     sum over the head dimension) or `col_frag` (a column's elements at 32 consecutive rows: products that sum over the streamed rows);
//   * the 16 results of a lane sit at rows 8 (i >> 2) + 4 (l >> 5) + (i & 3), i = 0 .. 15.  A product over those rows may take them in any
//     order as long as both operands agree, so the accumulator registers ARE the second product's operand: nothing moves between lanes,
//     and col_frag fetches rows in that order (16-bit types: the transposing 8-byte LDS read delivers exactly 4 consecutive rows of a column).
// LDS rows: 64-byte units, an odd number of them, and 16-byte chunk c of row r stored at c ^ ((r >> 2) & 3): the 16 rows of a 16-byte
// read and the 4 rows of a transposing read then fall on different banks.
#pragma once
#include "icg_common.h"
#include <math.h>

typedef float at_f16v __attribute__((ext_vector_type(16)));
typedef float at_f4 __attribute__((ext_vector_type(4)));
typedef short at_s4 __attribute__((ext_vector_type(4)));
typedef short at_s8 __attribute__((ext_vector_type(8)));
typedef _Float16 at_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 at_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 at_b8 __attribute__((ext_vector_type(8)));
typedef float at_f2 __attribute__((ext_vector_type(2)));
typedef unsigned at_u4 __attribute__((ext_vector_type(4)));

#define AT_LOWEST (-3.402823466e38f)      // a running maximum starts here: exp2(-inf - AT_LOWEST) is 0, where -inf - -inf has no value
#define AT_LOG2E 1.44269504088896340736f
#define AT_LN2 0.69314718055994530942f

struct AttnP {
  const void *q, *k, *v;
  const int *k_lens, *q_start;
  int B, Lq, Lk, H, G, d, dv;               // H query heads, G of them to a key head
  int64_t q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh;
  float scale;
  int causal;                               // (every row of q, k, v, o, do starts at a multiple of 16 bytes and holds whole 16-byte chunks)
  // forward
  void *o, *o_low;                          // o_low: what the rounding of o took away, NULL if nobody asks
  float* lse;
  float* part;                              // split over the keys: [split][B][H][Lq] rows of dv sums, then their (maximum, sum) pairs
  int nsplit, keys_per_split;
  // gradient
  const void* dout;
  int64_t do_sb, do_sl, do_sh;
  const float *stat;                        // [3][B][H][Lq]: l_i log2 e (less the shift of p), D_i, |do_i|; SCALED: then [B][Hk][ceil(Lk / 128)]: largest |v_j|
  void *dq, *dk, *dv_out;
  int tiles;                                // 32- or 128-row tiles of one head
  int64_t work;                             // workgroups in all
};

template <typename T> struct at_type;
template <> struct at_type<float> {
  typedef at_f4 frag;
  static constexpr int KSTEP = 8, P_SHIFT = 0;
  static constexpr bool SCALED = false;
  // whether step t of a sum over the head dimension holds elements: a step is 256 cycles here, worth a scalar branch
  static __device__ __forceinline__ bool step(int t, int len) { return KSTEP * t < len; }
  static __device__ __forceinline__ at_f16v mma(frag a, frag b, at_f16v c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], b[s], c, 0, 0, 0);
    return c;
  }
  // registers KSTEP / 2 t .. of an accumulator as an operand
  static __device__ __forceinline__ frag pack(const at_f16v& x, int t) { return frag{x[4 * t], x[4 * t + 1], x[4 * t + 2], x[4 * t + 3]}; }
};
template <> struct at_type<__bf16> {
  typedef at_b8 frag;
  static constexpr int KSTEP = 16, P_SHIFT = 0;
  static constexpr bool SCALED = false;
  static __device__ __forceinline__ bool step(int, int) { return true; }     // (32 cycles: the branch would cost more than the zeros)
  static __device__ __forceinline__ at_f16v mma(frag a, frag b, at_f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ frag pack(const at_f16v& x, int t) {
    frag f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const at_b2 c = __builtin_convertvector((at_f2{x[8 * t + 2 * j], x[8 * t + 2 * j + 1]}), at_b2);
      f[2 * j] = c[0], f[2 * j + 1] = c[1];
    }
    return f;
  }
};
// fp16 ends at 6e-8 and at 65504: in the gradient p is held 2^6 times as large, and ds is scaled by a power of two (undone on the 32-bit
// sums, exactly).  |p_j (do . v_j - do . o)| = p_j |sum_k p_k do . (v_j - v_k)| <= p_j (1 - p_j) |do| 2 max|v| <= |do| max|v| / 2, so the power
// that brings |do| max|v| to [512, 1024) holds ds below 2^15 for any values that the type has, with a factor of 2 to spare for the roundings
// of p and D; what is lost below is half of 2^-24 in that scale, 2^-40 |do| max|v|.
template <> struct at_type<_Float16> {
  typedef at_h8 frag;
  static constexpr int KSTEP = 16, P_SHIFT = 6;
  static constexpr bool SCALED = true;
  static __device__ __forceinline__ bool step(int, int) { return true; }
  static __device__ __forceinline__ at_f16v mma(frag a, frag b, at_f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ frag pack(const at_f16v& x, int t) {
    frag f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const at_h2 c = __builtin_convertvector((at_f2{x[8 * t + 2 * j], x[8 * t + 2 * j + 1]}), at_h2);
      f[2 * j] = c[0], f[2 * j + 1] = c[1];
    }
    return f;
  }
};

// a streamed tile of `ROWS` rows of `E` elements in LDS
template <typename T, int E>
struct at_tile {
  static constexpr int STRIDE = 64 * ((E * (int)sizeof(T) / 64) | 1);
  static constexpr int CHUNKS = E * (int)sizeof(T) / 16, PER = 16 / (int)sizeof(T);
  static_assert((E * sizeof(T)) % 64 == 0, "whole 64-byte units");
  static __device__ __forceinline__ int at(int row, int chunk) { return row * STRIDE + ((chunk ^ ((row >> 2) & 3)) << 4); }
};

// The registers of a streamed tile on its way from memory to LDS.  Loads go through a buffer descriptor of the tile's rows: a thread's
// offsets within a tile never change, so a tile costs no address arithmetic in the lanes, and rows past the end read as zeros by the
// descriptor's bound.  (A row's stride is at least its length, see at_row_ok.)
struct at_rows {
  uint64_t base;
  uint32_t stride, len;                     // bytes
  __device__ __forceinline__ at_rows(const void* p, int64_t stride_, int len_, int size)
      : stride((uint32_t)(stride_ * size)), len((uint32_t)(len_ * size)) {
    const uint64_t a = (uint64_t)p;
    // (the builtin returns a signed int: without the casts a low half from 2^31 on would extend its sign over the high half)
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)), lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    base = ((uint64_t)hi << 32) | lo;
  }
};

template <typename T, int E, int ROWS, int THREADS>
struct at_stage {
  typedef at_tile<T, E> tile;
  static constexpr int N = (ROWS * tile::CHUNKS + THREADS - 1) / THREADS;
  static constexpr bool EXACT = (ROWS * tile::CHUNKS) % THREADS == 0;
  at_u4 r[N];
  uint32_t off[N];
  __device__ __forceinline__ at_stage(const at_rows& m, int tid) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = tid + n * THREADS, row = i / tile::CHUNKS, c = i - row * tile::CHUNKS;
      off[n] = (EXACT || row < ROWS) && (uint32_t)c * 16u < m.len ? (uint32_t)row * m.stride + (uint32_t)c * 16u : 0x80000000u;
    }
  }
  __device__ __forceinline__ void fetch(const at_rows& m, int row0, int rows_end) {
    const int rows = min(rows_end - row0, ROWS);
    const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)(m.base + (uint64_t)row0 * m.stride), 0,
                                                                       (int)((uint32_t)(rows - 1) * m.stride + m.len), 0x00027000);
#pragma unroll
    for (int n = 0; n < N; ++n) r[n] = __builtin_amdgcn_raw_buffer_load_b128(d, off[n], 0, 0);
  }
  __device__ __forceinline__ void put(char* lds, int tid) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = tid + n * THREADS, row = i / tile::CHUNKS, c = i - row * tile::CHUNKS;
      if (EXACT || row < ROWS) *reinterpret_cast<at_u4*>(lds + tile::at(row, c)) = r[n];
    }
  }
};

// lane-constant parts of the fragment addresses
template <typename T, int E>
struct at_reader {
  typedef at_tile<T, E> tile;
  typedef typename at_type<T>::frag frag;
  int row_[2], col_[2];
  __device__ __forceinline__ explicit at_reader(int lane) {
    const int m = lane & 31, h = lane >> 5;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      row_[u] = m * tile::STRIDE + (((2 * u + h) ^ ((m >> 2) & 3)) << 4);
      if constexpr (sizeof(T) == 2) {       // u: which 4 of the 8 rows of an operand
        const int c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        col_[u] = (8 * u + 4 * h + ((lane & 15) >> 2)) * tile::STRIDE + ((c ^ (2 * u + h)) << 4) + ((lane & 1) << 3);
      } else {                              // u: parity of the 8-row step
        const int c = m >> 2;
        col_[u] = (4 * h) * tile::STRIDE + ((c ^ (2 * u + h)) << 4) + ((m & 3) << 2);
      }
    }
  }
  // element KSTEP t + KSTEP / 2 h .. of row row0 + (lane & 31)
  __device__ __forceinline__ frag row_frag(const char* lds, int row0, int t) const {
    return *reinterpret_cast<const frag*>(lds + row_[t & 1] + row0 * tile::STRIDE + (t >> 1) * 64);
  }
  // column 32 ct + (lane & 31) at the rows row0 + KSTEP t .. in accumulator order
  __device__ __forceinline__ frag col_frag(const char* lds, int row0, int ct, int t) const {
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) at_s4 lds4;
      const char* p = lds + (row0 + 16 * t) * tile::STRIDE + ct * 64;
      const at_s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + col_[0]));
      const at_s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + col_[1]));
      const at_s8 ab = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(frag, ab);
    } else {
      const char* p = lds + (row0 + 8 * t) * tile::STRIDE + ct * 128 + col_[t & 1];
      frag f;
#pragma unroll
      for (int s = 0; s < 4; ++s) f[s] = *reinterpret_cast<const float*>(p + s * tile::STRIDE);
      return f;
    }
  }
};

// the wave's own 32 rows as column-side operands, straight from memory (used once per workgroup)
template <typename T, int E>
__device__ __forceinline__ void at_own(typename at_type<T>::frag (&f)[E / at_type<T>::KSTEP], const T* row, bool valid, int len, int h) {
  constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
  for (int t = 0; t < E / at_type<T>::KSTEP; ++t) {
    at_u4 r = {0u, 0u, 0u, 0u};
    const int c = (2 * t + h) * PER;
    if (valid && c < len) r = *reinterpret_cast<const at_u4*>(row + c);
    f[t] = __builtin_bit_cast(typename at_type<T>::frag, r);
  }
}

__device__ __forceinline__ float at_other_half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float at_both_halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int at_row_of(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// four consecutive elements of an output row (len is a multiple of 4)
template <typename T>
__device__ __forceinline__ void at_store4(T* row, int c, int len, float a, float b, float e, float f) {
  if (c >= len) return;
  const T x[4] = {(T)a, (T)b, (T)e, (T)f};
  if constexpr (sizeof(T) == 2) { uint2 w; __builtin_memcpy(&w, x, 8); *reinterpret_cast<uint2*>(row + c) = w; }
  else { at_u4 w; __builtin_memcpy(&w, x, 16); *reinterpret_cast<at_u4*>(row + c) = w; }
}

// A mean of fp16 values is held to their range: p is rounded for the product with v and not in its sum, so the quotient can pass 65504 by a
// step of 2^-11, from where a conversion gives inf.  (A sum that is not finite has a value that is not, and stays.)
template <typename T>
__device__ __forceinline__ float at_hold(float x) {
  if constexpr (at_type<T>::SCALED) return __builtin_isfinite(x) ? __builtin_amdgcn_fmed3f(x, -65504.f, 65504.f) : x;
  return x;
}

// ... of the output, and of what its rounding took away
template <typename T>
__device__ __forceinline__ void at_store_out(const AttnP& p, int64_t row, int c, float a, float b, float e, float f) {
  a = at_hold<T>(a), b = at_hold<T>(b), e = at_hold<T>(e), f = at_hold<T>(f);
  at_store4<T>(reinterpret_cast<T*>(p.o) + row * p.dv, c, p.dv, a, b, e, f);
  if (p.o_low)
    at_store4<T>(reinterpret_cast<T*>(p.o_low) + row * p.dv, c, p.dv, a - (float)(T)a, b - (float)(T)b, e - (float)(T)e, f - (float)(T)f);
}

__device__ __forceinline__ int at_keys(const AttnP& p, int b) { return p.k_lens ? min(max(p.k_lens[b], 0), p.Lk) : p.Lk; }
// position of query 0 (clamped so that adding a query or key index cannot overflow)
__device__ __forceinline__ int at_start(const AttnP& p, int b) { return p.q_start ? min(max(p.q_start[b], -(1 << 30)), 1 << 30) : p.Lk - p.Lq; }

// A dimension of a grid holds fewer than 2^32 threads (the runtime does not refuse more, it leaves some out): rows of
// 2^22 workgroups
__device__ __forceinline__ int64_t at_block() { return blockIdx.x + (int64_t)gridDim.x * blockIdx.y; }
static inline dim3 at_grid(int64_t n) { return n <= (1 << 22) ? dim3((unsigned)n) : dim3(1u << 22, (unsigned)icg_cdiv(n, 1 << 22)); }

// Workgroups go to the 8 dies in turn; a run of consecutive work items per die keeps one head's keys in one die's L2.
// (negative for a workgroup behind the last item)
__device__ __forceinline__ int64_t at_work_item(int64_t n) {
  const int64_t i = at_block(), per = n >> 3, rest = n & 7;
  if (i >= n) return -1;
  const int64_t x = i & 7, j = i >> 3;
  return x * per + min(x, rest) + j;
}

int at_fwd_f32(const AttnP&, bool tokens, hipStream_t);
int at_fwd_f16(const AttnP&, bool tokens, hipStream_t);
int at_fwd_bf16(const AttnP&, bool tokens, hipStream_t);
int at_bwd_f32(const AttnP& dq, const AttnP& dkv, float* stat, hipStream_t);
int at_bwd_f16(const AttnP& dq, const AttnP& dkv, float* stat, hipStream_t);
int at_bwd_bf16(const AttnP& dq, const AttnP& dkv, float* stat, hipStream_t);
// (DP, DVP): the head dimensions a kernel is built for.  A head takes the first pair that covers it: equal dimensions, and values up to four
// times as wide as the keys, as the image models' blocks have them.
#define AT_FOR_HEAD(d, dv, RUN)                               \
  if (d <= 32 && dv <= 32) { RUN(32, 32); }                   \
  else if (d <= 32 && dv <= 96) { RUN(32, 96); }              \
  else if (d <= 64 && dv <= 64) { RUN(64, 64); }              \
  else if (d <= 32 && dv <= 128) { RUN(32, 128); }            \
  else if (d <= 96 && dv <= 96) { RUN(96, 96); }              \
  else if (d <= 64 && dv <= 192) { RUN(64, 192); }            \
  else if (d <= 128 && dv <= 128) { RUN(128, 128); }          \
  else { RUN(64, 256); }
