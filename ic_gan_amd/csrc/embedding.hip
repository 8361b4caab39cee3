// Embedding lookup with scaling, and its dense gradient by sorted tokens.
//
//   out[i] = s W[t_i]        dW[v] = s sum over i with t_i = v of dout[i], in the order of i, 32-bit sums, one rounding; rows without tokens are zero
//
// Bound by memory: n rows read and written forward; n rows read and V rows written in the gradient.  The order of the tokens is found without
// atomics and without a general sort: a workgroup owns a run of tokens, scans the whole list (it stays in L2), and learns in one
// sweep how often each of its tokens occurs in each wave's share of the list and how many entries belong to smaller tokens, which is where its
// part of the sorted list begins; a second sweep puts the positions in place.  Tokens that occur often are summed in pieces of
// EMB_CHUNK list entries first.  What one wave does in turn still grows with its token: n / EMB_CHUNK sums of pieces for a token that fills
// the list, and up to EMB_FEW entries, 8 loads at a time, where the list is short and not sorted.
// Measured (kernel trace), 50000 x 2048 bf16, 16384 skewed tokens: lookup 24 us (5.6 TB/s), order 16 us (the busiest run's entries, one after the
// other), pieces 13 us, rows 70 us (4.0 TB/s); 1000 x 128 fp32, 64 tokens: 3 us each way.
#include "icg_common.h"

typedef unsigned em_u4 __attribute__((ext_vector_type(4)));

struct EmbP {
  const void *idx, *w, *dout;
  void *out, *dw;
  int64_t n, V, D, pad;               // pad: a token whose gradient is zero (-1: none)
  int idx64;
  float scale;
  int run;                            // tokens per workgroup of the sort
  int *order, *start;                 // [n] positions by token; [V + 1]
  float* part;                        // [ceil(n / EMB_CHUNK)][2][D]
};

constexpr int EMB_CHUNK = 32;         // list entries of one piece
constexpr int EMB_RUN = 1024;         // most tokens a workgroup of the sort owns (64 KB of counts)
constexpr int EMB_FEW = 1024;         // up to here the gradient scans the list per row, in one launch

template <typename T, int VEC> struct em_vec { T e[VEC]; };
template <typename T, int VEC>
__device__ __forceinline__ em_vec<T, VEC> em_load(const T* p) {
  em_vec<T, VEC> r;
  if constexpr (VEC == 1) r.e[0] = *p;
  else { const em_u4 w = *reinterpret_cast<const em_u4*>(p); __builtin_memcpy(&r, &w, 16); }
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void em_store(T* p, const em_vec<T, VEC>& r) {
  if constexpr (VEC == 1) *p = r.e[0];
  else { em_u4 w; __builtin_memcpy(&w, &r, 16); *reinterpret_cast<em_u4*>(p) = w; }
}
__device__ __forceinline__ int64_t em_token(const EmbP& p, int64_t i) {
  return p.idx64 ? reinterpret_cast<const int64_t*>(p.idx)[i] : (int64_t)reinterpret_cast<const int*>(p.idx)[i];
}

// a token outside the table gives a row of NaN
template <typename T, int VEC>
__global__ __launch_bounds__(256) void icg_embedding_fwd_kernel(EmbP p) {
  const int64_t cols = p.D / VEC, all = p.n * cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / cols, c = (i - row * cols) * VEC, t = em_token(p, row);
    em_vec<T, VEC> o;
    if ((uint64_t)t < (uint64_t)p.V) {
      const em_vec<T, VEC> v = em_load<T, VEC>(reinterpret_cast<const T*>(p.w) + t * p.D + c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) o.e[j] = (T)((float)v.e[j] * p.scale);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) o.e[j] = (T)__builtin_nanf("");
    }
    em_store<T, VEC>(reinterpret_cast<T*>(p.out) + row * p.D + c, o);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void em_add(float (&a)[VEC], const EmbP& p, int64_t row, int64_t c) {
  const em_vec<T, VEC> v = em_load<T, VEC>(reinterpret_cast<const T*>(p.dout) + row * p.D + c);
#pragma unroll
  for (int j = 0; j < VEC; ++j) a[j] += (float)v.e[j];
}
template <typename T, int VEC>
__device__ __forceinline__ void em_write(const float (&a)[VEC], const EmbP& p, int64_t v, int64_t c) {
  em_vec<T, VEC> o;
#pragma unroll
  for (int j = 0; j < VEC; ++j) o.e[j] = (T)(a[j] * p.scale);
  em_store<T, VEC>(reinterpret_cast<T*>(p.dw) + v * p.D + c, o);
}

// few tokens: the list in LDS, a wave per column tile of a row of the table finds its entries by ballot and adds them in order, up to 8 loads in
// flight
template <typename T, int VEC>
__global__ __launch_bounds__(256) void icg_embedding_bwd_few_kernel(EmbP p, int tiles) {
  __shared__ int list[EMB_FEW];
  const int n = (int)p.n;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int64_t t = em_token(p, i);
    list[i] = (uint64_t)t < (uint64_t)p.V && t != p.pad ? (int)t : -1;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  for (int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); w < p.V * tiles; w += (int64_t)gridDim.x * 4) {
    const int64_t v = w / tiles, c = ((w - v * tiles) * 64 + lane) * VEC;
    float a[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) a[j] = 0.f;
    for (int i0 = 0; i0 < n; i0 += 64) {
      unsigned long long hit = __ballot(i0 + lane < n && list[min(i0 + lane, n - 1)] == (int)v);
      while (hit) {
        em_vec<T, VEC> x[8];
        int m = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (hit) {
            const int i = i0 + __builtin_ctzll(hit);
            hit &= hit - 1, ++m;
            if (c < p.D) x[q] = em_load<T, VEC>(reinterpret_cast<const T*>(p.dout) + (int64_t)i * p.D + c);
          }
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < m)
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] += (float)x[q].e[j];
      }
    }
    if (c < p.D) em_write<T, VEC>(a, p, v, c);
  }
}

// ---- the positions in the order of their tokens
constexpr int EMB_WAVES = 16, EMB_KEEP = 16;
__global__ __launch_bounds__(64 * EMB_WAVES) void icg_embedding_sort_kernel(EmbP p) {
  __shared__ int count[EMB_WAVES * EMB_RUN];               // [wave][token]: occurrences, then the next place
  __shared__ int less[EMB_WAVES], sums[EMB_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t v0 = (int64_t)blockIdx.x * p.run;
  const int own = (int)min((int64_t)p.run, p.V - v0);
  for (int i = tid; i < EMB_WAVES * p.run; i += 64 * EMB_WAVES) count[i] = 0;
  __syncthreads();
  const int64_t share = (p.n + EMB_WAVES * 64 - 1) / (EMB_WAVES * 64) * 64, i0 = wv * share, i1 = min(i0 + share, p.n);
  int below = 0;
  // a token of this workgroup's run, or -1
  auto local = [&](int64_t i) -> int {
    const int64_t t = i < i1 ? em_token(p, i) : -1;
    const bool valid = (uint64_t)t < (uint64_t)p.V && t != p.pad;
    below += __builtin_popcountll(__ballot(valid && t < v0));
    return valid && t >= v0 && t < v0 + own ? (int)(t - v0) : -1;
  };
  auto tally = [&](int u) {
    unsigned long long rest = __ballot(u >= 0);
    while (rest) {                                         // one distinct token at a time
      const int first = __builtin_ctzll(rest);
      const unsigned long long same = __ballot(u == __builtin_amdgcn_readlane(u, first));
      if (lane == first) count[wv * p.run + u] += __builtin_popcountll(same);
      rest &= ~same;
    }
    icg_wave_lds_sync();
  };
  int kept[EMB_KEEP];                                      // the share's first tokens stay in registers for the second sweep
#pragma unroll
  for (int k = 0; k < EMB_KEEP; ++k) kept[k] = i0 + 64 * k < i1 ? local(i0 + 64 * k + lane) : -1;
#pragma unroll
  for (int k = 0; k < EMB_KEEP; ++k) tally(kept[k]);
  for (int64_t i = i0 + 64 * EMB_KEEP; i < i1; i += 64) tally(local(i + lane));
  if (lane == 0) less[wv] = below;
  __syncthreads();
  // places: tokens in order, and within a token the waves in order.  Thread t takes token t (run <= 1024 = the threads).
  int mine = 0;
  if (tid < own)
#pragma unroll
    for (int w = 0; w < EMB_WAVES; ++w) mine += count[w * p.run + tid];
  int at = mine;                                           // inclusive sum over the wave
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int o = __shfl_up(at, s, 64);
    if (lane >= s) at += o;
  }
  if (lane == 63) sums[wv] = at;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < EMB_WAVES; ++w) base += less[w] + (w < wv ? sums[w] : 0);
  at += base - mine;
  if (tid < own) {
    p.start[v0 + tid] = at;
    int next = at;
#pragma unroll
    for (int w = 0; w < EMB_WAVES; ++w) {
      const int k = count[w * p.run + tid];
      count[w * p.run + tid] = next;
      next += k;
    }
    if (v0 + tid == p.V - 1) p.start[p.V] = next;
  }
  __syncthreads();
  auto place = [&](int64_t i, int u) {
    unsigned long long rest = __ballot(u >= 0);
    while (rest) {                                         // one distinct token at a time, its entries in lane order
      const int first = __builtin_ctzll(rest);
      const int tok = __builtin_amdgcn_readlane(u, first);
      const unsigned long long same = __ballot(u == tok);
      int* next = &count[wv * p.run + tok];
      const int at = *next;
      icg_wave_lds_sync();
      if (u == tok) p.order[at + __builtin_popcountll(same & ((1ull << lane) - 1))] = (int)(i + lane);
      if (lane == first) *next = at + __builtin_popcountll(same);
      icg_wave_lds_sync();
      rest &= ~same;
    }
  };
#pragma unroll
  for (int k = 0; k < EMB_KEEP; ++k) place(i0 + 64 * k, kept[k]);
  for (int64_t i = i0 + 64 * EMB_KEEP; i < i1; i += 64) place(i, local(i + lane));
}

// a token that fills more than a piece: the sum of its entries in piece k is part[k][0] if it began in an earlier piece, else part[k][1]
// (at most one token of each kind meets a piece)
template <typename T, int VEC>
__global__ __launch_bounds__(64) void icg_embedding_bwd_piece_kernel(EmbP p) {
  const int total = p.start[p.V];
  const int64_t k = blockIdx.x;
  const int e0 = (int)(k * EMB_CHUNK), e1 = min(e0 + EMB_CHUNK, total);
  if (e0 >= total) return;
  const int lane = threadIdx.x;
  const int64_t c = (int64_t)blockIdx.y * 64 * VEC + lane * VEC;
  const int side = blockIdx.z;
  const int64_t t = em_token(p, p.order[side == 0 ? e0 : e1 - 1]);
  const int b = p.start[t], e = p.start[t + 1];
  if (e - b <= EMB_CHUNK || (side == 0) != (b < e0) || c >= p.D) return;
  float a[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) a[j] = 0.f;
  int i = max(b, e0);
  const int to = min(e, e1);
  for (; i + 8 <= to; i += 8) {
    em_vec<T, VEC> v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = em_load<T, VEC>(reinterpret_cast<const T*>(p.dout) + (int64_t)p.order[i + q] * p.D + c);
#pragma unroll
    for (int q = 0; q < 8; ++q)
#pragma unroll
      for (int j = 0; j < VEC; ++j) a[j] += (float)v[q].e[j];
  }
  for (; i < to; ++i) em_add<T, VEC>(a, p, p.order[i], c);
  float* out = p.part + (k * 2 + side) * p.D + c;
#pragma unroll
  for (int j = 0; j < VEC; ++j) out[j] = a[j];
}

// a wave per column tile of a row of the table: the longest piece of work is a tile of EMB_CHUNK entries, or of one sum per EMB_CHUNK entries
template <typename T, int VEC>
__global__ __launch_bounds__(256) void icg_embedding_bwd_row_kernel(EmbP p, int tiles) {
  const int64_t w = (blockIdx.x + (int64_t)gridDim.x * blockIdx.y) * 4 + (threadIdx.x >> 6), v = w / tiles;
  const int64_t c = ((w - v * tiles) * 64 + (threadIdx.x & 63)) * VEC;
  if (v >= p.V || c >= p.D) return;
  const int b = p.start[v], e = p.start[v + 1];
  float a[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) a[j] = 0.f;
  if (e - b <= EMB_CHUNK) {
    const T* dout = reinterpret_cast<const T*>(p.dout) + c;
    int i = b;
    for (; i + 4 <= e; i += 4) {
      em_vec<T, VEC> x[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = em_load<T, VEC>(dout + (int64_t)p.order[i + q] * p.D);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j] += (float)x[q].e[j];
    }
    for (; i < e; ++i) em_add<T, VEC>(a, p, p.order[i], c);
  } else {
    const int k0 = b / EMB_CHUNK, k1 = (e - 1) / EMB_CHUNK;
    const float* in = p.part + c;
#pragma unroll 4
    for (int k = k0; k <= k1; ++k) {
      const float* q = in + ((int64_t)k * 2 + (b < k * EMB_CHUNK ? 0 : 1)) * p.D;
#pragma unroll
      for (int j = 0; j < VEC; ++j) a[j] += q[j];
    }
  }
  em_write<T, VEC>(a, p, v, c);
}
namespace {

// A dimension of a grid holds fewer than 2^32 threads, and the runtime does not refuse more, it leaves some out.  The lookup and the gradient of
// few tokens stride over what a capped grid leaves; the rows of the sorted gradient (a loop around them costs 4 %) take a second dimension.
unsigned em_blocks(int64_t n) { return (unsigned)(n < ICG_GRID_CAP ? n : ICG_GRID_CAP); }

// (column tiles of 64 elements at the narrowest are a grid's second dimension: at most 32768 of them)
bool em_shape_ok(int64_t n, int64_t V, int64_t D, int dtype) {
  return n > 0 && n < 0x7fffff00LL && V > 0 && V < 0x7fffff00LL && D > 0 && D < (1 << 21) && dtype >= 0 && dtype <= 2;
}
size_t em_align(size_t x) { return (x + 15) / 16 * 16; }

template <typename T, int VEC>
int em_fwd(const EmbP& p, hipStream_t st) {
  hipLaunchKernelGGL((icg_embedding_fwd_kernel<T, VEC>), dim3(em_blocks(icg_cdiv(p.n * (p.D / VEC), 256))), dim3(256), 0, st, p);
  return icg_check_launch();
}

template <typename T, int VEC>
int em_bwd(const EmbP& p, hipStream_t st) {
  const int64_t tiles = icg_cdiv(p.D, 64 * VEC), blocks = icg_cdiv(p.V * tiles, 4), wide = blocks < (1 << 22) ? blocks : 1 << 22;
  if (p.n <= EMB_FEW) {
    hipLaunchKernelGGL((icg_embedding_bwd_few_kernel<T, VEC>), dim3(em_blocks(blocks)), dim3(256), 0, st, p, (int)tiles);
    return icg_check_launch();
  }
  hipLaunchKernelGGL(icg_embedding_sort_kernel, dim3((unsigned)icg_cdiv(p.V, p.run)), dim3(64 * EMB_WAVES), 0, st, p);
  if (const int e = icg_check_launch()) return e;
  hipLaunchKernelGGL((icg_embedding_bwd_piece_kernel<T, VEC>), dim3((unsigned)icg_cdiv(p.n, EMB_CHUNK), (unsigned)icg_cdiv(p.D, 64 * VEC), 2), dim3(64), 0, st, p);
  if (const int e = icg_check_launch()) return e;
  ICG_REQUIRE(icg_cdiv(blocks, wide) < 65536);
  hipLaunchKernelGGL((icg_embedding_bwd_row_kernel<T, VEC>), dim3((unsigned)wide, (unsigned)icg_cdiv(blocks, wide)), dim3(256), 0, st, p, (int)tiles);
  return icg_check_launch();
}

}  // namespace

extern "C" int icg_embedding_fwd(const void* idx, const void* weight, void* out, int64_t n, int64_t V, int64_t D, float scale, int idx64, int dtype,
                                 void* stream) {
  ICG_REQUIRE(idx && weight && out && em_shape_ok(n, V, D, dtype));
  EmbP p = {};
  p.idx = idx, p.w = weight, p.out = out, p.n = n, p.V = V, p.D = D, p.idx64 = idx64 != 0, p.scale = scale;
  const bool al = ((uintptr_t)weight % 16) == 0 && ((uintptr_t)out % 16) == 0;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) return al && D % 4 == 0 ? em_fwd<float, 4>(p, st) : em_fwd<float, 1>(p, st);
  if (dtype == 1) return al && D % 8 == 0 ? em_fwd<_Float16, 8>(p, st) : em_fwd<_Float16, 1>(p, st);
  return al && D % 8 == 0 ? em_fwd<__bf16, 8>(p, st) : em_fwd<__bf16, 1>(p, st);
}

extern "C" size_t icg_embedding_bwd_workspace_bytes(int64_t n, int64_t V, int64_t D, int dtype) {
  if (!em_shape_ok(n, V, D, dtype) || n <= EMB_FEW) return 0;
  return em_align((size_t)n * 4) + em_align((size_t)(V + 1) * 4) + (size_t)icg_cdiv(n, EMB_CHUNK) * 2 * D * 4;
}

extern "C" int icg_embedding_bwd(const void* idx, const void* dout, void* dweight, int64_t n, int64_t V, int64_t D, float scale, int64_t pad, int idx64,
                                 int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  ICG_REQUIRE(idx && dout && dweight && em_shape_ok(n, V, D, dtype));
  EmbP p = {};
  p.idx = idx, p.dout = dout, p.dw = dweight, p.n = n, p.V = V, p.D = D, p.idx64 = idx64 != 0, p.scale = scale, p.pad = pad;
  if (n > EMB_FEW) {
    if (workspace_bytes < icg_embedding_bwd_workspace_bytes(n, V, D, dtype)) return ICG_ERR_WORKSPACE;
    ICG_REQUIRE(workspace && ((uintptr_t)workspace % 16) == 0);
    char* at = (char*)workspace;
    p.order = (int*)at, at += em_align((size_t)n * 4);
    p.start = (int*)at, at += em_align((size_t)(V + 1) * 4);
    p.part = (float*)at;
    // a workgroup for each compute unit, within the counts that fit (each reads the whole list: fewer read less)
    const int64_t run = icg_cdiv(V, 256);
    p.run = (int)(run < EMB_RUN ? run : EMB_RUN);
  }
  const bool al = ((uintptr_t)dweight % 16) == 0 && ((uintptr_t)dout % 16) == 0;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) return al && D % 4 == 0 ? em_bwd<float, 4>(p, st) : em_bwd<float, 1>(p, st);
  if (dtype == 1) return al && D % 8 == 0 ? em_bwd<_Float16, 8>(p, st) : em_bwd<_Float16, 1>(p, st);
  return al && D % 8 == 0 ? em_bwd<__bf16, 8>(p, st) : em_bwd<__bf16, 1>(p, st);
}
