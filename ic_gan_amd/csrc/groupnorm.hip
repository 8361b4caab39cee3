// Group norm with an activation on channels-last activations x[b][p][c] (p = 0 .. HW - 1), gain and bias per channel or per sample and channel:
//
//   m, v over a group's Cg channels and all p;   xh = (x - m) / sqrt(v + eps);   z = xh (g0 + gain) + bias;   y = act(z)
//   dz = dy act'(z);  dbias = sum_p dz;  dgain = sum_p dz xh;  dn = dz (g0 + gain);  dx = (dn - mean(dn) - xh mean(dn xh)) / sqrt(v + eps)
//
// Bound by memory: what counts is how often x (and dy) are read.  A thread owns one 16-byte column of channels and walks rows, so that its
// per-channel coefficients stay in registers and every row access is whole 16-byte pieces.
//   one pass     a group's slab [HW][Cg] fits one workgroup's registers (8 rows a thread): read once, normalised from registers
//   three passes (larger slabs) partial sums of row chunks -> one workgroup per group joins them -> apply; x is read twice
// Measured (kernel trace), 64 x 256 x 256 x 96 fp32 with ReLU (1.6 GB): first pass 327 us (4.9 TB/s), last 565 us (5.7 TB/s); 32 x 64 x 64 x 384
// bf16 with SiLU (100 MB): 28 and 43 us, its gradient 57 and 66 us (3.6 and 4.5 TB/s); 64 x 4 x 4 x 1536 fp32 in one pass: 10 and 11 us.
// Means and squared deviations are joined pairwise from sums about each part's own mean (no difference of large squares); across chunks in
// 64 bits.  All sums in 32 bits or more, in a fixed order, no atomics.
#include "icg_common.h"

typedef unsigned gn_u4 __attribute__((ext_vector_type(4)));

struct GnP {
  const void *x, *dy;
  const float *gain, *bias;
  void *y, *dx;
  float *mean, *rstd;                 // [B][G]
  float *dgain, *dbias;               // [B][C] per sample, else the per-sample sums of a shared gain (workspace)
  float* part;                        // three passes: [B][chunks][2][C], then [B][G][2]
  int64_t HW;
  int B, C, G, Cg, per_sample, act;
  float g0, eps;
  int cc, ncol, ny;                   // 16-byte columns per workgroup, column blocks, rows at a time
  int nchunks;
  int64_t rows;                       // rows per chunk
};

constexpr int GN_R = 8;               // rows a thread holds in registers (one pass)
constexpr int GN_P = 4;               // rows whose moments a thread forms at a time (three passes)

template <typename T, int VEC> struct gn_vec { T e[VEC]; };
template <typename T, int VEC>
__device__ __forceinline__ gn_vec<T, VEC> gn_load(const T* p) {
  gn_vec<T, VEC> r;
  if constexpr (VEC == 1) r.e[0] = *p;
  else { const gn_u4 w = *reinterpret_cast<const gn_u4*>(p); __builtin_memcpy(&r, &w, 16); }
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void gn_store(T* p, const gn_vec<T, VEC>& r) {
  if constexpr (VEC == 1) *p = r.e[0];
  else { gn_u4 w; __builtin_memcpy(&w, &r, 16); *reinterpret_cast<gn_u4*>(p) = w; }
}

__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504088896340736f)); }
// (a comparison and not a maximum, which would turn NaN into 0: a group with a value that is not finite shows it after a ReLU too)
__device__ __forceinline__ float gn_act(float z, int act) { return act == 0 ? z : act == 1 ? (z < 0.f ? 0.f : z) : z * gn_sigmoid(z); }
__device__ __forceinline__ float gn_dact(float z, int act) {
  if (act == 0) return 1.f;
  if (act == 1) return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;      // (NaN stays)
  const float s = gn_sigmoid(z);
  return s * (1.f + z * (1.f - s));
}

// a part's (sum, squared deviations from its own mean) joined with another's: what depends on the counts alone, then a channel
struct gn_joint {
  float ia, ib, f;
  __device__ __forceinline__ gn_joint(float na, float nb) : ia(na > 0.f ? 1.f / na : 0.f), ib(nb > 0.f ? 1.f / nb : 0.f), f(na > 0.f && nb > 0.f ? na * nb / (na + nb) : 0.f) {}
  __device__ __forceinline__ void operator()(float& sa, float& qa, float sb, float qb) const {
    const float d = sb * ib - sa * ia;
    qa += __builtin_fmaf(d * d, f, qb);
    sa += sb;
  }
};

// rows k = ty, ty + ny, .. of `n` rows, at most GN_R of them
__device__ __forceinline__ int gn_mine(int64_t n, int ty, int ny, int most = GN_R) { return n > ty ? (int)min((n - ty + ny - 1) / ny, (int64_t)most) : 0; }

// sum and squared deviations of a thread's `mine` rows, per channel
template <typename T, int VEC, int R>
__device__ __forceinline__ void gn_moments(const gn_vec<T, VEC> (&v)[R], int mine, float (&s)[VEC], float (&q)[VEC]) {
  const float inv = mine > 0 ? 1.f / (float)mine : 0.f;
#pragma unroll
  for (int c = 0; c < VEC; ++c) {
    s[c] = 0.f, q[c] = 0.f;
#pragma unroll
    for (int k = 0; k < R; ++k) s[c] += k < mine ? (float)v[k].e[c] : 0.f;
    const float mu = s[c] * inv;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const float d = (float)v[k].e[c] - mu;
      q[c] += k < mine ? d * d : 0.f;
    }
  }
}

// Two quantities per (row lane, channel) summed over the row lanes; the totals are left at row lane 0.
// MOMENTS: the pair is (sum, squared deviations) of n[row lane] values, else two plain sums.
template <int VEC, bool MOMENTS>
__device__ __forceinline__ void gn_reduce_rows(float* s1, float* s2, float* n, float (&a)[VEC], float (&b)[VEC], float count, int tx, int ty, int cc,
                                               int ny, bool active) {
  const int at = (ty * cc + tx) * VEC;
  if (active) {
#pragma unroll
    for (int c = 0; c < VEC; ++c) s1[at + c] = a[c], s2[at + c] = b[c];
    if (MOMENTS && tx == 0) n[ty] = count;
  }
  int half = 1;
  while (half < ny) half <<= 1;
  for (half >>= 1; half > 0; half >>= 1) {
    __syncthreads();
    const bool join = active && ty < half && ty + half < ny;
    float na = 0.f, nb = 0.f;
    if (join) {
      const int from = at + half * cc * VEC;
      if constexpr (MOMENTS) na = n[ty], nb = n[ty + half];
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        if constexpr (MOMENTS) gn_joint(na, nb)(s1[at + c], s2[at + c], s1[from + c], s2[from + c]);
        else s1[at + c] += s1[from + c], s2[at + c] += s2[from + c];
      }
    }
    if constexpr (MOMENTS) {
      __syncthreads();                                     // every column has read n[ty] before it grows
      if (join && tx == 0) n[ty] = na + nb;
    }
  }
  __syncthreads();
}

// Rows of a thread in the last pass.  A 4-byte type streams best in short workgroups (64 x 256 x 256 x 96: 561 us with 4 rows, 593 with 16); a
// 2-byte type has twice the channels' coefficients to fetch first (32 x 64 x 64 x 384: 68 us with 4 rows, 45 with 16; its gradient 84 and
// 73 with 4 and 8).
constexpr int gn_apply_rows(int vec, bool bwd) { return vec == 8 ? (bwd ? 8 : 16) : 4; }

template <int VEC>
struct gn_coef {
  float mean[VEC], rstd[VEC], gain[VEC], bias[VEC];
  __device__ __forceinline__ void affine(const GnP& p, int b, int c0) {
    const int64_t at = p.per_sample ? (int64_t)b * p.C + c0 : c0;
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      gain[c] = p.gain ? p.g0 + p.gain[at + c] : 1.f;
      bias[c] = p.bias ? p.bias[at + c] : 0.f;
    }
  }
  __device__ __forceinline__ void stat(const GnP& p, int b, int c0) {
    int64_t g = (int64_t)b * p.G + c0 / p.Cg;
    int in = c0 % p.Cg;
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      mean[c] = p.mean[g], rstd[c] = p.rstd[g];
      if (++in == p.Cg) in = 0, ++g;
    }
  }
  __device__ __forceinline__ float z(float x, int c, float& xh) const {
    xh = (x - mean[c]) * rstd[c];
    return __builtin_fmaf(xh, gain[c], bias[c]);
  }
};

// ---- one pass: a workgroup owns cc 16-byte columns (whole groups) of one sample and all its rows
template <typename T, int VEC, int THREADS, bool BWD>
__global__ __launch_bounds__(THREADS) void icg_groupnorm_slab_kernel(GnP p) {
  __shared__ float s1[THREADS * VEC], s2[THREADS * VEC], n[THREADS], gm[THREADS * VEC], gr[THREADS * VEC];
  const int tid = threadIdx.x, tx = tid % p.cc, ty = tid / p.cc;
  const bool active = ty < p.ny;
  const int b = blockIdx.x / p.ncol, col0 = (blockIdx.x - b * p.ncol) * p.cc * VEC, c0 = col0 + tx * VEC;
  const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)b * p.HW * p.C + c0;
  const int mine = active ? gn_mine(p.HW, ty, p.ny) : 0;
  gn_vec<T, VEC> v[GN_R], dv[BWD ? GN_R : 1];
#pragma unroll
  for (int k = 0; k < GN_R; ++k) {
    const int64_t r = ty + (int64_t)k * p.ny;
    if (k < mine) {
      v[k] = gn_load<T, VEC>(x + r * p.C);
      if constexpr (BWD) dv[k] = gn_load<T, VEC>(reinterpret_cast<const T*>(p.dy) + ((int64_t)b * p.HW + r) * p.C + c0);
    }
  }
  const int groups = p.cc * VEC / p.Cg, lane = tid & 63, wv = tid >> 6;
  gn_coef<VEC> k_;
  if (active) k_.affine(p, b, c0);
  float a[VEC], q[VEC];
  if constexpr (!BWD) {
    gn_moments<T, VEC, GN_R>(v, mine, a, q);
    gn_reduce_rows<VEC, true>(s1, s2, n, a, q, (float)mine, tx, ty, p.cc, p.ny, active);
    const float rows = (float)p.HW, all = rows * (float)p.Cg;
    for (int g = wv; g < groups; g += THREADS / 64) {
      float s = 0.f;
      for (int c = lane; c < p.Cg; c += 64) s += s1[g * p.Cg + c];
      const float mu = wave_sum(s) / all;
      float m2 = 0.f;
      for (int c = lane; c < p.Cg; c += 64) {
        const float d = s1[g * p.Cg + c] / rows - mu;
        m2 += s2[g * p.Cg + c] + rows * d * d;
      }
      m2 = wave_sum(m2);
      const float r = 1.f / sqrtf(m2 / all + p.eps);
      if (lane == 0) {
        gm[g] = mu, gr[g] = r;
        const int64_t at = (int64_t)b * p.G + col0 / p.Cg + g;
        p.mean[at] = mu, p.rstd[at] = r;
      }
    }
    __syncthreads();
    if (!active) return;
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      const int g = (tx * VEC + c) / p.Cg;
      k_.mean[c] = gm[g], k_.rstd[c] = gr[g];
    }
    T* y = reinterpret_cast<T*>(p.y) + (int64_t)b * p.HW * p.C + c0;
#pragma unroll
    for (int k = 0; k < GN_R; ++k)
      if (k < mine) {
        gn_vec<T, VEC> o;
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          float xh;
          o.e[c] = (T)gn_act(k_.z((float)v[k].e[c], c, xh), p.act);
        }
        gn_store<T, VEC>(y + (ty + (int64_t)k * p.ny) * p.C, o);
      }
  } else {
    if (active) k_.stat(p, b, c0);
#pragma unroll
    for (int c = 0; c < VEC; ++c) a[c] = 0.f, q[c] = 0.f;
#pragma unroll
    for (int k = 0; k < GN_R; ++k)
      if (k < mine)
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          float xh;
          const float z = k_.z((float)v[k].e[c], c, xh), dz = (float)dv[k].e[c] * gn_dact(z, p.act);
          a[c] += dz;
          q[c] = __builtin_fmaf(dz, xh, q[c]);
        }
    gn_reduce_rows<VEC, false>(s1, s2, n, a, q, 0.f, tx, ty, p.cc, p.ny, active);
    const float all = (float)p.HW * (float)p.Cg;
    for (int g = wv; g < groups; g += THREADS / 64) {
      float u = 0.f, w = 0.f;
      for (int c = lane; c < p.Cg; c += 64) {
        const int ch = col0 + g * p.Cg + c;
        const float gain = p.gain ? p.g0 + p.gain[p.per_sample ? (int64_t)b * p.C + ch : ch] : 1.f;
        u += s1[g * p.Cg + c] * gain, w += s2[g * p.Cg + c] * gain;
      }
      u = wave_sum(u), w = wave_sum(w);
      if (lane == 0) gm[g] = u / all, gr[g] = w / all;
    }
    if (p.dgain)
      for (int c = tid; c < p.cc * VEC; c += THREADS) {
        p.dbias[(int64_t)b * p.C + col0 + c] = s1[c];
        p.dgain[(int64_t)b * p.C + col0 + c] = s2[c];
      }
    __syncthreads();
    if (!active) return;
    T* dx = reinterpret_cast<T*>(p.dx) + (int64_t)b * p.HW * p.C + c0;
#pragma unroll
    for (int k = 0; k < GN_R; ++k)
      if (k < mine) {
        gn_vec<T, VEC> o;
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          const int g = (tx * VEC + c) / p.Cg;
          float xh;
          const float z = k_.z((float)v[k].e[c], c, xh), dz = (float)dv[k].e[c] * gn_dact(z, p.act);
          o.e[c] = (T)((dz * k_.gain[c] - gm[g] - xh * gr[g]) * k_.rstd[c]);
        }
        gn_store<T, VEC>(dx + (ty + (int64_t)k * p.ny) * p.C, o);
      }
  }
}

// ---- three passes, first: per-channel moments (forward) or sums of dz and dz xh (gradient) of a chunk of rows
template <typename T, int VEC, bool BWD>
__global__ __launch_bounds__(256) void icg_groupnorm_part_kernel(GnP p) {
  __shared__ float s1[256 * VEC], s2[256 * VEC], n[256];
  const int tid = threadIdx.x, tx = tid % p.cc, ty = tid / p.cc;
  const int c0 = (blockIdx.y * p.cc + tx) * VEC, b = blockIdx.z;
  const bool active = ty < p.ny && c0 < p.C;
  const int64_t r0 = (int64_t)blockIdx.x * p.rows, rows = min(p.rows, p.HW - r0);
  const T* x = reinterpret_cast<const T*>(p.x) + ((int64_t)b * p.HW + r0) * p.C + c0;
  float a[VEC], q[VEC], count = 0.f;
#pragma unroll
  for (int c = 0; c < VEC; ++c) a[c] = 0.f, q[c] = 0.f;
  gn_coef<VEC> k_;
  if constexpr (BWD) {
    if (active) k_.affine(p, b, c0), k_.stat(p, b, c0);
  }
  if (active) {
    if constexpr (BWD) {
      const T* dy = reinterpret_cast<const T*>(p.dy) + ((int64_t)b * p.HW + r0) * p.C + c0;
      for (int64_t r = ty; r < rows; r += p.ny) {
        const gn_vec<T, VEC> v = gn_load<T, VEC>(x + r * p.C), dv = gn_load<T, VEC>(dy + r * p.C);
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          float xh;
          const float z = k_.z((float)v.e[c], c, xh), dz = (float)dv.e[c] * gn_dact(z, p.act);
          a[c] += dz;
          q[c] = __builtin_fmaf(dz, xh, q[c]);
        }
      }
    } else {
      for (int64_t s = 0; s < rows; s += (int64_t)GN_P * p.ny) {
        const int mine = gn_mine(rows - s, ty, p.ny, GN_P);
        gn_vec<T, VEC> v[GN_P];
#pragma unroll
        for (int k = 0; k < GN_P; ++k)
          if (k < mine) v[k] = gn_load<T, VEC>(x + (s + ty + (int64_t)k * p.ny) * p.C);
        if (mine == 0) continue;
        float sa[VEC], qa[VEC];
        gn_moments<T, VEC, GN_P>(v, mine, sa, qa);
        const gn_joint join(count, (float)mine);
#pragma unroll
        for (int c = 0; c < VEC; ++c) join(a[c], q[c], sa[c], qa[c]);
        count += (float)mine;
      }
    }
  }
  gn_reduce_rows<VEC, !BWD>(s1, s2, n, a, q, count, tx, ty, p.cc, p.ny, active);
  float* out = p.part + ((int64_t)b * p.nchunks + blockIdx.x) * 2 * p.C;
  for (int c = tid; c < p.cc * VEC; c += 256) {
    const int ch = blockIdx.y * p.cc * VEC + c;
    if (ch < p.C) out[ch] = s1[c], out[p.C + ch] = s2[c];
  }
}

// ---- second: a workgroup joins the chunks of one (sample, group), in 64 bits
__device__ __forceinline__ double gn_block_sum(double v, double* red) {
  v = wave_sum_d(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(256) void icg_groupnorm_join_kernel(GnP p) {
  __shared__ double red[4];
  const int b = blockIdx.x / p.G, g = blockIdx.x - b * p.G;
  const float* part = p.part + (int64_t)b * p.nchunks * 2 * p.C + g * p.Cg;
  const int64_t n = (int64_t)p.nchunks * p.Cg;
  const double all = (double)p.HW * p.Cg;
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 256) s += part[i / p.Cg * 2 * p.C + i % p.Cg];
  const double mu = gn_block_sum(s, red) / all;
  double q = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 256) {
    const int64_t k = i / p.Cg;
    const double rows = (double)min(p.rows, p.HW - k * p.rows), d = part[k * 2 * p.C + i % p.Cg] / rows - mu;
    q += part[k * 2 * p.C + p.C + i % p.Cg] + rows * d * d;
  }
  q = gn_block_sum(q, red);
  if (threadIdx.x == 0) p.mean[blockIdx.x] = (float)mu, p.rstd[blockIdx.x] = (float)(1.0 / sqrt(q / all + (double)p.eps));
}

// gradient: per-channel sums over the chunks -> dbias, dgain of the sample; per group mean(dn), mean(dn xh)
__global__ __launch_bounds__(256) void icg_groupnorm_join_bwd_kernel(GnP p, float* coef) {
  __shared__ double red[4];
  const int b = blockIdx.x / p.G, g = blockIdx.x - b * p.G, wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const float* part = p.part + (int64_t)b * p.nchunks * 2 * p.C + g * p.Cg;
  double u = 0.0, w = 0.0;
  for (int c = wv; c < p.Cg; c += 4) {                     // a wave per channel
    double s = 0.0, q = 0.0;
    for (int k = lane; k < p.nchunks; k += 64) s += part[(int64_t)k * 2 * p.C + c], q += part[(int64_t)k * 2 * p.C + p.C + c];
    s = wave_sum_d(s), q = wave_sum_d(q);
    if (lane == 0) {
      const int ch = g * p.Cg + c;
      const double gain = p.gain ? (double)(p.g0 + p.gain[p.per_sample ? (int64_t)b * p.C + ch : ch]) : 1.0;
      u += s * gain, w += q * gain;
      if (p.dgain) p.dbias[(int64_t)b * p.C + ch] = (float)s, p.dgain[(int64_t)b * p.C + ch] = (float)q;
    }
  }
  u = gn_block_sum(u, red);
  w = gn_block_sum(w, red);
  const double all = (double)p.HW * p.Cg;
  if (threadIdx.x == 0) coef[2 * blockIdx.x] = (float)(u / all), coef[2 * blockIdx.x + 1] = (float)(w / all);
}

// ---- third: y, or dx.  Blocks run from the end of the tensor: what the first pass read last may still be in the caches.
template <typename T, int VEC, bool BWD>
__global__ __launch_bounds__(256) void icg_groupnorm_apply_kernel(GnP p, const float* coef, int per_block) {
  const int tid = threadIdx.x, tx = tid % p.cc, ty = tid / p.cc;
  const int c0 = (blockIdx.y * p.cc + tx) * VEC, b = p.B - 1 - blockIdx.z;
  if (ty >= p.ny || c0 >= p.C) return;
  const int64_t r0 = (int64_t)(gridDim.x - 1 - blockIdx.x) * per_block, rows = min((int64_t)per_block, p.HW - r0), base = ((int64_t)b * p.HW + r0) * p.C + c0;
  const T* x = reinterpret_cast<const T*>(p.x) + base;
  const T* dy = reinterpret_cast<const T*>(p.dy) + (BWD ? base : 0);
  T* out = reinterpret_cast<T*>(BWD ? p.dx : p.y) + base;
  gn_coef<VEC> k_;
  k_.affine(p, b, c0);
  k_.stat(p, b, c0);
  float m1[VEC], m2[VEC];
  if constexpr (BWD) {
    int64_t g = (int64_t)b * p.G + c0 / p.Cg;
    int in = c0 % p.Cg;
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      m1[c] = coef[2 * g], m2[c] = coef[2 * g + 1];
      if (++in == p.Cg) in = 0, ++g;
    }
  }
  for (int64_t r = ty; r < rows; r += p.ny) {
    const gn_vec<T, VEC> v = gn_load<T, VEC>(x + r * p.C);
    gn_vec<T, VEC> dv, o;
    if constexpr (BWD) dv = gn_load<T, VEC>(dy + r * p.C);
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      float xh;
      const float z = k_.z((float)v.e[c], c, xh);
      if constexpr (BWD) {
        const float dz = (float)dv.e[c] * gn_dact(z, p.act);
        o.e[c] = (T)((dz * k_.gain[c] - m1[c] - xh * m2[c]) * k_.rstd[c]);
      } else {
        o.e[c] = (T)gn_act(z, p.act);
      }
    }
    gn_store<T, VEC>(out + r * p.C, o);
  }
}

// a gain that all samples share: its gradient is the sum over the samples, in order
__global__ __launch_bounds__(256) void icg_groupnorm_batch_sum_kernel(const float* dgain_b, const float* dbias_b, float* dgain, float* dbias, int B, int C) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  double g = 0.0, s = 0.0;
#pragma unroll 8
  for (int b = 0; b < B; ++b) g += dgain_b[(int64_t)b * C + c], s += dbias_b[(int64_t)b * C + c];
  dgain[c] = (float)g, dbias[c] = (float)s;
}

namespace {

struct GnPlan {
  bool vec, slab;
  int threads, cc, ncol, ny, nchunks;
  int64_t rows;
};

bool gn_shape_ok(int B, int64_t HW, int C, int G, int dtype) {
  return B > 0 && B < 65536 && HW > 0 && HW < (1LL << 30) && C > 0 && C < (1 << 20) && G > 0 && C % G == 0 && dtype >= 0 && dtype <= 2 && (int64_t)B * G < 0x7fffffffL;
}

// whether the one-pass kernel has a form of 1024 threads (128 registers each: too few for 8 rows of x and dy in 16 bits)
constexpr bool gn_wide(int vec, bool bwd) { return !(bwd && vec == 8); }

GnPlan gn_plan(int B, int64_t HW, int C, int G, int dtype, bool vec, bool bwd) {
  GnPlan pl = {};
  const int per = dtype == 0 ? 4 : 8, v = vec && C % per == 0 ? per : 1, Cg = C / G;
  pl.vec = v > 1;
  // whole groups in whole 16-byte columns, as many as fit the registers of a workgroup while there are workgroups enough (512: two for each
  // compute unit): neighbouring groups share cache lines
  int gs = 1;
  while (gs <= G && (G % gs != 0 || (gs * Cg) % v != 0)) ++gs;
  auto fits = [&](int set, int threads) { const int cc = set * Cg / v; return cc <= threads && HW <= (int64_t)(threads / cc) * GN_R; };
  if (gs <= G && (fits(gs, 256) || (gn_wide(v, bwd) && fits(gs, 1024)))) {
    pl.slab = true;
    while (G % (2 * gs) == 0 && fits(2 * gs, 256) && (int64_t)B * (G / (2 * gs)) >= 512) gs *= 2;
    pl.threads = fits(gs, 256) ? 256 : 1024;
    pl.cc = gs * Cg / v, pl.ncol = G / gs, pl.ny = pl.threads / pl.cc;
    if (pl.ny > HW) pl.ny = (int)HW;
    return pl;
  }
  // column blocks that leave the fewest of the 256 threads idle
  const int cv = C / v;
  double best = -1.0;
  const int least = (int)icg_cdiv(cv, 256);
  for (int n = least; n < least + 4 && n <= cv; ++n) {
    const int cc = (int)icg_cdiv(cv, n), ny = 256 / cc;
    const double used = (double)cv / ((double)n * cc) * ny * cc / 256.0;
    if (used > best + 1e-9) best = used, pl.cc = cc, pl.ncol = (int)icg_cdiv(cv, cc), pl.ny = ny;
  }
  // chunks of whole batches; 4 workgroups for each compute unit, 8 in the gradient (64 x 256 x 256 x 96 fp32: 314 us with 4, 360 with 8, 333 with
  // 16; the gradient of 32 x 64 x 64 x 384 bf16: 54, 47, 57)
  const int64_t batch = (int64_t)pl.ny * GN_P;
  int64_t chunks = icg_cdiv(HW, batch);
  const int64_t most = icg_cdiv((bwd ? 8 : 4) * 256, (int64_t)B * pl.ncol);
  if (chunks > most) chunks = most;
  pl.rows = icg_cdiv(icg_cdiv(HW, chunks), batch) * batch;
  pl.nchunks = (int)icg_cdiv(HW, pl.rows);
  return pl;
}

// (the plan with 16-byte columns and the one without differ in their chunks: room for either)
size_t gn_part_bytes(int B, int64_t HW, int C, int G, int dtype, bool bwd) {
  size_t most = 0;
  for (int vec = 0; vec < 2; ++vec) {
    const GnPlan pl = gn_plan(B, HW, C, G, dtype, vec != 0, bwd);
    const size_t n = pl.slab ? 0 : (size_t)B * pl.nchunks * 2 * C * 4 + (size_t)B * G * 2 * 4;
    if (n > most) most = n;
  }
  return (most + 15) / 16 * 16;
}

GnP gn_params(const GnPlan& pl, int B, int64_t HW, int C, int G, int per_sample, float g0, float eps, int act) {
  GnP p = {};
  p.B = B, p.HW = HW, p.C = C, p.G = G, p.Cg = C / G, p.per_sample = per_sample != 0, p.g0 = g0, p.eps = eps, p.act = act;
  p.cc = pl.cc, p.ncol = pl.ncol, p.ny = pl.ny, p.nchunks = pl.nchunks, p.rows = pl.rows;
  return p;
}

int gn_width(const GnPlan& pl, int dtype) { return !pl.vec ? 1 : dtype == 0 ? 4 : 8; }
// A dimension of a grid holds fewer than 2^32 threads (the runtime does not refuse more, it leaves some out)
bool gn_grids_ok(const GnPlan& pl, int B, int64_t HW, int G, bool bwd, int vec) {
  const int64_t most = 1LL << 32;
  if (pl.slab) return (int64_t)B * pl.ncol * pl.threads < most;
  return pl.ncol < 65536 && (int64_t)B * G * 256 < most && (int64_t)pl.nchunks * 256 < most &&
         icg_cdiv(HW, pl.ny * gn_apply_rows(vec, bwd)) * 256 < most;
}
// both directions, with 16-byte columns and without
bool gn_applies(int B, int64_t HW, int C, int G, int dtype) {
  if (!gn_shape_ok(B, HW, C, G, dtype)) return false;
  for (int i = 0; i < 4; ++i) {
    const GnPlan pl = gn_plan(B, HW, C, G, dtype, i & 1, i >> 1);
    if (!gn_grids_ok(pl, B, HW, G, i >> 1, gn_width(pl, dtype))) return false;
  }
  return true;
}

template <typename T, int VEC, bool BWD>
int gn_run(const GnPlan& pl, const GnP& p, hipStream_t st) {
  if (pl.slab) {
    const dim3 grid((unsigned)((int64_t)p.B * p.ncol));
    if constexpr (gn_wide(VEC, BWD)) {
      if (pl.threads == 1024) {
        hipLaunchKernelGGL((icg_groupnorm_slab_kernel<T, VEC, 1024, BWD>), grid, dim3(1024), 0, st, p);
        return icg_check_launch();
      }
    }
    hipLaunchKernelGGL((icg_groupnorm_slab_kernel<T, VEC, 256, BWD>), grid, dim3(256), 0, st, p);
    return icg_check_launch();
  }
  const dim3 grid((unsigned)pl.nchunks, (unsigned)pl.ncol, (unsigned)p.B);
  float* coef = p.part + (int64_t)p.B * p.nchunks * 2 * p.C;
  hipLaunchKernelGGL((icg_groupnorm_part_kernel<T, VEC, BWD>), grid, dim3(256), 0, st, p);
  if (const int e = icg_check_launch()) return e;
  if (BWD) hipLaunchKernelGGL(icg_groupnorm_join_bwd_kernel, dim3((unsigned)(p.B * p.G)), dim3(256), 0, st, p, coef);
  else hipLaunchKernelGGL(icg_groupnorm_join_kernel, dim3((unsigned)(p.B * p.G)), dim3(256), 0, st, p);
  if (const int e = icg_check_launch()) return e;
  const int per_block = p.ny * gn_apply_rows(VEC, BWD);
  const dim3 apply((unsigned)icg_cdiv(p.HW, per_block), (unsigned)pl.ncol, (unsigned)p.B);
  hipLaunchKernelGGL((icg_groupnorm_apply_kernel<T, VEC, BWD>), apply, dim3(256), 0, st, p, (const float*)coef, per_block);
  return icg_check_launch();
}

template <bool BWD>
int gn_dispatch(const GnPlan& pl, const GnP& p, int dtype, hipStream_t st) {
  if (dtype == 0) return pl.vec ? gn_run<float, 4, BWD>(pl, p, st) : gn_run<float, 1, BWD>(pl, p, st);
  if (dtype == 1) return pl.vec ? gn_run<_Float16, 8, BWD>(pl, p, st) : gn_run<_Float16, 1, BWD>(pl, p, st);
  return pl.vec ? gn_run<__bf16, 8, BWD>(pl, p, st) : gn_run<__bf16, 1, BWD>(pl, p, st);
}

}  // namespace

extern "C" int icg_groupnorm_applies(int B, int64_t HW, int C, int G, int dtype) { return gn_applies(B, HW, C, G, dtype) ? 1 : 0; }

extern "C" size_t icg_groupnorm_fwd_workspace_bytes(int B, int64_t HW, int C, int G, int dtype) {
  return gn_shape_ok(B, HW, C, G, dtype) ? gn_part_bytes(B, HW, C, G, dtype, false) : 0;
}

extern "C" int icg_groupnorm_act_fwd(const void* x, const float* gain, const float* bias, void* y, float* mean, float* rstd, int B, int64_t HW, int C,
                                     int G, int per_sample, float gain_offset, float eps, int act, int dtype, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  ICG_REQUIRE(x && y && mean && rstd && gn_shape_ok(B, HW, C, G, dtype) && act >= 0 && act <= 2 && eps >= 0.f && eps < INFINITY);
  const bool vec = ((uintptr_t)x % 16) == 0 && ((uintptr_t)y % 16) == 0;
  const GnPlan pl = gn_plan(B, HW, C, G, dtype, vec, false);
  ICG_REQUIRE(gn_grids_ok(pl, B, HW, G, false, gn_width(pl, dtype)));
  GnP p = gn_params(pl, B, HW, C, G, per_sample, gain_offset, eps, act);
  p.x = x, p.gain = gain, p.bias = bias, p.y = y, p.mean = mean, p.rstd = rstd;
  if (!pl.slab) {
    if (workspace_bytes < gn_part_bytes(B, HW, C, G, dtype, false)) return ICG_ERR_WORKSPACE;
    ICG_REQUIRE(workspace && ((uintptr_t)workspace % 16) == 0);
    p.part = (float*)workspace;
  }
  return gn_dispatch<false>(pl, p, dtype, (hipStream_t)stream);
}

extern "C" size_t icg_groupnorm_bwd_workspace_bytes(int B, int64_t HW, int C, int G, int dtype) {
  return gn_shape_ok(B, HW, C, G, dtype) ? gn_part_bytes(B, HW, C, G, dtype, true) + (size_t)B * C * 2 * 4 : 0;
}

extern "C" int icg_groupnorm_act_bwd(const void* x, const void* dy, const float* gain, const float* bias, const float* mean, const float* rstd, void* dx,
                                     float* dgain, float* dbias, int B, int64_t HW, int C, int G, int per_sample, float gain_offset, float eps, int act,
                                     int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  ICG_REQUIRE(x && dy && dx && mean && rstd && gn_shape_ok(B, HW, C, G, dtype) && act >= 0 && act <= 2 && !dgain == !dbias);
  if (workspace_bytes < icg_groupnorm_bwd_workspace_bytes(B, HW, C, G, dtype)) return ICG_ERR_WORKSPACE;
  ICG_REQUIRE(workspace && ((uintptr_t)workspace % 16) == 0);
  const bool vec = ((uintptr_t)x % 16) == 0 && ((uintptr_t)dy % 16) == 0 && ((uintptr_t)dx % 16) == 0;
  const GnPlan pl = gn_plan(B, HW, C, G, dtype, vec, true);
  ICG_REQUIRE(gn_grids_ok(pl, B, HW, G, true, gn_width(pl, dtype)));
  GnP p = gn_params(pl, B, HW, C, G, per_sample, gain_offset, eps, act);
  p.x = x, p.dy = dy, p.gain = gain, p.bias = bias, p.dx = dx, p.mean = const_cast<float*>(mean), p.rstd = const_cast<float*>(rstd);
  p.part = (float*)workspace;
  float* sums = (float*)((char*)workspace + gn_part_bytes(B, HW, C, G, dtype, true));
  const bool shared = dgain && !per_sample;
  p.dgain = shared ? sums : dgain, p.dbias = shared ? sums + (size_t)B * C : dbias;
  if (const int e = gn_dispatch<true>(pl, p, dtype, (hipStream_t)stream)) return e;
  if (shared) {
    hipLaunchKernelGGL(icg_groupnorm_batch_sum_kernel, dim3((unsigned)icg_cdiv(C, 256)), dim3(256), 0, (hipStream_t)stream, p.dgain, p.dbias, dgain, dbias, B, C);
    return icg_check_launch();
  }
  return ICG_OK;
}
