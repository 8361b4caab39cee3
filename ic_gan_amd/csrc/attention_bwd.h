// Gradient kernels of csrc/attention.h (internal header, included once per element type).  The probabilities are computed again from the
// scores and the forward's l_i.  Two kernels, each owning what it sums -- keys (dk, dv) or queries (dq) -- so no atomics and the same bits on
// every run; the price is that scores and do . v are formed twice (7 products instead of 5).
#pragma once
#include "attention.h"

// Measured (kernel trace), 2 x 4096 causal, 16 heads of 128 over 4 key heads, bf16: row sums 23 us, dk and dv 375 us (733 TFLOP/s), their join
// 14 us, dq 272 us (758 TFLOP/s); 64 x 4096 queries, 1024 keys, 24 / 96 elements, fp32: 41, 1088 (118), -, 691 us (112 TFLOP/s); 6 x 777 queries, up to
// 1033 keys, 5 heads of 80, fp16: 10 (5 of them for the largest |v|), 50, -, 31 us.  Bound like the forward kernel: products and vector
// instructions of a SIMD add up to 0.93 of its cycles in fp32, 0.86 in the bf16 dq; dk and dv in bf16 have one wave a SIMD (0.73).

// D_i = do_i . o_i, |do_i| and the exponent's offset; o_i as it was before its rounding to 16 bits where the forward kept the rest (dp - D
// cancels: with the rounded o, a row of few keys had twice the error of its products' operands); `lanes` lanes (the power of two that covers a
// row's 16-byte chunks) to a row, rows in memory order.  SCALED: the workgroups from `row_blocks` on take 128 keys of a key head each and find their largest |v_j| (finite ones: a row
// that sees another has no finite gradient anyhow)
template <typename T>
__global__ __launch_bounds__(256) void icg_attention_rowstat_kernel(AttnP p, float* stat, int lanes, int64_t row_blocks) {
  constexpr int PER = 16 / (int)sizeof(T);
  const int64_t block = at_block(), rows = (int64_t)p.B * p.H * p.Lq, i = (block * 256 + threadIdx.x) / lanes;
  const int l = threadIdx.x & (lanes - 1);
  if constexpr (at_type<T>::SCALED) {
    if (block >= row_blocks) {
      __shared__ float red[4];
      const int64_t item = block - row_blocks, tiles = (p.Lk + 127) / 128, bh = item / tiles;
      const int Hk = p.H / p.G, b = (int)(bh / Hk), hk = (int)(bh - (int64_t)b * Hk), tile = (int)(item - bh * tiles), keys = b < p.B ? at_keys(p, b) : 0;
      if (b >= p.B) return;
      float most = 0.f;
      for (int j = 128 * tile + (int)threadIdx.x / lanes; j < min(keys, 128 * tile + 128); j += 256 / lanes) {
        float sq = 0.f;
        if (l * PER < p.dv) {
          const at_u4 a = *reinterpret_cast<const at_u4*>(reinterpret_cast<const T*>(p.v) + b * p.v_sb + j * p.v_sl + hk * p.v_sh + l * PER);
          T x[PER];
          __builtin_memcpy(x, &a, 16);
#pragma unroll
          for (int e = 0; e < PER; ++e) sq = __builtin_fmaf((float)x[e], (float)x[e], sq);
        }
        for (int s = lanes >> 1; s > 0; s >>= 1) sq += __shfl_xor(sq, s, 64);
        most = fmaxf(most, __builtin_isfinite(sq) ? sq : 0.f);
      }
      most = wave_max(most);
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
      __syncthreads();
      if (threadIdx.x == 0) stat[3 * rows + item] = sqrtf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
      return;
    }
  }
  if (i >= rows) return;
  const int64_t bq = i / p.H;
  const int hq = (int)(i - bq * p.H);
  const int64_t b = bq / p.Lq, qi = bq - b * p.Lq;
  float dot = 0.f, sq = 0.f;
  if (l * PER < p.dv) {
    const at_u4 a = *reinterpret_cast<const at_u4*>(reinterpret_cast<const T*>(p.o) + i * p.dv + l * PER);
    const at_u4 e = *reinterpret_cast<const at_u4*>(reinterpret_cast<const T*>(p.dout) + b * p.do_sb + qi * p.do_sl + hq * p.do_sh + l * PER);
    T x[PER], y[PER], z[PER] = {};
    if (p.o_low) {
      const at_u4 r = *reinterpret_cast<const at_u4*>(reinterpret_cast<const T*>(p.o_low) + i * p.dv + l * PER);
      __builtin_memcpy(z, &r, 16);
    }
    __builtin_memcpy(x, &a, 16);
    __builtin_memcpy(y, &e, 16);
#pragma unroll
    for (int j = 0; j < PER; ++j) dot = __builtin_fmaf((float)x[j] + (float)z[j], (float)y[j], dot), sq = __builtin_fmaf((float)y[j], (float)y[j], sq);
  }
  for (int s = lanes >> 1; s > 0; s >>= 1) dot += __shfl_xor(dot, s, 64), sq += __shfl_xor(sq, s, 64);
  if (l == 0) {
    const int64_t row = (b * p.H + hq) * p.Lq + qi;
    const float lse = p.lse[row];
    stat[row] = lse == -INFINITY ? INFINITY : __builtin_fmaf(lse, AT_LOG2E, -(float)at_type<T>::P_SHIFT);   // (a row that saw no key: p = exp2(s - inf) = 0)
    stat[rows + row] = dot;
    stat[2 * rows + row] = sqrtf(sq);
  }
}

// the power of two that brings a norm to [1, 2); 1 where there is none
__device__ __forceinline__ float at_to_one(float norm) {
  const unsigned e = (__float_as_uint(norm) >> 23) & 255u;
  return e == 0u || e >= 254u ? 1.f : __uint_as_float((254u - e) << 23);
}
// the power of two that ds of rows with |do| <= g is held by
__device__ __forceinline__ float at_ds_scale(float g, float vmax) { return 512.f * at_to_one(g * vmax); }
__device__ __forceinline__ float at_finite(float x) { return __builtin_isfinite(x) ? x : 0.f; }
// the largest of each thread's n, for all 256 threads (red: 4 floats of LDS, free again on return)
__device__ __forceinline__ float at_block_max(float n, float* red) {
  n = wave_max(n);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
  __syncthreads();
  n = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  return n;
}
// the largest |v_j| of a key head (SCALED)
__device__ __forceinline__ float at_vmax(const AttnP& p, int b, int hk, int64_t rows, float* red) {
  const int tiles = (p.Lk + 127) / 128;
  const float* of = p.stat + 3 * rows + ((int64_t)b * (p.H / p.G) + hk) * tiles;
  float n = 0.f;
  for (int i = threadIdx.x; i < tiles; i += 256) n = fmaxf(n, of[i]);
  return at_block_max(n, red);
}
__device__ __forceinline__ float at_ds(float pr, float dp, float s, float delta_s) { return pr * __builtin_fmaf(dp, s, -delta_s); }

// dq: a workgroup owns 128 queries of one head (a wave 32, as columns) and streams the keys, or its split of them
template <typename T, int DP, int DVP> constexpr int at_dq_waves() { return (DP + DVP) * (int)sizeof(T) / 8 + DP / 2 <= 144 ? 2 : 1; }
template <typename T, int DP, int DVP>
__global__ __launch_bounds__(256, (at_dq_waves<T, DP, DVP>())) void icg_attention_dq_kernel(AttnP p) {
  typedef at_type<T> X;
  typedef typename X::frag frag;
  constexpr int KT = sizeof(T) == 4 ? 32 : 64, KBYTES = KT * at_tile<T, DP>::STRIDE, SLOT = KBYTES + KT * at_tile<T, DVP>::STRIDE;
  __shared__ __attribute__((aligned(64))) char lds[2 * SLOT];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 31, h = lane >> 5;
  int64_t item = at_work_item(p.work);
  if (item < 0) return;
  const int split = (int)(item % p.nsplit);
  item /= p.nsplit;
  int tile = (int)(item % p.tiles);
  const int64_t bh = item / p.tiles;
  const int b = (int)(bh / p.H), hq = (int)(bh - (int64_t)b * p.H), hk = hq / p.G;
  if (p.causal) tile = p.tiles - 1 - tile;
  const int qi = 128 * tile + 32 * wv + m;
  const bool valid = qi < p.Lq;
  const int keys = at_keys(p, b), start = at_start(p, b);
  const int last = !valid ? -1 : (p.causal ? min(keys - 1, start + qi) : keys - 1);
  int kend = p.causal ? min(keys, start + min(p.Lq - 1, 128 * tile + 127) + 1) : keys;
  const int k0 = split * p.keys_per_split;
  if (p.nsplit > 1) kend = min(kend, k0 + p.keys_per_split);

  frag qf[DP / X::KSTEP], gf[DVP / X::KSTEP];
  at_own<T, DP>(qf, reinterpret_cast<const T*>(p.q) + b * p.q_sb + qi * p.q_sl + hq * p.q_sh, valid, p.d, h);
  at_own<T, DVP>(gf, reinterpret_cast<const T*>(p.dout) + b * p.do_sb + qi * p.do_sl + hq * p.do_sh, valid, p.dv, h);
  const int64_t rows = (int64_t)p.B * p.H * p.Lq, row = ((int64_t)b * p.H + hq) * p.Lq + qi;
  const float lse2 = valid ? p.stat[row] : INFINITY;
  float s1 = 1.f;
  if constexpr (X::SCALED) {
    const float vmax = at_vmax(p, b, hk, rows, reinterpret_cast<float*>(lds));
    s1 = valid ? at_ds_scale(p.stat[2 * rows + row], vmax) : 1.f;
  }
  const float delta = valid ? p.stat[rows + row] * s1 : 0.f;
  const at_rows kb(reinterpret_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh, p.k_sl, p.d, sizeof(T));
  const at_rows vb(reinterpret_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh, p.v_sl, p.dv, sizeof(T));
  const at_reader<T, DP> kr(lane);
  const at_reader<T, DVP> vr(lane);
  const float scl = p.scale * AT_LOG2E;

  at_f16v acc[DP / 32];
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[c][i] = 0.f;
  at_stage<T, DP, KT, 256> ks(kb, tid);
  at_stage<T, DVP, KT, 256> vs(vb, tid);
  auto fetch = [&](int j) {
    ks.fetch(kb, j, kend);
    vs.fetch(vb, j, kend);
  };
  auto put = [&](int cur) {
    ks.put(lds + cur * SLOT, tid);
    vs.put(lds + cur * SLOT + KBYTES, tid);
  };
  int cur = 0;
  if (k0 < kend) {
    fetch(k0);
    put(0);
    if (k0 + KT < kend) fetch(k0 + KT);
    __syncthreads();
  }
  for (int j0 = k0; j0 < kend; j0 += KT) {
    const char* kt = lds + cur * SLOT;
    const char* vt = kt + KBYTES;
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
      at_f16v s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f, dp[i] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / X::KSTEP; ++t)
        if (X::step(t, p.d)) s = X::mma(kr.row_frag(kt, 32 * u, t), qf[t], s);
#pragma unroll
      for (int t = 0; t < DVP / X::KSTEP; ++t) dp = X::mma(vr.row_frag(vt, 32 * u, t), gf[t], dp);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = at_ds(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scl, -lse2)), dp[i], s1, delta);
      if (__any(j0 + 32 * u + 31 > last)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = j0 + 32 * u + at_row_of(i, h) > last ? 0.f : s[i];
      }
      // ds is rounded to the inputs' type for the matrix product: half a step each, summed over the keys in 32 bits
#pragma unroll
      for (int q = 0; q < 32 / X::KSTEP; ++q) {
        const frag sf = X::pack(s, q);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) acc[c] = X::mma(kr.col_frag(kt, 32 * u, c, q), sf, acc[c]);
      }
    }
    if (j0 + KT < kend) {
      cur ^= 1;
      put(cur);
      if (j0 + 2 * KT < kend) fetch(j0 + 2 * KT);
      __syncthreads();
    }
  }
  if (!valid) return;
  const float f = p.scale * (1.f / (1 << X::P_SHIFT)) / s1;
  if (p.nsplit > 1) {
    float* out = p.part + (split * rows + row) * p.d;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        at_store4<float>(out, 32 * c + 8 * g + 4 * h, p.d, acc[c][4 * g] * f, acc[c][4 * g + 1] * f, acc[c][4 * g + 2] * f, acc[c][4 * g + 3] * f);
    return;
  }
  T* out = reinterpret_cast<T*>(p.dq) + (((int64_t)b * p.Lq + qi) * p.H + hq) * p.d;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      at_store4<T>(out, 32 * c + 8 * g + 4 * h, p.d, acc[c][4 * g] * f, acc[c][4 * g + 1] * f, acc[c][4 * g + 2] * f, acc[c][4 * g + 3] * f);
}

// dk, dv: a workgroup owns 128 keys of one key head (a wave 32, as columns) and streams the queries of every head of the group, so the
// gradient of a shared head is summed in registers
// Registers of a lane: own keys and values (DP + DVP) size / 8, sums (DP + DVP) / 2, about 100 beside them.  Two waves per SIMD (256) hold up
// to 144 of the first two.  A wave alone on its SIMD has nothing to run while a tile arrives: it streams 64 rows at a time (16-bit 128 + 128:
// 762 us with 32 rows, 581 with 64, at 2 x 4096 causal, 16 heads over 4).
template <typename T, int DP, int DVP>
struct at_dkv_shape {
  static constexpr int WAVES = (DP + DVP) * ((int)sizeof(T) + 4) / 8 <= 144 ? 2 : 1, QT = sizeof(T) == 2 && WAVES == 1 ? 64 : 32;
  static constexpr int QBYTES = QT * at_tile<T, DP>::STRIDE, GBYTES = QT * at_tile<T, DVP>::STRIDE, SLOT = QBYTES + GBYTES + 2 * QT * 4;
};
template <typename T, int DP, int DVP>
__global__ __launch_bounds__(256, (at_dkv_shape<T, DP, DVP>::WAVES)) void icg_attention_dkv_kernel(AttnP p) {
  typedef at_type<T> X;
  typedef typename X::frag frag;
  typedef at_dkv_shape<T, DP, DVP> S;
  constexpr int QT = S::QT, QBYTES = S::QBYTES, GBYTES = S::GBYTES, SLOT = S::SLOT;
  __shared__ __attribute__((aligned(64))) char lds[2 * SLOT];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 31, h = lane >> 5;
  int64_t item = at_work_item(p.work);
  if (item < 0) return;
  const int split = (int)(item % p.nsplit);
  item /= p.nsplit;
  const int tile = (int)(item % p.tiles);                // (the first keys, seen by the most queries of a causal triangle, first)
  const int64_t bh = item / p.tiles;
  const int Hk = p.H / p.G, b = (int)(bh / Hk), hk = (int)(bh - (int64_t)b * Hk);
  const int j = 128 * tile + 32 * wv + m;
  const int keys = at_keys(p, b), start = at_start(p, b);
  // a key that some query sees; the others are read as zeros (NaN or infinity there would meet the zero rows that fill the last query tile)
  const bool valid = j < keys && (!p.causal || j < start + p.Lq);
  const int64_t rows = (int64_t)p.B * p.H * p.Lq, row_b = ((int64_t)b * p.H + hk * p.G) * p.Lq;

  frag kf[DP / X::KSTEP], vf[DVP / X::KSTEP];
  at_own<T, DP>(kf, reinterpret_cast<const T*>(p.k) + b * p.k_sb + j * p.k_sl + hk * p.k_sh, valid, p.d, h);
  at_own<T, DVP>(vf, reinterpret_cast<const T*>(p.v) + b * p.v_sb + j * p.v_sl + hk * p.v_sh, valid, p.dv, h);
  const at_reader<T, DP> qr(lane);
  const at_reader<T, DVP> gr(lane);
  const float scl = p.scale * AT_LOG2E;

  float s1 = 1.f;
  if constexpr (X::SCALED) {                             // one scale for everything that is summed here
    float* red = reinterpret_cast<float*>(lds);
    float n = 0.f;
    for (int64_t i = tid; i < (int64_t)p.G * p.Lq; i += 256) n = fmaxf(n, at_finite(p.stat[2 * rows + row_b + i]));
    n = at_block_max(n, red);
    s1 = at_ds_scale(n, at_vmax(p, b, hk, rows, red));
  }

  at_f16v dk[DP / 32], dv[DVP / 32];
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[c][i] = 0.f;
#pragma unroll
  for (int c = 0; c < DVP / 32; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) dv[c][i] = 0.f;

  // query i sees key j from i = j - start on
  const int i0 = p.causal ? max(0, 128 * tile - start) / QT : 0;
  const int per = max(0, (p.Lq + QT - 1) / QT - i0), all = 128 * tile < keys ? p.G * per : 0;
  const int share = (all + p.nsplit - 1) / p.nsplit, n0 = min(split * share, all), n = min(share, all - n0);      // this split's tiles
  at_rows qb(reinterpret_cast<const T*>(p.q) + b * p.q_sb + (int64_t)hk * p.G * p.q_sh, p.q_sl, p.d, sizeof(T));
  at_rows gb(reinterpret_cast<const T*>(p.dout) + b * p.do_sb + (int64_t)hk * p.G * p.do_sh, p.do_sl, p.dv, sizeof(T));
  at_stage<T, DP, QT, 256> qs(qb, tid);
  at_stage<T, DVP, QT, 256> gs(gb, tid);
  float st = 0.f;                                        // threads 0 .. QT - 1: l_i, QT .. 2 QT - 1: D_i
  int fg = per > 0 ? n0 / per : 0, ft = n0 - fg * per;   // head and tile of the next fetch
  qb.base += (int64_t)fg * p.q_sh * (int64_t)sizeof(T), gb.base += (int64_t)fg * p.do_sh * (int64_t)sizeof(T);
  auto fetch = [&]() {
    const int r0 = (i0 + ft) * QT;
    qs.fetch(qb, r0, p.Lq);
    gs.fetch(gb, r0, p.Lq);
    if (tid < 2 * QT) {
      const int i = r0 + (tid & (QT - 1));
      const int64_t at = row_b + (int64_t)fg * p.Lq + i;
      st = tid < QT ? (i < p.Lq ? p.stat[at] : INFINITY) : (i < p.Lq ? p.stat[rows + at] * s1 : 0.f);
    }
    if (++ft == per) {
      ft = 0, ++fg;
      qb.base += p.q_sh * (int64_t)sizeof(T), gb.base += p.do_sh * (int64_t)sizeof(T);
    }
  };
  auto put = [&](int cur) {
    char* at = lds + cur * SLOT;
    qs.put(at, tid);
    gs.put(at + QBYTES, tid);
    if (tid < 2 * QT) reinterpret_cast<float*>(at + QBYTES + GBYTES)[tid] = st;
  };
  int cur = 0, t0 = ft;                                  // tile of the current one within its head
  if (n > 0) {
    fetch();
    put(0);
    if (n > 1) fetch();
    __syncthreads();
  }
  for (int it = 0; it < n; ++it) {
    const char* qt = lds + cur * SLOT;
    const char* gt = qt + QBYTES;
    const float* stat = reinterpret_cast<const float*>(gt + GBYTES);
#pragma unroll
    for (int u = 0; u < QT / 32; ++u) {
      at_f16v s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f, dp[i] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / X::KSTEP; ++t)
        if (X::step(t, p.d)) s = X::mma(qr.row_frag(qt, 32 * u, t), kf[t], s);
#pragma unroll
      for (int t = 0; t < DVP / X::KSTEP; ++t) dp = X::mma(gr.row_frag(gt, 32 * u, t), vf[t], dp);
      const int first = valid ? (p.causal ? j - start : -(1 << 30)) : 0x7fffffff;       // the first query that sees this lane's key
      const int r0 = (i0 + t0) * QT + 32 * u;
      const bool edge = __any(r0 < first);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const at_f4 l4 = *reinterpret_cast<const at_f4*>(stat + 32 * u + 8 * g + 4 * h), d4 = *reinterpret_cast<const at_f4*>(stat + QT + 32 * u + 8 * g + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * g + e;
          s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scl, -l4[e]));
          dp[i] = at_ds(s[i], dp[i], s1, d4[e]);
        }
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool off = r0 + at_row_of(i, h) < first;
          s[i] = off ? 0.f : s[i];
          dp[i] = off ? 0.f : dp[i];
        }
      }
      // p and ds are rounded to the inputs' type for the matrix products: half a step each, summed over the queries in 32 bits
#pragma unroll
      for (int q = 0; q < 32 / X::KSTEP; ++q) {
        const frag pf = X::pack(s, q), sf = X::pack(dp, q);
#pragma unroll
        for (int c = 0; c < DVP / 32; ++c) dv[c] = X::mma(gr.col_frag(gt, 32 * u, c, q), pf, dv[c]);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) dk[c] = X::mma(qr.col_frag(qt, 32 * u, c, q), sf, dk[c]);
      }
    }
    if (++t0 == per) t0 = 0;
    if (it + 1 < n) {
      cur ^= 1;
      put(cur);
      if (it + 2 < n) fetch();
      __syncthreads();
    }
  }
  if (j >= p.Lk) return;                                 // (keys from k_lens on have no gradient: their sums are zero)
  const float fv = 1.f / (1 << X::P_SHIFT), fk = p.scale * fv / s1;
  if (p.nsplit > 1) {
    float* out = p.part + ((((int64_t)split * p.B + b) * p.Lk + j) * Hk + hk) * (p.d + p.dv);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        at_store4<float>(out, 32 * c + 8 * g + 4 * h, p.d, dk[c][4 * g] * fk, dk[c][4 * g + 1] * fk, dk[c][4 * g + 2] * fk, dk[c][4 * g + 3] * fk);
#pragma unroll
    for (int c = 0; c < DVP / 32; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        at_store4<float>(out + p.d, 32 * c + 8 * g + 4 * h, p.dv, dv[c][4 * g] * fv, dv[c][4 * g + 1] * fv, dv[c][4 * g + 2] * fv, dv[c][4 * g + 3] * fv);
    return;
  }
  T* dk_out = reinterpret_cast<T*>(p.dk) + (((int64_t)b * p.Lk + j) * Hk + hk) * p.d;
  T* dv_out = reinterpret_cast<T*>(p.dv_out) + (((int64_t)b * p.Lk + j) * Hk + hk) * p.dv;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      at_store4<T>(dk_out, 32 * c + 8 * g + 4 * h, p.d, dk[c][4 * g] * fk, dk[c][4 * g + 1] * fk, dk[c][4 * g + 2] * fk, dk[c][4 * g + 3] * fk);
#pragma unroll
  for (int c = 0; c < DVP / 32; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      at_store4<T>(dv_out, 32 * c + 8 * g + 4 * h, p.dv, dv[c][4 * g] * fv, dv[c][4 * g + 1] * fv, dv[c][4 * g + 2] * fv, dv[c][4 * g + 3] * fv);
}

// sums the splits of dq in order: a thread takes 4 elements of a row
template <typename T>
__global__ __launch_bounds__(256) void icg_attention_join_dq_kernel(AttnP p) {
  const int64_t rows = (int64_t)p.B * p.H * p.Lq;
  const int quads = p.d / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / quads;
  if (row >= rows) return;
  const int c = (int)(i - row * quads) * 4;
  at_f4 x = *reinterpret_cast<const at_f4*>(p.part + row * p.d + c);
  for (int s = 1; s < p.nsplit; ++s) x += *reinterpret_cast<const at_f4*>(p.part + (s * rows + row) * p.d + c);
  const int64_t bh = row / p.Lq, qi = row - bh * p.Lq, b = bh / p.H, hq = bh - b * p.H;
  at_store4<T>(reinterpret_cast<T*>(p.dq) + ((b * p.Lq + qi) * p.H + hq) * p.d, c, p.d, x[0], x[1], x[2], x[3]);
}

// sums the splits of dk and dv in order: a thread takes 4 elements of a key's row [d + dv]
template <typename T>
__global__ __launch_bounds__(256) void icg_attention_join_dkv_kernel(AttnP p) {
  const int64_t rows = (int64_t)p.B * p.Lk * (p.H / p.G);
  const int w = p.d + p.dv, quads = w / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / quads;
  if (row >= rows) return;
  const int c = (int)(i - row * quads) * 4;
  at_f4 x = *reinterpret_cast<const at_f4*>(p.part + row * w + c);
  for (int s = 1; s < p.nsplit; ++s) x += *reinterpret_cast<const at_f4*>(p.part + (s * rows + row) * w + c);
  if (c < p.d) at_store4<T>(reinterpret_cast<T*>(p.dk) + row * p.d, c, p.d, x[0], x[1], x[2], x[3]);
  else at_store4<T>(reinterpret_cast<T*>(p.dv_out) + row * p.dv, c - p.d, p.dv, x[0], x[1], x[2], x[3]);
}

// p: planned for dq, pk: for dk and dv; the two take turns with the room for partial sums
template <typename T>
int at_bwd(AttnP p, AttnP pk, float* stat, hipStream_t st) {
  p.stat = pk.stat = stat;
  int lanes = 1;
  while (lanes * 16 < p.dv * (int)sizeof(T)) lanes <<= 1;        // (at most 64: rows of up to 256 fp32)
  const int64_t row_blocks = icg_cdiv((int64_t)p.B * p.H * p.Lq * lanes, 256);
  const int64_t key_blocks = at_type<T>::SCALED ? (int64_t)p.B * (p.H / p.G) * icg_cdiv(p.Lk, 128) : 0;
  hipLaunchKernelGGL((icg_attention_rowstat_kernel<T>), at_grid(row_blocks + key_blocks), dim3(256), 0, st, p, stat, lanes, row_blocks);
  if (const int e = icg_check_launch()) return e;
#define AT_RUN(DP, DVP)                                                                                                  \
  do {                                                                                                                   \
    hipLaunchKernelGGL((icg_attention_dkv_kernel<T, DP, DVP>), at_grid(pk.work), dim3(256), 0, st, pk);           \
    if (const int e = icg_check_launch()) return e;                                                                      \
    if (pk.nsplit > 1) {                                                                                                 \
      const int64_t quads = (int64_t)p.B * p.Lk * (p.H / p.G) * ((p.d + p.dv) / 4);                                      \
      hipLaunchKernelGGL((icg_attention_join_dkv_kernel<T>), dim3((unsigned)icg_cdiv(quads, 256)), dim3(256), 0, st, pk); \
      if (const int e = icg_check_launch()) return e;                                                                    \
    }                                                                                                                    \
    hipLaunchKernelGGL((icg_attention_dq_kernel<T, DP, DVP>), at_grid(p.work), dim3(256), 0, st, p);              \
    if (p.nsplit > 1) {                                                                                                  \
      if (const int e = icg_check_launch()) return e;                                                                    \
      const int64_t quads = (int64_t)p.B * p.H * p.Lq * (p.d / 4);                                                       \
      hipLaunchKernelGGL((icg_attention_join_dq_kernel<T>), dim3((unsigned)icg_cdiv(quads, 256)), dim3(256), 0, st, p);  \
    }                                                                                                                    \
  } while (0)
  AT_FOR_HEAD(p.d, p.dv, AT_RUN)
#undef AT_RUN
  return icg_check_launch();
}
