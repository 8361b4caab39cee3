// Forward kernels of csrc/attention.h: one pass over the keys with the running maximum and sum of the softmax (internal header, included
// once per element type).
#pragma once
#include "attention.h"

template <typename T, bool TOKENS>
struct at_fwd_shape {
  // ROWS: 4 waves, 32 queries of one head each, all of them against every streamed tile of KT keys.
  // TOKENS (few queries): ONE tile of 32 rows, the (query, head) pairs that share a key head; each wave takes 32 of the KT keys, so a
  // tile is read once for the whole group and the waves' results are joined at the end.
  static constexpr int WAVES = TOKENS && sizeof(T) == 4 ? 2 : 4;
  static constexpr int THREADS = 64 * WAVES;
  static constexpr int KT = TOKENS ? 32 * WAVES : (sizeof(T) == 4 ? 32 : 64);
  static constexpr int SUB = TOKENS ? 1 : KT / 32;      // 32-key tiles of one wave
  static constexpr int BUFFERS = TOKENS ? 1 : 2;
  // two waves per SIMD (256 registers) where own operands and sums leave room: one wave's exponentials run under the other's products
  template <int DP, int DVP> static constexpr int waves() { return DP * (int)sizeof(T) / 8 + DVP / 2 <= (TOKENS ? 96 : 128) ? 2 : 1; }
};

// Bound and measured.  A SIMD's matrix and vector instructions do not seem to overlap, not even those of its two waves: cycles of the products plus 4
// for each vector instruction (16 for an exponential) are 0.92 - 1.02 of a SIMD's busy cycles (counters: fp32, and bf16 at 2 x 8192; 0.88 at
// 2 x 4096, where the last workgroups leave SIMDs half empty), and reading operands further ahead, a third wave, or forming the next tile's
// scores beside the exponentials gained nothing (558 us -> 609 us).  So a lane does per score one fma, one exponential, one add, half a
// conversion and half a maximum, and nothing else.
//   2 x 8192 causal, 16 heads of 128 over 4 key heads, bf16:      575 us =  956 TFLOP/s (the library's 8192^3 product: 1234)
//   64 x 4096 queries, 1024 keys, 48 / 192 elements, fp32:        996 us =  129 TFLOP/s (154)
//   one token for 32 sequences of 2048 .. 8192 keys, 32 / 8 heads: 153 us = 4.4 TB/s   (a copy: 4.78; two workgroups a unit keep 128 KB in flight)
// One form spills (82 registers, compiled scratch): fp32, few queries, heads of 64 / 256.
template <typename T, int DP, int DVP, bool TOKENS>
__global__ __launch_bounds__((at_fwd_shape<T, TOKENS>::THREADS), (at_fwd_shape<T, TOKENS>::template waves<DP, DVP>())) void icg_attention_fwd_kernel(AttnP p) {
  typedef at_fwd_shape<T, TOKENS> S;
  typedef at_type<T> X;
  typedef typename X::frag frag;
  typedef at_tile<T, DP> KTile;
  typedef at_tile<T, DVP> VTile;
  constexpr int KBYTES = S::KT * KTile::STRIDE, VBYTES = S::KT * VTile::STRIDE, SLOT = KBYTES + VBYTES;
  constexpr int JOIN = TOKENS ? 32 * DVP * 4 + 2 * S::WAVES * 32 * 4 : 0;
  constexpr int LDS = S::BUFFERS * SLOT > JOIN ? S::BUFFERS * SLOT : JOIN;
  constexpr int NV = DVP / 32;
  __shared__ __attribute__((aligned(64))) char lds[LDS];

  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 31, h = lane >> 5;
  int64_t item = at_work_item(p.work);
  if (item < 0) return;
  const int split = (int)(item % p.nsplit);
  item /= p.nsplit;
  int tile = (int)(item % p.tiles);
  const int64_t bh = item / p.tiles;                     // (batch, query head), or (batch, key head) for TOKENS
  const int heads = TOKENS ? p.H / p.G : p.H;
  const int b = (int)(bh / heads), head = (int)(bh - (int64_t)b * heads);
  if (!TOKENS && p.causal) tile = p.tiles - 1 - tile;    // the long rows of a causal triangle first

  int qi, hq, qi_last;
  bool valid;
  if constexpr (TOKENS) {
    const int r = 32 * tile + m;
    valid = r < p.Lq * p.G;
    qi = r / p.G;
    hq = head * p.G + (r - qi * p.G);
    qi_last = min(p.Lq - 1, (32 * tile + 31) / p.G);
  } else {
    qi = 128 * tile + 32 * wv + m;
    valid = qi < p.Lq;
    hq = head;
    qi_last = min(p.Lq - 1, 128 * tile + 127);
  }
  const int hk = TOKENS ? head : head / p.G;
  const int keys = at_keys(p, b), start = at_start(p, b);
  const int last = !valid ? -1 : (p.causal ? min(keys - 1, start + qi) : keys - 1);      // the last key that this lane's query sees
  int kend = p.causal ? min(keys, start + qi_last + 1) : keys;
  int k0 = 0;
  if (p.nsplit > 1) {
    k0 = split * p.keys_per_split;
    kend = min(kend, k0 + p.keys_per_split);
  }

  frag qf[DP / X::KSTEP];
  at_own<T, DP>(qf, reinterpret_cast<const T*>(p.q) + b * p.q_sb + qi * p.q_sl + hq * p.q_sh, valid, p.d, h);
  const at_rows kb(reinterpret_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh, p.k_sl, p.d, sizeof(T));
  const at_rows vb(reinterpret_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh, p.v_sl, p.dv, sizeof(T));
  const at_reader<T, DP> kr(lane);
  const at_reader<T, DVP> vr(lane);

  at_f16v o[NV];
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = 0.f;
  float mx = AT_LOWEST, sum = 0.f;                       // running maximum (of s log2 e) and this half's part of the sum
  const float scl = p.scale * AT_LOG2E;

  at_stage<T, DP, S::KT, S::THREADS> ks(kb, tid);
  at_stage<T, DVP, S::KT, S::THREADS> vs(vb, tid);
  if (k0 < kend) {
    ks.fetch(kb, k0, kend);
    vs.fetch(vb, k0, kend);
  }
  int cur = 0;
  if (S::BUFFERS == 2 && k0 < kend) {
    ks.put(lds, tid);
    vs.put(lds + KBYTES, tid);
    if (k0 + S::KT < kend) {
      ks.fetch(kb, k0 + S::KT, kend);
      vs.fetch(vb, k0 + S::KT, kend);
    }
    __syncthreads();
  }
  for (int j0 = k0; j0 < kend; j0 += S::KT) {
    if constexpr (S::BUFFERS == 1) {
      __syncthreads();                                   // every wave has read the tile before
      ks.put(lds, tid);
      vs.put(lds + KBYTES, tid);
      if (j0 + S::KT < kend) {
        ks.fetch(kb, j0 + S::KT, kend);
        vs.fetch(vb, j0 + S::KT, kend);
      }
      __syncthreads();
    }
    const char* kt = lds + cur * SLOT;
    const char* vt = kt + KBYTES;
    const int sub0 = TOKENS ? 32 * wv : 0;
    at_f16v s[S::SUB];
#pragma unroll
    for (int u = 0; u < S::SUB; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / X::KSTEP; ++t)
        if (X::step(t, p.d)) s[u] = X::mma(kr.row_frag(kt, sub0 + 32 * u, t), qf[t], s[u]);
    }
    const int jw = j0 + sub0;
    if (__any(jw + 32 * S::SUB - 1 > last)) {
#pragma unroll
      for (int u = 0; u < S::SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = jw + 32 * u + at_row_of(i, h) > last ? -INFINITY : s[u][i];
    }
    float t = s[0][0];
#pragma unroll
    for (int u = 0; u < S::SUB; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) t = fmaxf(t, s[u][i]);
    t = at_other_half_max(t) * scl;
    // the sums are brought to a new maximum only when it grew by more than 2^8: p stays below 256, exact in the products' types
    if (__any(t > mx + 8.f)) {
      const float next = fmaxf(mx, t), a = __builtin_amdgcn_exp2f(mx - next);
      mx = next;
      sum *= a;
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i] *= a;
    }
#pragma unroll
    for (int u = 0; u < S::SUB; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], scl, -mx));
      float a = 0.f, c = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i += 2) a += s[u][i], c += s[u][i + 1];
      sum += a + c;
      // p is rounded to the inputs' type for the matrix product (half a step of values whose errors average out over the keys); its sum is not
#pragma unroll
      for (int q = 0; q < 32 / X::KSTEP; ++q) {
        const frag pf = X::pack(s[u], q);
#pragma unroll
        for (int cc = 0; cc < NV; ++cc) o[cc] = X::mma(vr.col_frag(vt, sub0 + 32 * u, cc, q), pf, o[cc]);
      }
    }
    if constexpr (S::BUFFERS == 2) {
      if (j0 + S::KT < kend) {
        cur ^= 1;
        ks.put(lds + cur * SLOT, tid);
        vs.put(lds + cur * SLOT + KBYTES, tid);
        if (j0 + 2 * S::KT < kend) {
          ks.fetch(kb, j0 + 2 * S::KT, kend);
          vs.fetch(vb, j0 + 2 * S::KT, kend);
        }
        __syncthreads();
      }
    }
  }
  sum = at_both_halves_sum(sum);

  if constexpr (TOKENS) {                                // join the waves in a fixed order
    float* joined = reinterpret_cast<float*>(lds);       // [32 rows][DVP], then the waves' maxima and sums
    float* stat = joined + 32 * DVP;
    __syncthreads();
    if (h == 0) {
      stat[(2 * wv) * 32 + m] = mx;
      stat[(2 * wv + 1) * 32 + m] = sum;
    }
    __syncthreads();
    float all = stat[m];
#pragma unroll
    for (int w = 1; w < S::WAVES; ++w) all = fmaxf(all, stat[2 * w * 32 + m]);
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < S::WAVES; ++w) sum += stat[(2 * w + 1) * 32 + m] * __builtin_amdgcn_exp2f(stat[2 * w * 32 + m] - all);
    const float a = __builtin_amdgcn_exp2f(mx - all);
    mx = all;
#pragma unroll
    for (int w = 0; w < S::WAVES; ++w) {
      if (wv == w) {
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float* at = joined + (32 * c + at_row_of(i, h)) * 32 + m;      // (column-major: the lanes of a half on different banks)
            *at = w == 0 ? o[c][i] * a : *at + o[c][i] * a;
          }
      }
      __syncthreads();
    }
    // wave w takes the columns of tiles c = w, w + WAVES, ...
#pragma unroll
    for (int c = 0; c < NV; ++c)
      if (c % S::WAVES == wv)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i] = joined[(32 * c + at_row_of(i, h)) * 32 + m];
  }
  if (!valid) return;
  const int64_t row = ((int64_t)b * p.H + hq) * p.Lq + qi;
  const bool writes_stat = h == 0 && (!TOKENS || wv == 0);
  if (p.nsplit > 1) {
    const int64_t rows = (int64_t)p.B * p.H * p.Lq;
    if (writes_stat) reinterpret_cast<at_f2*>(p.part + p.nsplit * rows * p.dv)[split * rows + row] = at_f2{mx, sum};
    if (sum == 0.f) return;                              // (the join does not read the sums of a split that saw no key)
    float* out = p.part + (split * rows + row) * p.dv;
#pragma unroll
    for (int c = 0; c < NV; ++c)
      if (!TOKENS || c % S::WAVES == wv)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          at_store4<float>(out, 32 * c + 8 * g + 4 * h, p.dv, o[c][4 * g], o[c][4 * g + 1], o[c][4 * g + 2], o[c][4 * g + 3]);
    return;
  }
  if (writes_stat) p.lse[row] = sum == 0.f ? -INFINITY : mx * AT_LN2 + __logf(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;        // a row that sees no key is zero
  const int64_t out = ((int64_t)b * p.Lq + qi) * p.H + hq;
#pragma unroll
  for (int c = 0; c < NV; ++c)
    if (!TOKENS || c % S::WAVES == wv)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        at_store_out<T>(p, out, 32 * c + 8 * g + 4 * h, o[c][4 * g] * inv, o[c][4 * g + 1] * inv, o[c][4 * g + 2] * inv, o[c][4 * g + 3] * inv);
}

// joins the splits of a row: a wave per row, 4 columns a lane, splits in order (one pass over the partial sums)
template <typename T>
__global__ __launch_bounds__(256) void icg_attention_join_kernel(AttnP p) {
  const int64_t rows = (int64_t)p.B * p.H * p.Lq, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & 63, c = 4 * lane;
  const at_f2* stat = reinterpret_cast<const at_f2*>(p.part + p.nsplit * rows * p.dv) + row;
  float mx = AT_LOWEST;
  for (int s = 0; s < p.nsplit; ++s) mx = fmaxf(mx, stat[s * rows][0]);
  float sum = 0.f;
  at_f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < p.nsplit; ++s) {
    const at_f2 ms = stat[s * rows];
    if (ms[1] == 0.f) continue;                          // (a split that saw no key wrote no sums)
    const float a = __builtin_amdgcn_exp2f(ms[0] - mx);
    sum += ms[1] * a;
    if (c < p.dv) o += *reinterpret_cast<const at_f4*>(p.part + (s * rows + row) * p.dv + c) * a;
  }
  if (lane == 0) p.lse[row] = sum == 0.f ? -INFINITY : mx * AT_LN2 + __logf(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t bh = row / p.Lq, qi = row - bh * p.Lq, b = bh / p.H, hq = bh - b * p.H;
  at_store_out<T>(p, (b * p.Lq + qi) * p.H + hq, c, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
}

template <typename T>
int at_fwd(const AttnP& p, bool tokens, hipStream_t st) {
#define AT_RUN(DP, DVP)                                                                                                                    \
  do {                                                                                                                                     \
    if (tokens) hipLaunchKernelGGL((icg_attention_fwd_kernel<T, DP, DVP, true>), at_grid(p.work), dim3(at_fwd_shape<T, true>::THREADS), 0, st, p); \
    else hipLaunchKernelGGL((icg_attention_fwd_kernel<T, DP, DVP, false>), at_grid(p.work), dim3(at_fwd_shape<T, false>::THREADS), 0, st, p);      \
  } while (0)
  AT_FOR_HEAD(p.d, p.dv, AT_RUN)
#undef AT_RUN
  if (const int e = icg_check_launch()) return e;
  if (p.nsplit > 1) {
    hipLaunchKernelGGL((icg_attention_join_kernel<T>), dim3((unsigned)icg_cdiv((int64_t)p.B * p.H * p.Lq, 4)), dim3(256), 0, st, p);
    return icg_check_launch();
  }
  return ICG_OK;
}
