// C entry points of the attention without a stored probability matrix (kernels: csrc/attention.h, attention_fwd.h, attention_bwd.h).
#include "attention.h"

namespace {

constexpr int kTokenRows = 32;     // rows of the kernel for few queries

// Few queries: a 128-row tile would be mostly padding, and the heads that share a key head would each read it again.
bool at_tokens(int Lq, int G) { return Lq <= 16 || (int64_t)Lq * G <= kTokenRows; }

// The keys in splits for `want` workgroups, no split shorter than 256 keys (below that the join costs more than it saves); 3/4 of the wanted
// number is enough
void at_split_keys(AttnP& p, int64_t items, int64_t want) {
  const int64_t unit = 256, most = icg_cdiv(p.Lk, unit);
  int64_t n = 4 * items >= 3 * want ? 1 : icg_cdiv(want, items);
  n = n < most ? n : most;
  n = n > 1 ? n : 1;
  p.keys_per_split = (int)(icg_cdiv(icg_cdiv(p.Lk, n), unit) * unit);
  p.nsplit = (int)icg_cdiv(p.Lk, p.keys_per_split);
  p.work = items * p.nsplit;
}

// Forward: with few queries two workgroups for each of the 256 compute units (what is read is all that counts, and it takes two to keep the
// memory busy), with many one for each.
void at_plan(AttnP& p) {
  const bool tok = at_tokens(p.Lq, p.G);
  p.tiles = (int)(tok ? icg_cdiv((int64_t)p.Lq * p.G, kTokenRows) : icg_cdiv(p.Lq, 128));
  at_split_keys(p, (int64_t)p.B * (tok ? p.H / p.G : p.H) * p.tiles, tok ? 512 : 256);
}

// dq
void at_plan_dq(AttnP& p) {
  p.tiles = (int)icg_cdiv(p.Lq, 128);
  at_split_keys(p, (int64_t)p.B * p.H * p.tiles, 256);
}

// How the queries of a key tile are split in the key gradient: a workgroup for each compute unit, twice as many where a causal triangle makes
// them uneven (the long ones start first and the short ones fill up behind them); at least 4 query tiles each
void at_plan_dkv(AttnP& p) {
  p.tiles = (int)icg_cdiv(p.Lk, 128);
  const int64_t items = (int64_t)p.B * (p.H / p.G) * p.tiles, steps = (int64_t)p.G * icg_cdiv(p.Lq, 64), want = p.causal ? 512 : 256;
  int64_t n = 4 * items >= 3 * want ? 1 : icg_cdiv(want, items);
  n = n < steps / 4 ? n : steps / 4;
  n = n < 16 ? n : 16;
  p.nsplit = (int)(n > 1 ? n : 1);
  p.work = items * p.nsplit;
}
// three numbers a query, and for fp16 one for every 128 keys
size_t at_stat_bytes(const AttnP& p, int dtype) {
  const size_t keys = dtype == 1 ? (size_t)p.B * (p.H / p.G) * icg_cdiv(p.Lk, 128) : 0;
  return (((size_t)3 * p.B * p.H * p.Lq + keys) * 4 + 15) / 16 * 16;
}
size_t at_bwd_bytes(const AttnP& dq, const AttnP& dkv, int dtype) {
  const size_t a = dq.nsplit > 1 ? (size_t)dq.nsplit * dq.B * dq.H * dq.Lq * dq.d * 4 : 0;
  const size_t b = dkv.nsplit > 1 ? (size_t)dkv.nsplit * dkv.B * dkv.Lk * (dkv.H / dkv.G) * (dkv.d + dkv.dv) * 4 : 0;
  return at_stat_bytes(dq, dtype) + (a > b ? a : b);
}

size_t at_part_bytes(const AttnP& p) {
  return p.nsplit > 1 ? (size_t)p.nsplit * p.B * p.H * p.Lq * ((size_t)p.dv + 2) * 4 : 0;
}

bool at_shape_ok(int B, int Lq, int Lk, int H, int Hk, int d, int dv, int dtype) {
  if (B <= 0 || Lq <= 0 || Lk <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0) return false;
  if (dtype < 0 || dtype > 2) return false;
  if (Lq > (1 << 24) || Lk > (1 << 24) || H > (1 << 16) || (int64_t)B * H * Lq >= 0x7fffffffL || (int64_t)B * Hk * icg_cdiv(Lk, 128) >= 0x7fffffffL) return false;
  const int per = dtype == 0 ? 4 : 8;
  return d > 0 && dv > 0 && d % per == 0 && dv % per == 0 && ((d <= 128 && dv <= 128) || (d <= 64 && dv <= 256));
}

// whole 16-byte chunks at multiples of 16 bytes; positions at least a row apart, and 128 of them within the reach of a descriptor
bool at_row_ok(const void* x, int64_t sb, int64_t sl, int64_t sh, int len, int size) {
  const int per = 16 / size;
  return ((uintptr_t)x % 16) == 0 && sb % per == 0 && sl % per == 0 && sh % per == 0 && sl >= len && sl * size < (1 << 24);
}

}  // namespace

extern "C" int icg_attention_applies(int B, int Lq, int Lk, int H, int Hk, int d, int dv, int dtype) {
  return at_shape_ok(B, Lq, Lk, H, Hk, d, dv, dtype) ? 1 : 0;
}

extern "C" size_t icg_attention_fwd_workspace_bytes(int B, int Lq, int Lk, int H, int Hk, int d, int dv, int dtype) {
  if (!at_shape_ok(B, Lq, Lk, H, Hk, d, dv, dtype)) return 0;
  AttnP p = {};
  p.B = B, p.Lq = Lq, p.Lk = Lk, p.H = H, p.G = H / Hk, p.d = d, p.dv = dv;
  at_plan(p);
  return at_part_bytes(p);
}

extern "C" size_t icg_attention_bwd_workspace_bytes(int B, int Lq, int Lk, int H, int Hk, int d, int dv, int causal, int dtype) {
  if (!at_shape_ok(B, Lq, Lk, H, Hk, d, dv, dtype)) return 0;
  AttnP p = {};
  p.B = B, p.Lq = Lq, p.Lk = Lk, p.H = H, p.G = H / Hk, p.d = d, p.dv = dv, p.causal = causal != 0;
  AttnP pk = p;
  at_plan_dq(p);
  at_plan_dkv(pk);
  return at_bwd_bytes(p, pk, dtype);
}

extern "C" int icg_attention_fwd(const void* q, const void* k, const void* v, const int* k_lens, const int* q_start, void* o, void* o_low,
                                 float* lse, int B, int Lq, int Lk, int H, int Hk, int d, int dv, int64_t q_sb, int64_t q_sl, int64_t q_sh,
                                 int64_t k_sb, int64_t k_sl, int64_t k_sh, int64_t v_sb, int64_t v_sl, int64_t v_sh, float scale, int causal, int dtype,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  ICG_REQUIRE(q && k && v && o && lse && at_shape_ok(B, Lq, Lk, H, Hk, d, dv, dtype));
  ICG_REQUIRE(scale > 0.f && scale < INFINITY && ((uintptr_t)o % 16) == 0 && ((uintptr_t)o_low % 16) == 0);
  const int size = dtype == 0 ? 4 : 2;
  AttnP p = {};
  p.q = q, p.k = k, p.v = v, p.k_lens = k_lens, p.q_start = q_start, p.o = o, p.o_low = o_low, p.lse = lse;
  p.B = B, p.Lq = Lq, p.Lk = Lk, p.H = H, p.G = H / Hk, p.d = d, p.dv = dv;
  p.q_sb = q_sb, p.q_sl = q_sl, p.q_sh = q_sh, p.k_sb = k_sb, p.k_sl = k_sl, p.k_sh = k_sh, p.v_sb = v_sb, p.v_sl = v_sl, p.v_sh = v_sh;
  p.scale = scale, p.causal = causal != 0;
  ICG_REQUIRE(at_row_ok(q, q_sb, q_sl, q_sh, d, size) && at_row_ok(k, k_sb, k_sl, k_sh, d, size) && at_row_ok(v, v_sb, v_sl, v_sh, dv, size));
  at_plan(p);
  ICG_REQUIRE(p.work < 0x7fffffffL);
  if (p.nsplit > 1) {
    if (workspace_bytes < at_part_bytes(p)) return ICG_ERR_WORKSPACE;
    ICG_REQUIRE(workspace && ((uintptr_t)workspace % 16) == 0);
    p.part = (float*)workspace;
  }
  const bool tok = at_tokens(Lq, p.G);
  hipStream_t st = (hipStream_t)stream;
  return dtype == 0 ? at_fwd_f32(p, tok, st) : dtype == 1 ? at_fwd_f16(p, tok, st) : at_fwd_bf16(p, tok, st);
}

extern "C" int icg_attention_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_low, const void* dout,
                                 const float* lse, const int* k_lens,
                                 const int* q_start, void* dq, void* dk, void* dv_out, int B, int Lq, int Lk, int H, int Hk, int d, int dv,
                                 int64_t q_sb, int64_t q_sl, int64_t q_sh, int64_t k_sb, int64_t k_sl, int64_t k_sh, int64_t v_sb, int64_t v_sl,
                                 int64_t v_sh, int64_t do_sb, int64_t do_sl, int64_t do_sh, float scale, int causal, int dtype, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  ICG_REQUIRE(q && k && v && o && dout && lse && dq && dk && dv_out && at_shape_ok(B, Lq, Lk, H, Hk, d, dv, dtype));
  ICG_REQUIRE(scale > 0.f && scale < INFINITY);
  ICG_REQUIRE(((uintptr_t)o % 16) == 0 && ((uintptr_t)dq % 16) == 0 && ((uintptr_t)dk % 16) == 0 && ((uintptr_t)dv_out % 16) == 0 &&
              ((uintptr_t)o_low % 16) == 0);
  if (workspace_bytes < icg_attention_bwd_workspace_bytes(B, Lq, Lk, H, Hk, d, dv, causal, dtype)) return ICG_ERR_WORKSPACE;
  ICG_REQUIRE(workspace && ((uintptr_t)workspace % 16) == 0);
  const int size = dtype == 0 ? 4 : 2;
  AttnP p = {};
  p.q = q, p.k = k, p.v = v, p.k_lens = k_lens, p.q_start = q_start, p.o = const_cast<void*>(o), p.o_low = const_cast<void*>(o_low), p.lse = const_cast<float*>(lse), p.dout = dout;
  p.dq = dq, p.dk = dk, p.dv_out = dv_out;
  p.B = B, p.Lq = Lq, p.Lk = Lk, p.H = H, p.G = H / Hk, p.d = d, p.dv = dv;
  p.q_sb = q_sb, p.q_sl = q_sl, p.q_sh = q_sh, p.k_sb = k_sb, p.k_sl = k_sl, p.k_sh = k_sh, p.v_sb = v_sb, p.v_sl = v_sl, p.v_sh = v_sh;
  p.do_sb = do_sb, p.do_sl = do_sl, p.do_sh = do_sh;
  p.scale = scale, p.causal = causal != 0;
  ICG_REQUIRE(at_row_ok(q, q_sb, q_sl, q_sh, d, size) && at_row_ok(k, k_sb, k_sl, k_sh, d, size) && at_row_ok(v, v_sb, v_sl, v_sh, dv, size));
  ICG_REQUIRE(at_row_ok(dout, do_sb, do_sl, do_sh, dv, size));
  float* stat = (float*)workspace;
  p.part = (float*)((char*)workspace + at_stat_bytes(p, dtype));
  AttnP pk = p;
  at_plan_dq(p);
  at_plan_dkv(pk);
  ICG_REQUIRE(p.work < 0x7fffffffL && pk.work < 0x7fffffffL);
  hipStream_t st = (hipStream_t)stream;
  return dtype == 0 ? at_bwd_f32(p, pk, stat, st) : dtype == 1 ? at_bwd_f16(p, pk, stat, st) : at_bwd_bf16(p, pk, stat, st);
}
