// extern "C" entry points of the attention operators (declared in
// include/rvc_cuda.h): checks of the arguments, then the launches, on the
// caller's stream and with the caller's workspace.
#include "../../include/rvc_cuda.h"
#include "attn_common.cuh"
#include "context.cuh"
#include "norm_rope.cuh"

#include <cmath>

using namespace rvc;

// Defined beside the registry of capi.cu.
std::shared_ptr<Context> rvc_capi_context(int64_t h);

namespace {

template <typename F>
int32_t on_ctx(int64_t h, F&& f) {
  try {
    std::shared_ptr<Context> c = rvc_capi_context(h);
    std::lock_guard<std::mutex> lk(c->mu);
    DeviceGuard dg(c->device);
    f(c.get());
    return kOk;
  } catch (const Error& e) {
    set_error(e.msg);
    return e.code;
  } catch (const std::exception& e) {
    set_error(std::string("internal error: ") + e.what());
    return kErrState;
  } catch (...) {
    set_error("internal error");
    return kErrState;
  }
}

constexpr int64_t kMaxLen = 1 << 30;
constexpr int64_t kMaxBlocks = 2147483647ll;

BucketRule bucket_rule(int64_t buckets, int64_t both, const int32_t* borders, int32_t nborders, const char* who) {
  const std::string w = who;
  BucketRule r;
  RVC_CHECK_ARG(both == 0 || both == 1, w + ": bidirectional is 0 or 1");
  RVC_CHECK_ARG(buckets >= 1 && buckets <= kMaxBuckets, w + ": 1 to " + std::to_string(kMaxBuckets) + " buckets");
  RVC_CHECK_ARG(!both || buckets % 2 == 0, w + ": both directions need an even number of buckets");
  const int64_t half = both ? buckets / 2 : buckets;
  RVC_CHECK_ARG(nborders == half - 1, w + ": expected " + std::to_string(half - 1) + " borders, got " +
                                          std::to_string(nborders));
  RVC_CHECK_ARG(borders || nborders == 0, w + ": null borders");
  r.n = (int)buckets;
  r.both = (int)both;
  r.nb = nborders;
  for (int i = 0; i < nborders; ++i) {
    RVC_CHECK_ARG(borders[i] >= 1 && (i == 0 || borders[i] >= borders[i - 1]), w + ": borders must be positive and ascend");
    r.border[i] = borders[i];
  }
  return r;
}

AttnArgs attn_args(const int64_t* d, int32_t n, const char* who) {
  const std::string w = who;
  RVC_CHECK_ARG(d && n == 29, w + ": desc holds 29 values");
  AttnArgs a;
  RVC_CHECK_ARG(d[0] >= 0 && d[0] <= 2, w + ": type is 0 (float32), 1 (bfloat16) or 2 (float16)");
  for (int i = 1; i <= 6; ++i) RVC_CHECK_ARG(d[i] >= 0 && d[i] <= kMaxLen, w + ": size out of range");
  RVC_CHECK_ARG(d[2] >= 1 && d[3] >= 1 && d[2] % d[3] == 0, w + ": Hq must be a multiple of Hkv");
  RVC_CHECK_ARG(d[6] >= 1 && d[6] <= 128, w + ": head dimensions 1 to 128 are supported");
  a.type = (int)d[0];
  a.B = (int)d[1], a.Hq = (int)d[2], a.Hkv = (int)d[3], a.Lq = (int)d[4], a.Lk = (int)d[5], a.D = (int)d[6];
  // grids are one-dimensional over (batch, head, tile)
  RVC_CHECK_ARG(d[1] * d[2] <= kMaxBlocks && (d[1] * d[2] == 0 || (d[4] + d[5]) / 64 + 2 <= kMaxBlocks / (d[1] * d[2])),
                w + ": batch x heads x length out of range");
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = d[7 + i], a.ks[i] = d[10 + i], a.vs[i] = d[13 + i];
    a.dos[i] = d[23 + i], a.os[i] = d[26 + i];
  }
  RVC_CHECK_ARG(d[16] == 0 || d[16] == 32 || d[16] == 64, w + ": kv_lens are int32 or int64");
  a.lens64 = d[16] == 64;
  a.mask_b = d[17], a.mask_k = d[18];
  a.causal = d[19] != 0;
  RVC_CHECK_ARG(d[20] >= -2 * kMaxLen && d[20] <= 2 * kMaxLen, w + ": q_offset out of range");
  a.q_off = d[20];
  RVC_CHECK_ARG(d[21] >= 0 && (d[21] == 0 || d[2] <= 65535), w + ": buckets or heads of the bias out of range");
  return a;
}

// Kernels hold the scale, and the scale times log2 e, in 32 bits.
float scale_arg(const char* who, double scale) {
  RVC_CHECK_ARG(std::abs(scale) <= 0x1p127, std::string(who) + ": the scale is not finite in float32");
  return (float)scale;
}

void check_ws(const char* who, const void* ws, int64_t have, int64_t need) {
  RVC_CHECK_ARG(need == 0 || (ws && reinterpret_cast<uintptr_t>(ws) % 16 == 0),
                std::string(who) + ": the workspace is null or not aligned to 16 bytes");
  RVC_CHECK_ARG(have >= need, std::string(who) + ": the workspace holds " + std::to_string(have) + " of " +
                                  std::to_string(need) + " bytes");
}

// Values of a type lie on a multiple of its size.
void check_ptr(const char* who, const char* name, const void* p, int64_t size) {
  RVC_CHECK_ARG(p, std::string(who) + ": null " + name);
  RVC_CHECK_ARG(reinterpret_cast<uintptr_t>(p) % size == 0, std::string(who) + ": misaligned " + name);
}

void check_opt(const char* who, const char* name, const void* p, int64_t size) {
  if (p && size) check_ptr(who, name, p, size);
}

void zero(void* p, int64_t bytes, cudaStream_t st) {
  if (bytes > 0) RVC_CUDA_TRY(cudaMemsetAsync(p, 0, bytes, st));
}

}  // namespace

extern "C" {

int32_t rvc_cuda_attention_workspace(int64_t ctx, const int64_t* desc, int32_t ndesc, int32_t backward, int64_t* bytes) {
  return on_ctx(ctx, [&](Context* c) {
    const AttnArgs a = attn_args(desc, ndesc, "attention");
    RVC_CHECK_ARG(bytes, "attention: null result");
    *bytes = attn_workspace(a, desc[21] > 0, backward != 0, c->num_sms());
  });
}

int32_t rvc_cuda_attention_device(int64_t ctx, void* stream, const int64_t* desc, int32_t ndesc, double scale,
                                  const void* q, const void* k, const void* v, const void* kv_lens,
                                  const uint8_t* key_mask, const void* table, const int32_t* borders, int32_t nborders,
                                  void* out, float* lse, void* ws, int64_t ws_bytes) {
  return on_ctx(ctx, [&](Context* c) {
    const char* who = "attention";
    AttnArgs a = attn_args(desc, ndesc, who);
    const int64_t es = type_size(a.type), rows = (int64_t)a.B * a.Hq * a.Lq;
    if (rows == 0) return;
    check_ptr(who, "q", q, es);
    if (a.Lk > 0) check_ptr(who, "k", k, es), check_ptr(who, "v", v, es);
    check_ptr(who, "out", out, es);
    check_ptr(who, "lse", lse, 4);
    RVC_CHECK_ARG((desc[16] != 0) == (kv_lens != nullptr), "attention: kv_lens and their width do not agree");
    RVC_CHECK_ARG((desc[21] != 0) == (table != nullptr), "attention: table and bucket count do not agree");
    check_opt(who, "kv_lens", kv_lens, desc[16] / 8);
    check_opt(who, "table", table, es);
    a.q = q, a.k = k, a.v = v, a.lens = kv_lens, a.mask = key_mask;
    a.out = out, a.lse = lse, a.scale = scale_arg(who, scale), a.err = c->d_err;
    BucketRule rule;
    if (desc[21]) rule = bucket_rule(desc[21], desc[22], borders, nborders, who);
    check_ws(who, ws, ws_bytes, attn_workspace(a, desc[21] > 0, false, c->num_sms()));
    attn_forward(a, table, desc[21] ? &rule : nullptr, ws, c->num_sms(), (cudaStream_t)stream);
  });
}

int32_t rvc_cuda_attention_backward_device(int64_t ctx, void* stream, const int64_t* desc, int32_t ndesc, double scale,
                                           const void* dout, const void* q, const void* k, const void* v,
                                           const void* out, const float* lse, const void* kv_lens,
                                           const uint8_t* key_mask, const void* table, const int32_t* borders,
                                           int32_t nborders, void* dq, void* dk, void* dv, void* dtable, void* ws,
                                           int64_t ws_bytes) {
  return on_ctx(ctx, [&](Context* c) {
    const char* who = "attention_backward";
    AttnArgs a = attn_args(desc, ndesc, who);
    const int64_t es = type_size(a.type), rows = (int64_t)a.B * a.Hq * a.Lq, keys = (int64_t)a.B * a.Hkv * a.Lk;
    RVC_CHECK_ARG((desc[16] != 0) == (kv_lens != nullptr) || a.B == 0,
                  "attention_backward: kv_lens and their width do not agree");
    RVC_CHECK_ARG((desc[21] != 0) == (table != nullptr), "attention_backward: table and bucket count do not agree");
    check_opt(who, "kv_lens", kv_lens, desc[16] / 8);
    check_opt(who, "table", table, es);
    if (rows > 0) {
      check_ptr(who, "dout", dout, es), check_ptr(who, "q", q, es), check_ptr(who, "out", out, es);
      check_ptr(who, "lse", lse, 4);
      check_ptr(who, "dq", dq, es);
    }
    if (keys > 0) {
      check_ptr(who, "k", k, es), check_ptr(who, "v", v, es);
      check_ptr(who, "dk", dk, es), check_ptr(who, "dv", dv, es);
    }
    BucketRule rule;
    if (desc[21]) {
      rule = bucket_rule(desc[21], desc[22], borders, nborders, who);
      check_ptr(who, "dtable", dtable, es);
    }
    cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0 || keys == 0) {  // no pair: every gradient is zero
      zero(dq, rows * a.D * es, st);
      zero(dk, keys * a.D * es, st);
      zero(dv, keys * a.D * es, st);
      if (desc[21]) zero(dtable, desc[21] * a.Hq * es, st);
      return;
    }
    a.q = q, a.k = k, a.v = v, a.lens = kv_lens, a.mask = key_mask;
    a.dout = dout, a.fout = out, a.lse = const_cast<float*>(lse), a.scale = scale_arg(who, scale);
    a.dq = dq, a.dk = dk, a.dv = dv, a.err = c->d_err;
    check_ws(who, ws, ws_bytes, attn_workspace(a, desc[21] > 0, true, c->num_sms()));
    attn_backward(a, table, desc[21] ? &rule : nullptr, dtable, ws, c->num_sms(), st);
  });
}

// desc of relative_bias
static void bias_sizes(const int64_t* d, int32_t n, const char* who) {
  const std::string w = who;
  RVC_CHECK_ARG(d && n == 11, w + ": desc holds 11 values");
  RVC_CHECK_ARG(d[0] >= 0 && d[0] <= 2, w + ": type is 0 (float32), 1 (bfloat16) or 2 (float16)");
  // lengths and heads are grid dimensions of 65535 blocks at most
  RVC_CHECK_ARG(d[1] >= 0 && d[2] >= 0 && d[1] <= 65535 && d[2] <= 65535 && d[1] * d[2] <= 65535,
                w + ": batch x heads out of range");
  RVC_CHECK_ARG(d[3] >= 0 && d[4] >= 0 && d[3] <= (1 << 21) - 32 && d[4] <= kMaxLen, w + ": length out of range");
  RVC_CHECK_ARG(d[5] >= -2 * kMaxLen && d[5] <= 2 * kMaxLen, w + ": q_offset out of range");
}

int32_t rvc_cuda_relative_bias_device(int64_t ctx, void* stream, const int64_t* desc, int32_t ndesc, const void* table,
                                      const int32_t* borders, int32_t nborders, void* out) {
  return on_ctx(ctx, [&](Context*) {
    const char* who = "relative_bias";
    bias_sizes(desc, ndesc, who);
    const BucketRule rule = bucket_rule(desc[6], desc[7], borders, nborders, who);
    if (desc[2] * desc[3] * desc[4] == 0) return;
    const int64_t es = type_size((int)desc[0]);
    check_ptr(who, "table", table, es);
    check_ptr(who, "out", out, es);
    relbias_forward((int)desc[0], (int)desc[2], desc[3], desc[4], desc[5], table, rule, out, (cudaStream_t)stream);
  });
}

int32_t rvc_cuda_relative_bias_workspace(int64_t ctx, const int64_t* desc, int32_t ndesc, int64_t* bytes) {
  return on_ctx(ctx, [&](Context* c) {
    bias_sizes(desc, ndesc, "relative_bias_backward");
    RVC_CHECK_ARG(bytes, "relative_bias_backward: null result");
    *bytes = desc[1] * desc[2] * desc[3] * desc[4] == 0
                 ? 0
                 : relbias_backward_workspace((int)desc[1], (int)desc[2], desc[3], desc[4], c->num_sms());
  });
}

int32_t rvc_cuda_relative_bias_backward_device(int64_t ctx, void* stream, const int64_t* desc, int32_t ndesc,
                                               const void* dbias, const int32_t* borders, int32_t nborders,
                                               void* dtable, void* ws, int64_t ws_bytes) {
  return on_ctx(ctx, [&](Context* c) {
    const char* who = "relative_bias_backward";
    bias_sizes(desc, ndesc, who);
    const BucketRule rule = bucket_rule(desc[6], desc[7], borders, nborders, who);
    const int64_t es = type_size((int)desc[0]);
    if (desc[2] == 0) return;
    check_ptr(who, "dtable", dtable, es);
    if (desc[1] * desc[3] * desc[4] == 0) return zero(dtable, desc[6] * desc[2] * es, (cudaStream_t)stream);
    check_ptr(who, "dbias", dbias, es);
    check_ws(who, ws, ws_bytes,
             relbias_backward_workspace((int)desc[1], (int)desc[2], desc[3], desc[4], c->num_sms()));
    relbias_backward((int)desc[0], (int)desc[1], (int)desc[2], desc[3], desc[4], desc + 8, desc[5], dbias, rule, dtable,
                     ws, c->num_sms(), (cudaStream_t)stream);
  });
}

static RopeArgs rope_args(const int64_t* d, int32_t n, double eps, const char* who) {
  const std::string w = who;
  RVC_CHECK_ARG(d && n == 25, w + ": desc holds 25 values");
  RopeArgs a;
  RVC_CHECK_ARG(d[0] >= 0 && d[0] <= 2, w + ": type is 0 (float32), 1 (bfloat16) or 2 (float16)");
  RVC_CHECK_ARG(d[1] == 0 || d[1] == d[0], w + ": weights are float32 or of the inputs' type");
  RVC_CHECK_ARG(d[2] >= 0 && d[3] >= 0 && d[2] <= kMaxLen && d[3] <= kMaxLen, w + ": size out of range");
  RVC_CHECK_ARG(d[4] >= 1 && d[5] >= 0 && d[4] + d[5] <= 65536, w + ": heads out of range");
  RVC_CHECK_ARG(d[6] >= 2 && d[6] <= 256 && d[6] % 2 == 0, w + ": head dimensions 2 to 256, even, are supported");
  RVC_CHECK_ARG(d[7] >= 0 && d[7] <= d[6] && d[7] % 2 == 0, w + ": the rotated part is even and at most the head dimension");
  RVC_CHECK_ARG(d[8] >= 0, w + ": negative table length");
  RVC_CHECK_ARG(d[10] == 0 || d[10] == 32 || d[10] == 64, w + ": positions are int32 or int64");
  RVC_CHECK_ARG(eps >= 0.0, w + ": eps must not be negative");
  a.type = (int)d[0], a.wtype = (int)d[1], a.B = (int)d[2], a.L = (int)d[3], a.Hq = (int)d[4], a.Hk = (int)d[5];
  a.D = (int)d[6], a.R = (int)d[7], a.P = d[8], a.interleaved = d[9] != 0, a.pos64 = d[10] == 64;
  a.pos_b = d[11], a.pos_l = d[12];
  for (int i = 0; i < 3; ++i) a.qs[i] = d[13 + i], a.ks[i] = d[16 + i], a.gqs[i] = d[19 + i], a.gks[i] = d[22 + i];
  a.eps = (float)eps;
  return a;
}

static void rope_tables(RopeArgs& a, const int64_t* d, const float* cos, const float* sin, const void* pos,
                        const char* who) {
  if (a.R > 0 && a.P > 0) check_ptr(who, "cos", cos, 4), check_ptr(who, "sin", sin, 4);
  RVC_CHECK_ARG((d[10] != 0) == (pos != nullptr), std::string(who) + ": positions and their width do not agree");
  check_opt(who, "positions", pos, d[10] / 8);
  RVC_CHECK_ARG(pos || a.R == 0 || a.L <= a.P, std::string(who) + ": the tables hold " + std::to_string(a.P) +
                                                   " positions, fewer than the rows");
  a.cos = cos, a.sin = sin, a.pos = pos;
}

int32_t rvc_cuda_qk_norm_rope_device(int64_t ctx, void* stream, const int64_t* desc, int32_t ndesc, double eps,
                                     const void* q, const void* k, const void* q_weight, const void* k_weight,
                                     const float* cos, const float* sin, const void* positions, void* qo, void* ko) {
  return on_ctx(ctx, [&](Context* c) {
    const char* who = "qk_norm_rope";
    RopeArgs a = rope_args(desc, ndesc, eps, who);
    if ((int64_t)a.B * a.L == 0) return;
    const int64_t es = type_size(a.type), wsz = type_size(a.wtype);
    check_ptr(who, "q", q, es), check_ptr(who, "qo", qo, es), check_ptr(who, "q_weight", q_weight, wsz);
    if (a.Hk) check_ptr(who, "k", k, es), check_ptr(who, "ko", ko, es), check_ptr(who, "k_weight", k_weight, wsz);
    rope_tables(a, desc, cos, sin, positions, who);
    a.q = q, a.k = k, a.wq = q_weight, a.wk = a.Hk ? k_weight : q_weight, a.oq = qo, a.ok = ko;
    rope_forward(a, c->num_sms(), (cudaStream_t)stream);
  });
}

int32_t rvc_cuda_qk_norm_rope_workspace(int64_t ctx, const int64_t* desc, int32_t ndesc, int64_t* bytes) {
  return on_ctx(ctx, [&](Context* c) {
    const RopeArgs a = rope_args(desc, ndesc, 0.0, "qk_norm_rope_backward");
    RVC_CHECK_ARG(bytes, "qk_norm_rope_backward: null result");
    *bytes = rope_backward_workspace(a, c->num_sms());
  });
}

int32_t rvc_cuda_qk_norm_rope_backward_device(int64_t ctx, void* stream, const int64_t* desc, int32_t ndesc, double eps,
                                              const void* dqo, const void* dko, const void* q, const void* k,
                                              const void* q_weight, const void* k_weight, const float* cos,
                                              const float* sin, const void* positions, void* dq, void* dk,
                                              void* dq_weight, void* dk_weight, void* ws, int64_t ws_bytes) {
  return on_ctx(ctx, [&](Context* c) {
    const char* who = "qk_norm_rope_backward";
    RopeArgs a = rope_args(desc, ndesc, eps, who);
    const int64_t es = type_size(a.type), wsz = type_size(a.wtype);
    check_ptr(who, "dq_weight", dq_weight, wsz);
    if (a.Hk) check_ptr(who, "dk_weight", dk_weight, wsz);
    cudaStream_t st = (cudaStream_t)stream;
    if ((int64_t)a.B * a.L == 0) {
      zero(dq_weight, a.D * wsz, st);
      if (a.Hk) zero(dk_weight, a.D * wsz, st);
      return;
    }
    check_ptr(who, "dqo", dqo, es), check_ptr(who, "q", q, es), check_ptr(who, "dq", dq, es);
    check_ptr(who, "q_weight", q_weight, wsz);
    if (a.Hk) {
      check_ptr(who, "dko", dko, es), check_ptr(who, "k", k, es), check_ptr(who, "dk", dk, es);
      check_ptr(who, "k_weight", k_weight, wsz);
    }
    rope_tables(a, desc, cos, sin, positions, who);
    check_ws(who, ws, ws_bytes, rope_backward_workspace(a, c->num_sms()));
    a.q = q, a.k = k, a.gq = dqo, a.gk = dko, a.wq = q_weight, a.wk = a.Hk ? k_weight : q_weight;
    a.oq = dq, a.ok = dk, a.dwq = dq_weight, a.dwk = a.Hk ? dk_weight : nullptr;
    rope_backward(a, ws, c->num_sms(), st);
  });
}

}  // extern "C"
