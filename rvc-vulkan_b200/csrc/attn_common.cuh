// Shared pieces of the attention operators (attention / attention_backward,
// relative_bias, qk_norm_rope): arguments, the bucket rule of the learned
// relative position bias, element types.
//
//   s_ij = scale q_i . k_j + T[bucket(j - i - q_offset), h]
//   out_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp(s_ij)
// over the keys j that are alive: j < kv_len, key_mask[j], and (causal)
// j <= i + q_offset.  A row with no key alive gives out = 0, lse = -inf and
// zero gradients.  Scores are kept in the base-2 domain (scale and bias times
// log2 e) so that the exponential is one ex2.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>
#include <stdint.h>

namespace rvc {

struct Context;

enum AttnType : int { kF32 = 0, kBf16 = 1, kF16 = 2 };
constexpr int kMaxBuckets = 1024;  // rows of a bias table (the rule travels as a kernel parameter, 4 KB)
constexpr int kDiagTile = 256;     // granule of the expanded bias (one value per diagonal)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// border[b - 1] is the smallest distance of bucket b; `nb` of them.  With both
// directions the second half of the table's rows holds the keys ahead.
struct BucketRule {
  int n = 0, both = 0, nb = 0;
  int32_t border[kMaxBuckets];
};

__host__ __device__ __forceinline__ int bucket_of(const BucketRule& r, long long rel) {
  const long long a = r.both ? (rel < 0 ? -rel : rel) : (rel < 0 ? -rel : 0);
  int lo = 0, hi = r.nb;  // number of borders <= a
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((long long)r.border[mid] <= a)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo + (r.both && rel > 0 ? r.n / 2 : 0);
}

struct AttnArgs {
  int type = 0;
  int B = 0, Hq = 0, Hkv = 0, Lq = 0, Lk = 0, D = 0;
  const void *q = nullptr, *k = nullptr, *v = nullptr;
  // strides in elements: batch, row, head (the head's D values are contiguous)
  int64_t qs[3] = {0, 0, 0}, ks[3] = {0, 0, 0}, vs[3] = {0, 0, 0};
  const void* lens = nullptr;  // [B] int32 or int64, clamped to [0, Lk]; read through kv_len
  int lens64 = 0;
  const uint8_t* mask = nullptr;  // [B, Lk] bytes, non-zero = alive
  int64_t mask_b = 0, mask_k = 0;
  int causal = 0;
  int64_t q_off = 0;
  float scale = 0.f;             // of q . k
  const float* diag = nullptr;   // [Hq][diag_ld]: log2 e T[bucket], index j - i + diag0; nullptr = no bias
  int64_t diag_ld = 0;
  int diag0 = 0;
  void* out = nullptr;           // [B, Lq, Hq, D]
  float* lse = nullptr;          // [B, Hq, Lq]
  // keys split over nsplit blocks: unnormalised partial rows and their (max, sum)
  int nsplit = 1;
  float* po = nullptr;           // [nsplit][B][Hq][Lq][D]
  float* pml = nullptr;          // [nsplit][B][Hq][Lq][2]
  // (backward: shares of the query heads of a group, parts of dK and dV [nsplit][B][Lk][Hkv][D])
  // backward
  const void *dout = nullptr, *fout = nullptr;
  int64_t dos[3] = {0, 0, 0}, os[3] = {0, 0, 0};
  float* delta = nullptr;        // [B, Hq, row_ld] sum_j P dP of every query (attn_tc_bwd.cu: its negative)
  float* lse2 = nullptr;         // [B, Hq, row_ld] -log2 sums, -inf for a row without a key (attn_tc_bwd.cu)
  int64_t row_ld = 0;
  void *dq = nullptr, *dk = nullptr, *dv = nullptr;  // contiguous [B, L, H, D]
  float* dws = nullptr;          // diagonal sums of dS: [B][Hq][tiles][dws_ld], see attn_api.cu
  int64_t dws_ld = 0;
  int far = 0, far_both = 0;     // first distance of the last bucket; both directions have one
  int* err = nullptr;            // the context's error word, set by a bounded wait that gave up
};

// Keys of batch entry b that some query of the call may meet.  What lies behind
// is neither read as it is nor left to a product: a cache that is filled up to
// the last query's limit may hold anything past it.
__device__ __forceinline__ int kv_len(const AttnArgs& a, int b) {
  long long n = a.Lk;
  if (a.lens) n = min(n, a.lens64 ? static_cast<const long long*>(a.lens)[b] : (long long)static_cast<const int*>(a.lens)[b]);
  if (a.causal) n = min(n, a.Lq + (long long)a.q_off);
  return (int)max(n, 0ll);
}

// The second key that is alive by the mask's bytes, `len` when there is none.
// Called by whole warps; all but nearly empty masks end the search with the first
// 256 keys.  (Not inlined: inside the gradients' kernels it cost the fp32 ones
// registers and 3 % of their time.)
static __device__ __noinline__ int second_key(const uint8_t* mb, int64_t stride, int len) {
  const int lane = threadIdx.x & 31;
  int seen = 0, second = len;
  for (int j0 = 0; j0 < len && seen < 2; j0 += 256) {
    uint8_t byte[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int j = j0 + 32 * x + lane;
      byte[x] = j < len ? mb[(int64_t)j * stride] : 0;
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const uint32_t word = __ballot_sync(0xffffffffu, byte[x] != 0), rest = seen ? word : word & (word - 1);
      if (seen < 2 && rest) second = j0 + 32 * x + __ffs(rest) - 1;
      seen += __popc(word);
    }
  }
  return second;
}

// Queries before this one can meet one key of batch entry b at most, by length,
// mask and causal limit (entries of the bias that mask a pair are not looked at).
// Such a query's weight is 1 whatever the score: its dS is zero, not what the
// roundings of P and delta leave of it.  Called by whole warps.
__device__ __forceinline__ int lone_queries(const AttnArgs& a, int b, int len) {
  const int second = a.mask ? second_key(a.mask + (int64_t)b * a.mask_b, a.mask_k, len) : 1;
  if (len <= second) return a.Lq;
  return a.causal ? (int)max(0ll, min((long long)a.Lq, second - (long long)a.q_off)) : 0;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a row's sum of weights L (held over the maximum M) makes of it.  L is 0
// only where no key is alive or every score is -inf: out = 0, lse = -inf.  A NaN
// sum (a live NaN or infinity) is no such row: it goes on into both.
__device__ __forceinline__ float row_inv(float L) { return L == 0.f ? 0.f : 1.f / L; }
__device__ __forceinline__ float row_lse(float M, float L) { return L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2; }

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
// Two values in one word, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

inline int type_size(int t) { return t == kF32 ? 4 : 2; }
inline bool aligned16(const AttnArgs& a, const void* p, const int64_t* s) {
  const int64_t e = type_size(a.type);
  return (reinterpret_cast<uintptr_t>(p) % 16 == 0) && (a.D * e % 16 == 0) && (s[0] * e % 16 == 0) &&
         (s[1] * e % 16 == 0) && (s[2] * e % 16 == 0);
}

// ------------------------------------------------------------- entry points
// Each queues its kernels on `st`; throws Error on a launch error.
int64_t attn_workspace(const AttnArgs& a, bool bias, bool backward, int sms);
void attn_forward(AttnArgs a, const void* table, const BucketRule* rule, void* ws, int sms, cudaStream_t st);
void attn_backward(AttnArgs a, const void* table, const BucketRule* rule, void* dtable, void* ws, int sms,
                   cudaStream_t st);
// expanded bias: diag[h][x] = log2 e T[bucket(x - diag0 - q_off), h]
void attn_expand_bias(const AttnArgs& a, const void* table, const BucketRule& rule, float* diag, cudaStream_t st);
// kernels of attn_mma.cu (every type, stride and size)
void attn_mma_forward(const AttnArgs& a, cudaStream_t st);
void attn_mma_backward(const AttnArgs& a, cudaStream_t st);
// joins the splits of the rows in a.po, a.pml (nothing to do without them)
void attn_join(const AttnArgs& a, cudaStream_t st);
int attn_mma_splits(const AttnArgs& a, int sms, bool* workspace);

// kernels of attn_tc.cu (16-bit types, rows aligned to 16 bytes, many queries)
bool attn_tc_fits(const AttnArgs& a);
int attn_tc_splits(const AttnArgs& a, int sms);  // of attn_tc_f32.cu as well
void attn_tc_forward(const AttnArgs& a, cudaStream_t st);
// kernels of attn_tc_f32.cu (fp32, heads of up to 64 values, many queries)
bool attn_tc_f32_fits(const AttnArgs& a);
int64_t attn_tc_f32_workspace(const AttnArgs& a);
void attn_tc_f32_forward(const AttnArgs& a, void* ws, int sms, cudaStream_t st);
// kernels of attn_tc_bwd.cu (as attn_tc.cu)
bool attn_tc_bwd_fits(const AttnArgs& a);
int attn_tc_bwd_shares(const AttnArgs& a, int sms);
int attn_tc_bwd_arrays(const AttnArgs& a);  // arrays of diagonal sums to a tile of keys
void attn_tc_backward(const AttnArgs& a, cudaStream_t st);

void relbias_forward(int type, int H, int64_t Lq, int64_t Lk, int64_t q_off, const void* table, const BucketRule& rule,
                     void* out, cudaStream_t st);
int64_t relbias_backward_workspace(int B, int H, int64_t Lq, int64_t Lk, int sms);
void relbias_backward(int type, int B, int H, int64_t Lq, int64_t Lk, const int64_t* strides, int64_t q_off,
                      const void* dbias, const BucketRule& rule, void* dtable, void* ws, int sms, cudaStream_t st);
// diagonal sums [H][Lq + Lk - 1] (fp64) -> dtable [n][H] in `type`; far [H][2]
// (or nullptr): sums that lie whole in the last bucket behind / ahead
void relbias_bucket_sums(int type, int H, int64_t Lq, int64_t Lk, int64_t q_off, const double* sums,
                         const double* far, const BucketRule& rule, void* dtable, cudaStream_t st);

}  // namespace rvc
