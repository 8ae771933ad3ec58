// Attention operators: choice of kernel, workspace, the expanded bias and the
// gradient of its table.
#include "attn_common.cuh"
#include "context.cuh"

#include <algorithm>

namespace rvc {

namespace {

constexpr int64_t kAlign = 256;
int64_t up(int64_t n, int64_t g = kAlign) { return (n + g - 1) / g * g; }

// Entries below this mask their pairs, as -inf does.  Further down a score keeps
// nothing of its product in 32 bits, and the log sum of a row that meets only
// such entries, which the backward pass takes the weights from, is off by more
// than the weights themselves: at -1e9 by factors of 2^64.  The lowest float16
// (-65504) is still a number; its log sums are good to 2^-8.
constexpr float kMasked = -65536.f;

template <typename T>
__global__ void expand_bias_kernel(const T* __restrict__ table, int H, long long ld, long long d0, float mul,
                                   const __grid_constant__ BucketRule rule, float* __restrict__ diag) {
  const long long x = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (x >= ld) return;
  const int b = bucket_of(rule, x - d0);
  for (int h = 0; h < H; ++h) {
    const float t = to_f(table[(long long)b * H + h]);
    diag[h * ld + x] = t < kMasked ? -INFINITY : t * mul;
  }
}

// sums[h][x] = sum over batch entries and tiles of the diagonal j - i = x - (Lq - 1).
// Tiles of BM queries (by_key = 0) hold it at x - (Lq - 1) + BM - 1 + t BM, tiles
// of BM keys (by_key arrays each) at (Lq - 1) - x + BM - 1 + t BM; there the last
// two entries of an array are sums that lie whole in the last bucket behind / ahead.
// Block: 32 diagonals x 8 shares of the (tile, batch) list, joined in order.
__global__ void __launch_bounds__(256) diag_sums_kernel(const float* __restrict__ ws, int B, int H, int nt, int BM,
                                                        int by_key, long long ld, long long Lq, long long Lk,
                                                        double* __restrict__ sums, double* __restrict__ far) {
  __shared__ double red[8][32];
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  const long long x = (long long)blockIdx.x * 32 + lane;
  const int h = blockIdx.y;
  const long long n = Lq + Lk - 1;
  const long long d = x - (Lq - 1), top = by_key ? ld - 2 : ld;
  const int na = by_key ? by_key : 1;
  double s = 0.0;
  if (x < n || (x < n + 2 && by_key))
#pragma unroll 4
    for (long long k = y; k < (long long)B * nt * na; k += 8) {
      const long long u = k / B, b = k % B, t = u / na;
      const long long e = x < n ? (by_key ? -d : d) + BM - 1 + t * BM : top + (x - n);
      if (e >= 0 && (e < top || x >= n)) s += ws[((b * H + h) * nt * na + u) * ld + e];
    }
  red[y][lane] = s;
  __syncthreads();
  if (y) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += red[k][lane];
  if (x < n) sums[h * n + x] = s;
  else if (x < n + 2) far[h * 2 + (x - n)] = s;
}

// One block per (bucket, head): its diagonals are a run, found with the borders.
template <typename T>
__global__ void bucket_sums_kernel(const double* __restrict__ sums, const double* __restrict__ far_sums, int H,
                                   long long Lq, long long Lk, long long q_off,
                                   const __grid_constant__ BucketRule rule, T* __restrict__ dtable) {
  __shared__ double red[128];
  const int b = blockIdx.x, h = blockIdx.y;
  // relative positions [lo, hi) of bucket b
  const long long far = (long long)1 << 40;
  const int half = rule.both ? rule.n / 2 : rule.n;
  const bool ahead = rule.both && b >= half;
  const int f = ahead ? b - half : b;
  const long long a0 = f == 0 ? 0 : (f <= rule.nb ? rule.border[f - 1] : far), a1 = f < rule.nb ? rule.border[f] : far;
  long long lo, hi;  // distances [a0, a1): behind r = -a, ahead r = a (a > 0)
  if (ahead) {
    lo = a0 > 1 ? a0 : 1;
    hi = a1;
  } else {
    lo = 1 - a1;
    hi = 1 - a0;
    if (!rule.both && f == 0) hi = far;  // one direction: every key ahead has distance 0
  }
  // diagonal x holds r = x - (Lq - 1) - q_off
  const long long x0 = max(0ll, lo + (Lq - 1) + q_off), x1 = min(Lq + Lk - 1, hi + (Lq - 1) + q_off);
  double s = 0.0;
  for (long long x = x0 + threadIdx.x; x < x1; x += 128) s += sums[h * (Lq + Lk - 1) + x];
  if (far_sums && threadIdx.x == 0) {
    if (!ahead && f == rule.nb) s += far_sums[2 * h];
    if (rule.both ? ahead && f == rule.nb : f == 0) s += far_sums[2 * h + 1];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int n = 64; n; n >>= 1) {
    if (threadIdx.x < n) red[threadIdx.x] += red[threadIdx.x + n];
    __syncthreads();
  }
  if (threadIdx.x == 0) dtable[(long long)b * H + h] = from_f<T>((float)red[0]);
}

// Workspace.  The largest part is the table's gradient: the diagonal sums of every
// tile of every (batch entry, query head), 4 B Hq (Lk / 128) (Lq + 130) bytes on the
// 16-bit tiles (twice for heads above 64), 4 B Hq (Lq / 64) (Lk + 64) elsewhere: 8.6
// GB for 32 heads of 128 at 65536 x 65536.
struct Layout {
  int64_t diag = -1, po = -1, pml = -1, delta = -1, lse2 = -1, dws = -1, sums = -1, far = -1, split = -1, bytes = 0;
  int nsplit = 1, BM = 64, nt = 0;
  int64_t diag_ld = 0, diag0 = 0, dws_ld = 0, row_ld = 0;
  bool tc = false;
};

Layout plan(const AttnArgs& a, bool bias, bool backward, int sms, bool tc) {
  Layout l;
  l.tc = tc;
  auto take = [&](int64_t n) {
    const int64_t at = l.bytes;
    l.bytes += up(n);
    return at;
  };
  const int64_t rows = (int64_t)a.B * a.Hq * a.Lq;
  if (rows == 0 || (backward && a.Lk == 0)) return l;  // no launch
  if (bias) {
    l.diag0 = up(a.Lq, kDiagTile);
    l.diag_ld = l.diag0 + up(a.Lk, 128) + 128;
    l.diag = take(4 * l.diag_ld * a.Hq);
  }
  if (!backward) {
    bool parts = false;
    if (!tc) l.nsplit = attn_mma_splits(a, sms, &parts);
    else parts = (l.nsplit = attn_tc_splits(a, sms)) > 1;
    if (tc && a.type == kF32) l.split = take(attn_tc_f32_workspace(a));
    if (parts) {
      l.po = take(4 * rows * a.D * l.nsplit);
      l.pml = take(8 * rows * l.nsplit);
    }
    return l;
  }
  l.row_ld = tc ? up(a.Lq, 128) : a.Lq;
  l.delta = take(4 * l.row_ld * a.B * a.Hq);
  if (tc && (l.nsplit = attn_tc_bwd_shares(a, sms)) > 1) {
    const int64_t n = 4ll * l.nsplit * a.B * a.Lk * a.Hkv * a.D;
    l.po = take(n);
    l.pml = take(n);
  }
  if (tc) l.lse2 = take(4 * l.row_ld * a.B * a.Hq);
  if (bias) {
    l.BM = tc ? 128 : 64;
    const int64_t tiled = tc ? a.Lk : a.Lq, along = tc ? a.Lq : a.Lk;
    l.nt = (int)((tiled + l.BM - 1) / l.BM);
    l.dws_ld = up(along, l.BM) + l.BM + (tc ? 2 : 0);
    l.dws = take(4 * l.dws_ld * l.nt * (tc ? attn_tc_bwd_arrays(a) : 1) * a.B * a.Hq);
    l.sums = take(8 * ((int64_t)a.Lq + a.Lk - 1) * a.Hq);
    l.far = take(16 * a.Hq);
  }
  return l;
}

bool use_tc(const AttnArgs& a, bool backward) { return backward ? attn_tc_bwd_fits(a) : attn_tc_fits(a) || attn_tc_f32_fits(a); }

template <typename P>
P* at(void* ws, int64_t off) {
  return off < 0 ? nullptr : reinterpret_cast<P*>(static_cast<char*>(ws) + off);
}

void apply(AttnArgs& a, const Layout& l, void* ws) {
  a.diag = at<float>(ws, l.diag);
  a.diag_ld = l.diag_ld;
  a.diag0 = (int)l.diag0;
  a.nsplit = l.nsplit;
  a.po = at<float>(ws, l.po);
  a.pml = at<float>(ws, l.pml);
  a.delta = at<float>(ws, l.delta);
  a.lse2 = at<float>(ws, l.lse2);
  a.row_ld = l.row_ld;
  a.dws = at<float>(ws, l.dws);
  a.dws_ld = l.dws_ld;
}

}  // namespace

void attn_expand_bias(const AttnArgs& a, const void* table, const BucketRule& rule, float* diag, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.diag_ld + 255) / 256);
  const long long d0 = a.diag0 + a.q_off;
  switch (a.type) {
    case kF32:
      expand_bias_kernel<<<grid, 256, 0, st>>>((const float*)table, a.Hq, a.diag_ld, d0, kLog2e, rule, diag);
      break;
    case kBf16:
      expand_bias_kernel<<<grid, 256, 0, st>>>((const __nv_bfloat16*)table, a.Hq, a.diag_ld, d0, kLog2e, rule, diag);
      break;
    default:
      expand_bias_kernel<<<grid, 256, 0, st>>>((const __half*)table, a.Hq, a.diag_ld, d0, kLog2e, rule, diag);
  }
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
}

void relbias_bucket_sums(int type, int H, int64_t Lq, int64_t Lk, int64_t q_off, const double* sums,
                         const double* far, const BucketRule& rule, void* dtable, cudaStream_t st) {
  const dim3 grid(rule.n, H);
  switch (type) {
    case kF32: bucket_sums_kernel<<<grid, 128, 0, st>>>(sums, far, H, Lq, Lk, q_off, rule, (float*)dtable); break;
    case kBf16: bucket_sums_kernel<<<grid, 128, 0, st>>>(sums, far, H, Lq, Lk, q_off, rule, (__nv_bfloat16*)dtable); break;
    default: bucket_sums_kernel<<<grid, 128, 0, st>>>(sums, far, H, Lq, Lk, q_off, rule, (__half*)dtable);
  }
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
}

// Enough for either choice of kernel: the choice asks for aligned pointers,
// which a query for the size does not have.
int64_t attn_workspace(const AttnArgs& a, bool bias, bool backward, int sms) {
  const int64_t n = plan(a, bias, backward, sms, false).bytes;
  return use_tc(a, backward) ? std::max(n, plan(a, bias, backward, sms, true).bytes) : n;
}

void attn_forward(AttnArgs a, const void* table, const BucketRule* rule, void* ws, int sms, cudaStream_t st) {
  const Layout l = plan(a, rule != nullptr, false, sms, use_tc(a, false));
  apply(a, l, ws);
  if (rule) {
    a.far = rule->nb ? rule->border[rule->nb - 1] : 1;
    a.far_both = rule->both;
    attn_expand_bias(a, table, *rule, const_cast<float*>(a.diag), st);
  }
  if (l.tc && a.type == kF32)
    attn_tc_f32_forward(a, at<char>(ws, l.split), sms, st);
  else if (l.tc)
    attn_tc_forward(a, st);
  else
    attn_mma_forward(a, st);
}

void attn_backward(AttnArgs a, const void* table, const BucketRule* rule, void* dtable, void* ws, int sms,
                   cudaStream_t st) {
  const Layout l = plan(a, rule != nullptr, true, sms, use_tc(a, true));
  apply(a, l, ws);
  if (rule) {
    a.far = rule->nb ? rule->border[rule->nb - 1] : 1;
    a.far_both = rule->both;
    attn_expand_bias(a, table, *rule, const_cast<float*>(a.diag), st);
  }
  if (l.tc)
    attn_tc_backward(a, st);
  else
    attn_mma_backward(a, st);
  if (rule) {
    double *sums = at<double>(ws, l.sums), *far = at<double>(ws, l.far);
    const int64_t n = (int64_t)a.Lq + a.Lk + 1;
    diag_sums_kernel<<<dim3((unsigned)((n + 31) / 32), a.Hq), 256, 0, st>>>(
        a.dws, a.B, a.Hq, l.nt, l.BM, l.tc ? attn_tc_bwd_arrays(a) : 0, l.dws_ld, a.Lq, a.Lk, sums, far);
    note_launch();
    RVC_CUDA_TRY(cudaGetLastError());
    relbias_bucket_sums(a.type, a.Hq, a.Lq, a.Lk, a.q_off, sums, far, *rule, dtable, st);
  }
}

}  // namespace rvc
