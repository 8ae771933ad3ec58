// The learned relative position bias as a tensor and the gradient of its table.
//   bias[h][i][j] = T[bucket(j - i - q_offset)][h]
//   dT[b][h] = sum of dbias[.][h][i][j] over the batch and the pairs of bucket b
// Both hold one value per diagonal: the forward pass writes every pair once
// from a row of Lq + Lk - 1 values, the backward pass reads every pair once
// into as many sums, and a small kernel adds those up per bucket.
//
// Measured: 12 x 499 x 1499 fp32 written in 11 us (36 MB; that is the kernel, alone
// and cold: each block waits for its look-ups, which search the borders with
// divergent indices, and then stores four bytes a thread); the gradient of 4 x 16 x
// 4095 x 4095 bf16 (2.1 GB) in 424 to 439 us, 368 of them the pass (73 % of DRAM).
#include "attn_common.cuh"
#include "context.cuh"

#include <algorithm>

namespace rvc {

namespace {

constexpr int kRows = 64;  // rows of one block

// Block: kRows rows x 256 columns of one head; the 256 + kRows - 1 values of
// its diagonals are looked up once, in shared memory.
template <typename T>
__global__ void __launch_bounds__(256) relbias_fwd_kernel(const T* __restrict__ table, int H, long long Lq,
                                                          long long Lk, long long q_off,
                                                          const __grid_constant__ BucketRule rule,
                                                          T* __restrict__ out) {
  __shared__ T val[256 + kRows];
  const long long j0 = (long long)blockIdx.x * 256, i0 = (long long)blockIdx.y * kRows;
  const int h = blockIdx.z;
  for (int x = threadIdx.x; x < 256 + kRows - 1; x += 256)
    val[x] = table[(long long)bucket_of(rule, j0 + x - (kRows - 1) - i0 - q_off) * H + h];
  __syncthreads();
  const long long j = j0 + threadIdx.x;
  if (j >= Lk) return;
  T* o = out + ((long long)h * Lq + i0) * Lk + j;
  const int n = (int)min((long long)kRows, Lq - i0);
#pragma unroll 8
  for (int r = 0; r < n; ++r) o[(long long)r * Lk] = val[threadIdx.x + (kRows - 1) - r];
}

// Sums along the diagonals of kBwdRows rows.  A step down and right moves si + 1
// values on, so along E rows (E values to 16 bytes) the alignment of a diagonal
// comes back: the rows go by in E classes of equal alignment (one, when E
// divides si + 1), in each of which every thread reads aligned runs of 16 bytes,
// E diagonals wide, into registers; between the classes the sums move to shared
// memory, where the runs of the next class start elsewhere.
constexpr int kBwdRows = 256, kBwdThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kBwdThreads + 32) relbias_bwd_kernel(const T* __restrict__ dbias, int H, long long Lq,
                                                                  long long Lk, long long sb, long long sh,
                                                                  long long si, float* __restrict__ part) {
  constexpr int E = 16 / (int)sizeof(T), W = kBwdThreads * E;  // diagonals of a block
  __shared__ float sum[W + E];
  const long long n = Lq + Lk - 1;
  const long long x0 = (long long)blockIdx.x * W;              // diagonals x0 .. x0 + W - 1: j - i = x - (Lq - 1)
  const long long r0 = (long long)blockIdx.y * kBwdRows, r1 = min(Lq, r0 + kBwdRows);
  const int h = blockIdx.z % H, b = blockIdx.z / H;
  // nothing of these rows meets these diagonals: the join leaves them out too
  if (x0 - (Lq - 1) + r0 >= Lk || x0 + W - 1 - (Lq - 1) + r1 - 1 < 0) return;
  const T* base = dbias + b * sb + h * sh;
  for (int x = threadIdx.x; x < W + E; x += kBwdThreads + 32) sum[x] = 0.f;
  __syncthreads();
  int classes = E;  // E / gcd(E, si + 1)
  while (classes > 1 && ((si + 1) * (classes / 2)) % E == 0) classes /= 2;
  for (int c = 0; c < classes; ++c) {
    // the first value of this thread's run lies `off` diagonals before x0 + E tid
    const long long a0 = (long long)(reinterpret_cast<uintptr_t>(base) / sizeof(T)) + (r0 + c) * (si + 1) + x0 - (Lq - 1);
    const int off = (int)((a0 % E + E) % E);
    float acc[E];
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] = 0.f;
    // one run more than the threads' reaches the last diagonals when off > 0
    if (const int run = threadIdx.x; run < kBwdThreads + (off > 0)) {
      const long long d = x0 - (Lq - 1) + (long long)run * E - off;  // j - i of the run's first value
      const T* p = base + d;
      // the first row of the class from x on
      const auto from = [&](long long x) { return r0 + c + (max(0ll, x - r0 - c) + classes - 1) / classes * classes; };
      // rows where the whole run lies inside [0, Lk), and the few before and
      // behind them where a part of it does
      const long long in0 = max(r0, -d), in1 = min(r1, Lk - (E - 1) - d);
#pragma unroll 8
      for (long long i = from(in0); i < in1; i += classes) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p + i * si + i));
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] += to_f(e[k]);
      }
      const auto edge = [&](long long lo, long long hi) {
        for (long long i = from(lo); i < hi; i += classes)
#pragma unroll
          for (int k = 0; k < E; ++k)
            if (d + i + k >= 0 && d + i + k < Lk) acc[k] += to_f(p[i * si + i + k]);
      };
      edge(max(r0, -d - (E - 1)), min(r1, -d));
      edge(max(in0, Lk - (E - 1) - d), min(r1, Lk - d));
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const int at = run * E - off + k;
        if (at >= 0 && at < W) sum[at] += acc[k];
      }
    }
    __syncthreads();
  }
  float* o = part + ((long long)blockIdx.y * gridDim.z + blockIdx.z) * n;
  for (int x = threadIdx.x; x < W; x += kBwdThreads + 32)
    if (x0 + x < n) o[x0 + x] = sum[x];
}

// Joins the row chunks and the batch in 64 bits; chunk blocks that met no pair
// left nothing.
// Block: 32 diagonals x 8 shares of the list, joined in order.
__global__ void __launch_bounds__(256) relbias_join_kernel(const float* __restrict__ part, int chunks, int B, int H,
                                                           long long Lq, long long Lk, int W,
                                                           double* __restrict__ sums) {
  __shared__ double red[8][32];
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  const long long n = Lq + Lk - 1;
  const long long x = (long long)blockIdx.x * 32 + lane;
  const int h = blockIdx.y;
  const long long x0 = x / W * W;
  double s = 0.0;
  if (x < n)
#pragma unroll 4
    for (int e = y; e < chunks * B; e += 8) {
      const int c = e / B, b = e % B;
      const long long r0 = (long long)c * kBwdRows, r1 = min(Lq, r0 + kBwdRows);
      if (x0 - (Lq - 1) + r0 < Lk && x0 + W - 1 - (Lq - 1) + r1 - 1 >= 0)
        s += part[(((long long)c * B + b) * H + h) * n + x];
    }
  red[y][lane] = s;
  __syncthreads();
  if (y || x >= n) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += red[k][lane];
  sums[h * n + x] = s;
}

template <typename T>
void fwd_t(int H, int64_t Lq, int64_t Lk, int64_t q_off, const void* table, const BucketRule& rule, void* out,
           cudaStream_t st) {
  const dim3 grid((unsigned)((Lk + 255) / 256), (unsigned)((Lq + kRows - 1) / kRows), H);
  relbias_fwd_kernel<T><<<grid, 256, 0, st>>>((const T*)table, H, Lq, Lk, q_off, rule, (T*)out);
}
template <typename T>
int bwd_t(int B, int H, int64_t Lq, int64_t Lk, const int64_t* s, const void* dbias, float* part, cudaStream_t st) {
  constexpr int W = kBwdThreads * 16 / (int)sizeof(T);
  const dim3 grid((unsigned)((Lq + Lk - 1 + W - 1) / W), (unsigned)((Lq + kBwdRows - 1) / kBwdRows), B * H);
  relbias_bwd_kernel<T><<<grid, kBwdThreads + 32, 0, st>>>((const T*)dbias, H, Lq, Lk, s[0], s[1], s[2], part);
  return W;
}

}  // namespace

void relbias_forward(int type, int H, int64_t Lq, int64_t Lk, int64_t q_off, const void* table, const BucketRule& rule,
                     void* out, cudaStream_t st) {
  switch (type) {
    case kF32: fwd_t<float>(H, Lq, Lk, q_off, table, rule, out, st); break;
    case kBf16: fwd_t<__nv_bfloat16>(H, Lq, Lk, q_off, table, rule, out, st); break;
    default: fwd_t<__half>(H, Lq, Lk, q_off, table, rule, out, st);
  }
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
}

int64_t relbias_backward_workspace(int B, int H, int64_t Lq, int64_t Lk, int) {
  const int64_t n = Lq + Lk - 1, chunks = (Lq + kBwdRows - 1) / kBwdRows;
  return (8 * n * H + 255) / 256 * 256 + 4 * n * chunks * B * H;
}

void relbias_backward(int type, int B, int H, int64_t Lq, int64_t Lk, const int64_t* strides, int64_t q_off,
                      const void* dbias, const BucketRule& rule, void* dtable, void* ws, int, cudaStream_t st) {
  const int64_t n = Lq + Lk - 1;
  const int chunks = (int)((Lq + kBwdRows - 1) / kBwdRows);
  double* sums = static_cast<double*>(ws);
  float* part = reinterpret_cast<float*>(static_cast<char*>(ws) + (8 * n * H + 255) / 256 * 256);
  int W;
  switch (type) {
    case kF32: W = bwd_t<float>(B, H, Lq, Lk, strides, dbias, part, st); break;
    case kBf16: W = bwd_t<__nv_bfloat16>(B, H, Lq, Lk, strides, dbias, part, st); break;
    default: W = bwd_t<__half>(B, H, Lq, Lk, strides, dbias, part, st);
  }
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
  relbias_join_kernel<<<dim3((unsigned)((n + 31) / 32), H), 256, 0, st>>>(part, chunks, B, H, Lq, Lk, W, sums);
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
  relbias_bucket_sums(type, H, Lq, Lk, q_off, sums, nullptr, rule, dtable, st);
}

}  // namespace rvc
