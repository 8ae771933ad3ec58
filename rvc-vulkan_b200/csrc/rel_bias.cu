// The learned relative position bias as a tensor and the gradient of its table.
//   bias[h][i][j] = T[bucket(j - i - q_offset)][h]
//   dT[b][h] = sum of dbias[.][h][i][j] over the batch and the pairs of bucket b
// Both hold one value per diagonal: the forward pass writes every pair once
// from a row of Lq + Lk - 1 values, the backward pass reads every pair once
// into as many sums, and a small kernel adds those up per bucket.
#include "attn_common.cuh"
#include "context.cuh"

#include <algorithm>

namespace rvc {

namespace {

constexpr int kRows = 32;  // rows of one block

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

// Thread = one diagonal of a chunk of rows: consecutive threads read
// consecutive columns of every row.
template <typename T>
__global__ void __launch_bounds__(256) relbias_bwd_kernel(const T* __restrict__ dbias, int B, int H, long long Lq,
                                                          long long Lk, long long sb, long long sh, long long si,
                                                          int rows, float* __restrict__ part) {
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;  // diagonal: j - i = x - (Lq - 1)
  const long long n = Lq + Lk - 1;
  if (x >= n) return;
  const int h = blockIdx.z % H, b = blockIdx.z / H;
  const long long d = x - (Lq - 1);
  const long long r0 = (long long)blockIdx.y * rows;
  const long long i0 = max(r0, -d), i1 = min(min(r0 + rows, Lq), Lk - d);
  const T* p = dbias + b * sb + h * sh + d;
  float s = 0.f;
#pragma unroll 8
  for (long long i = i0; i < i1; ++i) s += to_f(p[i * si + i]);
  part[((long long)blockIdx.y * gridDim.z + blockIdx.z) * n + x] = s;
}

__global__ void relbias_join_kernel(const float* __restrict__ part, int chunks, int B, int H, long long n,
                                    double* __restrict__ sums) {
  const long long x = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int h = blockIdx.y;
  if (x >= n) return;
  double s = 0.0;
  for (int c = 0; c < chunks; ++c)
    for (int b = 0; b < B; ++b) s += part[(((long long)c * B + b) * H + h) * n + x];
  sums[h * n + x] = s;
}

constexpr int kBwdRows = 256;

template <typename T>
void fwd_t(int H, int64_t Lq, int64_t Lk, int64_t q_off, const void* table, const BucketRule& rule, void* out,
           cudaStream_t st) {
  const dim3 grid((unsigned)((Lk + 255) / 256), (unsigned)((Lq + kRows - 1) / kRows), H);
  relbias_fwd_kernel<T><<<grid, 256, 0, st>>>((const T*)table, H, Lq, Lk, q_off, rule, (T*)out);
}
template <typename T>
void bwd_t(int B, int H, int64_t Lq, int64_t Lk, const int64_t* s, const void* dbias, float* part, cudaStream_t st) {
  const dim3 grid((unsigned)((Lq + Lk - 1 + 255) / 256), (unsigned)((Lq + kBwdRows - 1) / kBwdRows), B * H);
  relbias_bwd_kernel<T><<<grid, 256, 0, st>>>((const T*)dbias, B, H, Lq, Lk, s[0], s[1], s[2], kBwdRows, part);
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
  switch (type) {
    case kF32: bwd_t<float>(B, H, Lq, Lk, strides, dbias, part, st); break;
    case kBf16: bwd_t<__nv_bfloat16>(B, H, Lq, Lk, strides, dbias, part, st); break;
    default: bwd_t<__half>(B, H, Lq, Lk, strides, dbias, part, st);
  }
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
  relbias_join_kernel<<<dim3((unsigned)((n + 255) / 256), H), 256, 0, st>>>(part, chunks, B, H, n, sums);
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
  relbias_bucket_sums(type, H, Lq, Lk, q_off, sums, nullptr, rule, dtable, st);
}

}  // namespace rvc
