// Norm of queries and keys for each head and the rotation of their positions,
// in one pass over the data, forward and backward.
//   n = x rsqrt(mean x^2 + eps),  y = n w,  pairs (a, b) of the first R values
//   -> (a c - b s, a s + b c) with (c, s) of the row's position
//   backward: g = the output's gradient rotated back, dw = sum g n,
//   dx = r (g w - n mean(g w n)), r = rsqrt(mean x^2 + eps)
// Bound by memory: every value is read once and written once (backward: two
// reads, one write).  A group of lanes holds one head of one token, four pairs
// to a lane, both members of a pair in the same lane, so the rotation needs no
// exchange; the group walks over the token's heads and keeps the position's
// cosines, sines and the weights in registers meanwhile.  Statistics and the
// weight gradients are held in 32 bits, the latter joined over the blocks in
// 64 bits in a fixed order.
#include "norm_rope.cuh"
#include "context.cuh"

#include <algorithm>

namespace rvc {

namespace {

constexpr int kThreads = 256;

template <typename T> struct Raw4;  // four consecutive values as they lie in memory
template <> struct Raw4<float> { using V = float4; };
template <> struct Raw4<__nv_bfloat16> { using V = uint2; };
template <> struct Raw4<__half> { using V = uint2; };

template <typename T> __device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  const typename Raw4<T>::V r = *reinterpret_cast<const typename Raw4<T>::V*>(p);
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f(e[i]);
}
template <typename T> __device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  typename Raw4<T>::V r;
  T* e = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f<T>(v[i]);
  *reinterpret_cast<typename Raw4<T>::V*>(p) = r;
}

// The four pairs of a lane.  VEC: pairs 4 lane .. 4 lane + 3, read as two runs
// of four values; otherwise pairs lane, lane + 32, ... read one by one.
template <bool VEC>
struct Slots {
  int first[4], second[4];  // element of either member; -1 = no pair
  int pair[4];              // rotated pair, or -1
  bool inter;               // VEC: the runs hold the pairs interleaved
  __device__ Slots(const RopeArgs& a, int lane) {
    inter = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = VEC ? 4 * lane + i : lane + 32 * i;
      const int half = a.R / 2;
      pair[i] = p < half ? p : -1;
      if (p >= a.D / 2) {
        first[i] = second[i] = -1;
      } else if (p < half) {
        first[i] = a.interleaved ? 2 * p : p;
        second[i] = a.interleaved ? 2 * p + 1 : p + half;
      } else {
        first[i] = a.R + (p - half);
        second[i] = first[i] + (a.D - a.R) / 2;
      }
    }
    if (VEC) inter = a.interleaved && pair[0] >= 0;
  }
  template <typename T> __device__ __forceinline__ void load(const T* x, float (&u)[4], float (&v)[4]) const {
    if constexpr (VEC) {
      if (first[0] < 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = v[i] = 0.f;
      } else if (inter) {
        float s[4], e[4];
        load4(x + first[0], s);
        load4(x + first[0] + 4, e);
        u[0] = s[0], v[0] = s[1], u[1] = s[2], v[1] = s[3];
        u[2] = e[0], v[2] = e[1], u[3] = e[2], v[3] = e[3];
      } else {
        load4(x + first[0], u);
        load4(x + second[0], v);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[i] = first[i] >= 0 ? to_f(x[first[i]]) : 0.f;
        v[i] = first[i] >= 0 ? to_f(x[second[i]]) : 0.f;
      }
    }
  }
  template <typename T> __device__ __forceinline__ void store(T* y, const float (&u)[4], const float (&v)[4]) const {
    if constexpr (VEC) {
      if (first[0] < 0) return;
      if (inter) {
        const float s[4] = {u[0], v[0], u[1], v[1]}, e[4] = {u[2], v[2], u[3], v[3]};
        store4(y + first[0], s);
        store4(y + first[0] + 4, e);
      } else {
        store4(y + first[0], u);
        store4(y + second[0], v);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (first[i] >= 0) {
          y[first[i]] = from_f<T>(u[i]);
          y[second[i]] = from_f<T>(v[i]);
        }
    }
  }
  __device__ __forceinline__ void weights(const void* w, int wtype, float (&u)[4], float (&v)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = v[i] = 0.f;
      if (first[i] < 0) continue;
      if (wtype == kF32) {
        u[i] = static_cast<const float*>(w)[first[i]], v[i] = static_cast<const float*>(w)[second[i]];
      } else if (wtype == kBf16) {
        u[i] = to_f(static_cast<const __nv_bfloat16*>(w)[first[i]]);
        v[i] = to_f(static_cast<const __nv_bfloat16*>(w)[second[i]]);
      } else {
        u[i] = to_f(static_cast<const __half*>(w)[first[i]]), v[i] = to_f(static_cast<const __half*>(w)[second[i]]);
      }
    }
  }
  // Cosine and sine of the lane's pairs at table row `pos`; a row outside the
  // table reads nothing and gives NaN.
  __device__ __forceinline__ void angles(const RopeArgs& a, long long pos, float (&c)[4], float (&s)[4]) const {
    const bool in = pos >= 0 && pos < a.P;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = 1.f, s[i] = 0.f;
      if (pair[i] < 0) continue;
      c[i] = in ? __ldg(a.cos + pos * (a.R / 2) + pair[i]) : __int_as_float(0x7fffffff);
      s[i] = in ? __ldg(a.sin + pos * (a.R / 2) + pair[i]) : __int_as_float(0x7fffffff);
    }
  }
};

template <int LANES> __device__ __forceinline__ float group_sum(float s) {
#pragma unroll
  for (int x = LANES / 2; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
  return s;
}

__device__ __forceinline__ long long position(const RopeArgs& a, int b, int l) {
  if (!a.pos) return l;
  const int64_t at = b * a.pos_b + l * a.pos_l;
  return a.pos64 ? static_cast<const long long*>(a.pos)[at] : (long long)static_cast<const int*>(a.pos)[at];
}

template <typename T, bool VEC, int LANES>
__global__ void __launch_bounds__(kThreads) rope_fwd_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int U = 4;
  const int lane = threadIdx.x % LANES;
  const int H = a.Hq + a.Hk, nhb = (H + a.head_block - 1) / a.head_block;
  const long long items = (long long)a.B * a.L * nhb;
  const Slots<VEC> sl(a, lane);
  // groups that have no item keep step with their warp (shuffles)
  const long long step = (long long)gridDim.x * (kThreads / LANES);
  const long long first = (long long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const long long lead = first - (threadIdx.x % 32) / LANES;
  float wq[2][4], wk[2][4];
  sl.weights(a.wq, a.wtype, wq[0], wq[1]);
  sl.weights(a.wk, a.wtype, wk[0], wk[1]);
  for (long long base = lead, it = first; base < items; base += step, it += step) {
    const bool on = it < items;
    const long long item = on ? it : items - 1;
    const long long tok = item / nhb;
    const int hb = (int)(item % nhb), b = (int)(tok / a.L), l = (int)(tok % a.L);
    float c[4], s[4];
    sl.angles(a, position(a, b, l), c, s);
    const int h1 = min(H, (hb + 1) * a.head_block);
    // the same trip count for every group of the warp
    for (int x = 0; x < a.head_block; x += U) {
      float u[U][4], v[U][4];
#pragma unroll
      for (int y = 0; y < U; ++y) {
        const int h = min(hb * a.head_block + x + y, h1 - 1);
        const T* src = h < a.Hq ? static_cast<const T*>(a.q) + b * a.qs[0] + l * a.qs[1] + h * a.qs[2]
                                : static_cast<const T*>(a.k) + b * a.ks[0] + l * a.ks[1] + (h - a.Hq) * a.ks[2];
        sl.load(src, u[y], v[y]);
      }
#pragma unroll
      for (int y = 0; y < U; ++y) {
        const int h = hb * a.head_block + x + y;
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = fmaf(u[y][i], u[y][i], fmaf(v[y][i], v[y][i], ss));
        ss = group_sum<LANES>(ss);
        const float r = rsqrtf(ss / (float)a.D + a.eps);
        if (on && x + y < a.head_block && h < h1) {
          const bool isq = h < a.Hq;
          float p[4], q[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = u[y][i] * r * (isq ? wq[0][i] : wk[0][i]), f = v[y][i] * r * (isq ? wq[1][i] : wk[1][i]);
            p[i] = e * c[i] - f * s[i];
            q[i] = e * s[i] + f * c[i];
          }
          T* dst = isq ? static_cast<T*>(a.oq) + (tok * a.Hq + h) * a.D : static_cast<T*>(a.ok) + (tok * a.Hk + h - a.Hq) * a.D;
          sl.store(dst, p, q);
        }
      }
    }
  }
}

template <typename T, bool VEC, int LANES>
__global__ void __launch_bounds__(kThreads) rope_bwd_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int U = 2;
  extern __shared__ float red[];  // [groups][D]
  const int lane = threadIdx.x % LANES;
  const int H = a.Hq + a.Hk, nhb = (H + a.head_block - 1) / a.head_block;
  const long long items = (long long)a.B * a.L * nhb;
  const Slots<VEC> sl(a, lane);
  const long long step = (long long)gridDim.x * (kThreads / LANES);
  const long long first = (long long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const long long lead = first - (threadIdx.x % 32) / LANES;
  float wq[2][4], wk[2][4], aq[2][4], ak[2][4];
  sl.weights(a.wq, a.wtype, wq[0], wq[1]);
  sl.weights(a.wk, a.wtype, wk[0], wk[1]);
#pragma unroll
  for (int i = 0; i < 4; ++i) aq[0][i] = aq[1][i] = ak[0][i] = ak[1][i] = 0.f;
  for (long long base = lead, it = first; base < items; base += step, it += step) {
    const bool on = it < items;
    const long long item = on ? it : items - 1;
    const long long tok = item / nhb;
    const int hb = (int)(item % nhb), b = (int)(tok / a.L), l = (int)(tok % a.L);
    float c[4], s[4];
    sl.angles(a, position(a, b, l), c, s);
    const int h1 = min(H, (hb + 1) * a.head_block);
    for (int x = 0; x < a.head_block; x += U) {
      float u[U][4], v[U][4], p[U][4], q[U][4];
#pragma unroll
      for (int y = 0; y < U; ++y) {
        const int h = min(hb * a.head_block + x + y, h1 - 1);
        const bool isq = h < a.Hq;
        const T* src = isq ? static_cast<const T*>(a.q) + b * a.qs[0] + l * a.qs[1] + h * a.qs[2]
                           : static_cast<const T*>(a.k) + b * a.ks[0] + l * a.ks[1] + (h - a.Hq) * a.ks[2];
        const T* grd = isq ? static_cast<const T*>(a.gq) + b * a.gqs[0] + l * a.gqs[1] + h * a.gqs[2]
                           : static_cast<const T*>(a.gk) + b * a.gks[0] + l * a.gks[1] + (h - a.Hq) * a.gks[2];
        sl.load(src, u[y], v[y]);
        sl.load(grd, p[y], q[y]);
      }
#pragma unroll
      for (int y = 0; y < U; ++y) {
        const int h = hb * a.head_block + x + y;
        const bool live = on && x + y < a.head_block && h < h1, isq = h < a.Hq;
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = fmaf(u[y][i], u[y][i], fmaf(v[y][i], v[y][i], ss));
        const float r = rsqrtf(group_sum<LANES>(ss) / (float)a.D + a.eps);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = p[y][i] * c[i] + q[y][i] * s[i], f = q[y][i] * c[i] - p[y][i] * s[i];
          u[y][i] *= r;
          v[y][i] *= r;
          if (live && isq) {
            aq[0][i] = fmaf(e, u[y][i], aq[0][i]);
            aq[1][i] = fmaf(f, v[y][i], aq[1][i]);
          } else if (live) {
            ak[0][i] = fmaf(e, u[y][i], ak[0][i]);
            ak[1][i] = fmaf(f, v[y][i], ak[1][i]);
          }
          p[y][i] = e * (isq ? wq[0][i] : wk[0][i]);
          q[y][i] = f * (isq ? wq[1][i] : wk[1][i]);
          dot = fmaf(p[y][i], u[y][i], fmaf(q[y][i], v[y][i], dot));
        }
        dot = group_sum<LANES>(dot) / (float)a.D;
        if (live) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[y][i] = r * (p[y][i] - u[y][i] * dot);
            q[y][i] = r * (q[y][i] - v[y][i] * dot);
          }
          T* dst = isq ? static_cast<T*>(a.oq) + (tok * a.Hq + h) * a.D : static_cast<T*>(a.ok) + (tok * a.Hk + h - a.Hq) * a.D;
          sl.store(dst, p[y], q[y]);
        }
      }
    }
  }
  // this block's part of the weight gradients, groups in order
  const int grp = threadIdx.x / LANES;
  constexpr int NG = kThreads / LANES;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (sl.first[i] >= 0) {
        red[grp * a.D + sl.first[i]] = w ? ak[0][i] : aq[0][i];
        red[grp * a.D + sl.second[i]] = w ? ak[1][i] : aq[1][i];
      }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += kThreads) {
      float t = 0.f;
      for (int n = 0; n < NG; ++n) t += red[n * a.D + d];
      a.part[((long long)blockIdx.x * 2 + w) * a.D + d] = t;
    }
  }
}

// dw[d] = sum over the blocks: one warp per value, in 64 bits.
__global__ void rope_dw_kernel(const float* __restrict__ part, int blocks, int D, int wtype, void* dwq, void* dwk) {
  const int e = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (e >= 2 * D) return;
  double s = 0.0;
  for (int b = lane; b < blocks; b += 32) s += part[(long long)b * 2 * D + e];
#pragma unroll
  for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
  if (lane) return;
  void* dst = e < D ? dwq : dwk;
  if (!dst) return;  // no keys
  const int d = e % D;
  if (wtype == kF32) static_cast<float*>(dst)[d] = (float)s;
  else if (wtype == kBf16) static_cast<__nv_bfloat16*>(dst)[d] = __float2bfloat16_rn((float)s);
  else static_cast<__half*>(dst)[d] = __float2half_rn((float)s);
}

bool run4(const RopeArgs& a, const void* p, const int64_t* s) {
  const int64_t e = 4 * type_size(a.type);
  return reinterpret_cast<uintptr_t>(p) % e == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
}

// Runs of four: both halves of the rotated and of the plain values come in fours.
bool vec_ok(const RopeArgs& a, bool backward) {
  return a.R % 8 == 0 && a.D % 8 == 0 && run4(a, a.q, a.qs) && (a.Hk == 0 || run4(a, a.k, a.ks)) &&
         (!backward || (run4(a, a.gq, a.gqs) && (a.Hk == 0 || run4(a, a.gk, a.gks))));
}

int lanes_of(const RopeArgs& a, bool vec) {
  int n = 32;
  if (vec)
    while (n / 2 * 8 >= a.D && n > 4) n /= 2;
  return n;
}

// Heads of one item: all of a token's where the tokens alone fill the GPU, else
// fewer, so that the groups are many (the angles are then read again).
int head_block(const RopeArgs& a, int lanes, int sms) {
  const int H = a.Hq + a.Hk;
  int hb = H;
  while (hb > 1 && (long long)a.B * a.L * ((H + hb - 1) / hb) * lanes < (long long)sms * 1024) hb = (hb + 1) / 2;
  return hb;
}

int blocks_of(const RopeArgs& a, int lanes, int hb, int per_sm, int sms) {
  const int H = a.Hq + a.Hk;
  const long long items = (long long)a.B * a.L * ((H + hb - 1) / hb);
  return (int)std::min<long long>((items + kThreads / lanes - 1) / (kThreads / lanes), (long long)sms * per_sm);
}

constexpr int kBwdPerSm = 4;

template <typename T, bool BWD>
void launch_t(const RopeArgs& a, bool vec, int lanes, int blocks, cudaStream_t st) {
  const size_t smem = BWD ? sizeof(float) * a.D * (kThreads / lanes) : 0;
#define RVC_ROPE(V, N)                                              \
  do {                                                              \
    if constexpr (BWD)                                              \
      rope_bwd_kernel<T, V, N><<<blocks, kThreads, smem, st>>>(a);  \
    else                                                            \
      rope_fwd_kernel<T, V, N><<<blocks, kThreads, 0, st>>>(a);     \
  } while (0)
  if (!vec) RVC_ROPE(false, 32);
  else if (lanes == 4) RVC_ROPE(true, 4);
  else if (lanes == 8) RVC_ROPE(true, 8);
  else if (lanes == 16) RVC_ROPE(true, 16);
  else RVC_ROPE(true, 32);
#undef RVC_ROPE
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
}

template <bool BWD>
void launch(const RopeArgs& a, bool vec, int lanes, int blocks, cudaStream_t st) {
  if (a.type == kF32) launch_t<float, BWD>(a, vec, lanes, blocks, st);
  else if (a.type == kBf16) launch_t<__nv_bfloat16, BWD>(a, vec, lanes, blocks, st);
  else launch_t<__half, BWD>(a, vec, lanes, blocks, st);
}

}  // namespace

int64_t rope_backward_workspace(const RopeArgs& a, int sms) { return (int64_t)sms * kBwdPerSm * 2 * a.D * 4; }

void rope_forward(RopeArgs a, int sms, cudaStream_t st) {
  const bool vec = vec_ok(a, false);
  const int lanes = lanes_of(a, vec);
  a.head_block = head_block(a, lanes, sms);
  launch<false>(a, vec, lanes, blocks_of(a, lanes, a.head_block, 8, sms), st);
}

void rope_backward(RopeArgs a, void* ws, int sms, cudaStream_t st) {
  const bool vec = vec_ok(a, true);
  const int lanes = lanes_of(a, vec);
  a.head_block = head_block(a, lanes, sms);
  a.part = static_cast<float*>(ws);
  const int blocks = blocks_of(a, lanes, a.head_block, kBwdPerSm, sms);
  launch<true>(a, vec, lanes, blocks, st);
  rope_dw_kernel<<<(2 * a.D + 7) / 8, 256, 0, st>>>(a.part, blocks, a.D, a.wtype, a.dwq, a.dwk);
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
}

}  // namespace rvc
