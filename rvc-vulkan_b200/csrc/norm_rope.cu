// Norm of queries and keys for each head and the rotation of their positions,
// in one pass over the data, forward and backward.
//   n = x rsqrt(mean x^2 + eps),  y = n w,  pairs (a, b) of the first R values
//   -> (a c - b s, a s + b c) with (c, s) of the row's position
//   backward: g = the output's gradient rotated back, dw = sum g n,
//   dx = r (g w - n mean(g w n)), r = rsqrt(mean x^2 + eps)
// Bound by memory: every value is read once and written once (backward: two
// reads, one write).  A group of lanes holds one head of one token, eight pairs
// to a lane in runs of 16 bytes, both members of a pair in the same lane, so the
// rotation needs no exchange and a sum over the head takes three shuffles at 128
// values; the group walks over the token's heads and keeps the position's
// cosines and sines and the weight in registers meanwhile.  Queries and keys are
// shared out to blocks of their own.  Statistics and the weight gradients are
// held in 32 bits, the latter joined over the blocks in 64 bits in a fixed order.
// Measured: backward of 8 x 4096 tokens, 16 + 4 heads of 128, bf16 (508 MB): 134 us,
// 3.8 TB/s at two blocks to an SM (128 registers, 8 bytes of them spilled; the fp32
// forms spill 76 to 108).  64 tokens: 6 us alone and cold, 17 with the host's part.
#include "norm_rope.cuh"
#include "context.cuh"

#include <algorithm>

namespace rvc {

namespace {

constexpr int kThreads = 256;

// Two fp32 operations to an instruction, each rounded on its own.
__device__ __forceinline__ uint64_t b64(float2 v) { return *reinterpret_cast<uint64_t*>(&v); }
__device__ __forceinline__ float2 f2(uint64_t v) { return *reinterpret_cast<float2*>(&v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(b64(a)), "l"(b64(b)), "l"(b64(c)));
  return f2(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(b64(a)), "l"(b64(b)));
  return f2(r);
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return make_float2(a.x - b.x, a.y - b.y); }
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// Eight consecutive values as they lie in memory.
template <typename T> struct Run8 {
  static constexpr int N = (int)sizeof(T) / 2;  // 16-byte words
  uint4 r[N];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ float get(int i) const { return to_f(reinterpret_cast<const T*>(r)[i]); }
};
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}

// The pairs of a lane.  VEC: pairs 8 lane .. 8 lane + 7, read as two runs of
// eight values; otherwise pairs lane, lane + 32, ... (four of them) one by one.
template <bool VEC>
struct Slots {
  static constexpr int N = VEC ? 8 : 4;
  int one, two;  // VEC: the two runs, -1 = none; otherwise the lane
  int rot;       // VEC: first rotated pair, or -1
  bool inter;    // VEC: the runs hold the pairs interleaved
  int D, R, interleaved;
  __device__ Slots(const RopeArgs& a, int lane) : D(a.D), R(a.R), interleaved(a.interleaved) {
    const int half = R / 2, p = 8 * lane;
    if (!VEC) {
      one = lane, two = 0, rot = 0, inter = false;
      return;
    }
    rot = p < half ? p : -1;
    inter = interleaved && p < half;
    if (p >= D / 2) one = two = -1;
    else if (p < half) one = interleaved ? 2 * p : p, two = interleaved ? 2 * p + 8 : p + half;
    else one = R + (p - half), two = one + (D - R) / 2;
  }
  // element of a member of pair i (not VEC), -1 = no pair
  __device__ __forceinline__ int at(int i, int member) const {
    const int p = one + 32 * i, half = R / 2;
    if (p >= D / 2) return -1;
    if (p < half) return interleaved ? 2 * p + member : p + member * half;
    return R + (p - half) + member * ((D - R) / 2);
  }
  template <typename T> __device__ __forceinline__ void fetch(const T* x, Run8<T>& a, Run8<T>& b) const {
    if (VEC && one >= 0) {
      a.load(x + one);
      b.load(x + two);
    }
  }
  template <typename T>
  __device__ __forceinline__ void unpack(const T* x, const Run8<T>& a, const Run8<T>& b, float2 (&u)[N / 2],
                                         float2 (&v)[N / 2]) const {
    if constexpr (VEC) {
      if (inter) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          u[i] = make_float2(a.get(4 * i), a.get(4 * i + 2)), v[i] = make_float2(a.get(4 * i + 1), a.get(4 * i + 3));
          u[2 + i] = make_float2(b.get(4 * i), b.get(4 * i + 2));
          v[2 + i] = make_float2(b.get(4 * i + 1), b.get(4 * i + 3));
        }
      } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
          u[i] = make_float2(a.get(2 * i), a.get(2 * i + 1)), v[i] = make_float2(b.get(2 * i), b.get(2 * i + 1));
      }
      if (one < 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) u[i] = v[i] = both(0.f);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float e = at(i, 0) >= 0 ? to_f(x[at(i, 0)]) : 0.f, f = at(i, 0) >= 0 ? to_f(x[at(i, 1)]) : 0.f;
        if (i & 1) u[i / 2].y = e, v[i / 2].y = f;
        else u[i / 2].x = e, v[i / 2].x = f;
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* y, const float2 (&u)[N / 2], const float2 (&v)[N / 2]) const {
    if constexpr (VEC) {
      if (one < 0) return;
      if (inter) {
        const float s[8] = {u[0].x, v[0].x, u[0].y, v[0].y, u[1].x, v[1].x, u[1].y, v[1].y};
        const float e[8] = {u[2].x, v[2].x, u[2].y, v[2].y, u[3].x, v[3].x, u[3].y, v[3].y};
        store8(y + one, s);
        store8(y + two, e);
      } else {
        const float s[8] = {u[0].x, u[0].y, u[1].x, u[1].y, u[2].x, u[2].y, u[3].x, u[3].y};
        const float e[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
        store8(y + one, s);
        store8(y + two, e);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (at(i, 0) >= 0) {
          y[at(i, 0)] = from_f<T>(i & 1 ? u[i / 2].y : u[i / 2].x);
          y[at(i, 1)] = from_f<T>(i & 1 ? v[i / 2].y : v[i / 2].x);
        }
    }
  }
  __device__ __forceinline__ int element(int i, int member) const {
    if constexpr (VEC) {
      if (one < 0) return -1;
      if (inter) return one + 2 * i + member;
      return (member ? two : one) + i;
    } else {
      return at(i, member);
    }
  }
  __device__ __forceinline__ void weights(const void* w, int wtype, float2 (&u)[N / 2], float2 (&v)[N / 2]) const {
    const auto get = [&](int e) {
      if (e < 0) return 0.f;
      if (wtype == kF32) return static_cast<const float*>(w)[e];
      return wtype == kBf16 ? to_f(static_cast<const __nv_bfloat16*>(w)[e]) : to_f(static_cast<const __half*>(w)[e]);
    };
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      u[i] = make_float2(get(element(2 * i, 0)), get(element(2 * i + 1, 0)));
      v[i] = make_float2(get(element(2 * i, 1)), get(element(2 * i + 1, 1)));
    }
  }
  // Cosine and sine of the lane's pairs at table row `pos`; a row outside the
  // table reads nothing and gives NaN.
  __device__ __forceinline__ void angles(const RopeArgs& a, long long pos, float2 (&c)[N / 2], float2 (&s)[N / 2]) const {
    const bool in = pos >= 0 && pos < a.P;
    const float none = __int_as_float(0x7fffffff);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) c[i] = both(1.f), s[i] = both(0.f);
    if constexpr (VEC) {
      if (rot < 0) return;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) c[i] = s[i] = both(none);
      if (!in) return;
      const float4* pc = reinterpret_cast<const float4*>(a.cos + pos * (R / 2) + rot);
      const float4* ps = reinterpret_cast<const float4*>(a.sin + pos * (R / 2) + rot);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 x = __ldg(pc + i), y = __ldg(ps + i);
        c[2 * i] = make_float2(x.x, x.y), c[2 * i + 1] = make_float2(x.z, x.w);
        s[2 * i] = make_float2(y.x, y.y), s[2 * i + 1] = make_float2(y.z, y.w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int p = one + 32 * i;
        if (p >= R / 2) continue;
        const float x = in ? __ldg(a.cos + pos * (R / 2) + p) : none, y = in ? __ldg(a.sin + pos * (R / 2) + p) : none;
        if (i & 1) c[i / 2].y = x, s[i / 2].y = y;
        else c[i / 2].x = x, s[i / 2].x = y;
      }
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

// Blocks [0, q_blocks) take the queries, the others the keys.  An item is a
// head block of one token; groups without an item keep step with their warp.
template <typename T, bool VEC, int LANES, bool BWD>
__global__ void __launch_bounds__(kThreads, BWD ? 2 : 3) rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int N = Slots<VEC>::N;
  extern __shared__ float red[];  // backward: [groups][D]
  const int lane = threadIdx.x % LANES;
  const bool isq = (int)blockIdx.x < a.q_blocks;
  const int H = isq ? a.Hq : a.Hk;
  const int block = isq ? blockIdx.x : blockIdx.x - a.q_blocks, blocks = isq ? a.q_blocks : gridDim.x - a.q_blocks;
  const int64_t sb = isq ? a.qs[0] : a.ks[0], sl_ = isq ? a.qs[1] : a.ks[1], sh = isq ? a.qs[2] : a.ks[2];
  const int64_t gb = isq ? a.gqs[0] : a.gks[0], gl = isq ? a.gqs[1] : a.gks[1], gh = isq ? a.gqs[2] : a.gks[2];
  const T* x = static_cast<const T*>(isq ? a.q : a.k);
  const T* gr = static_cast<const T*>(isq ? a.gq : a.gk);
  T* y = static_cast<T*>(isq ? a.oq : a.ok);
  const int hb = min(a.head_block, H), nhb = (H + hb - 1) / hb;
  const long long items = (long long)a.B * a.L * nhb;
  const Slots<VEC> sl(a, lane);
  const long long step = (long long)blocks * (kThreads / LANES);
  const long long first = (long long)block * (kThreads / LANES) + threadIdx.x / LANES;
  const long long lead = first - (threadIdx.x % 32) / LANES;
  const float inv_d = 1.f / (float)a.D;
  float2 w[2][N / 2], acc[2][BWD ? N / 2 : 1];
  sl.weights(isq ? a.wq : a.wk, a.wtype, w[0], w[1]);
  if (BWD)
#pragma unroll
    for (int i = 0; i < (BWD ? N / 2 : 1); ++i) acc[0][i] = acc[1][i] = both(0.f);
  for (long long base = lead, it = first; base < items; base += step, it += step) {
    const bool on = it < items;
    const long long item = on ? it : items - 1;
    const long long tok = item / nhb;
    const int h0 = (int)(item % nhb) * hb, b = (int)(tok / a.L), l = (int)(tok % a.L);
    float2 c[N / 2], s[N / 2];
    sl.angles(a, position(a, b, l), c, s);
    const T* xp = x + b * sb + l * sl_;
    const T* gp = gr + b * gb + l * gl;
    T* yp = y + tok * H * a.D;
    auto one = [&](int h, bool live, float2 (&u)[N / 2], float2 (&v)[N / 2], float2 (&p)[N / 2], float2 (&q)[N / 2]) {
      float2 ss = both(0.f);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) ss = fma2(u[i], u[i], fma2(v[i], v[i], ss));
      const float r = rsqrtf(fmaf(group_sum<LANES>(ss.x + ss.y), inv_d, a.eps));
      const float2 r2 = both(r);
      if constexpr (!BWD) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 e = mul2(mul2(u[i], r2), w[0][i]), f = mul2(mul2(v[i], r2), w[1][i]);
          u[i] = sub2(mul2(e, c[i]), mul2(f, s[i]));
          v[i] = fma2(e, s[i], mul2(f, c[i]));
        }
        if (live) sl.store(yp + (int64_t)h * a.D, u, v);
      } else {
        if (!live) {  // a head that another group or nobody has
#pragma unroll
          for (int i = 0; i < N / 2; ++i) p[i] = q[i] = u[i] = v[i] = both(0.f);
        }
        float2 dot = both(0.f);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 e = fma2(p[i], c[i], mul2(q[i], s[i])), f = sub2(mul2(q[i], c[i]), mul2(p[i], s[i]));
          u[i] = mul2(u[i], r2);
          v[i] = mul2(v[i], r2);
          acc[0][i] = fma2(e, u[i], acc[0][i]);
          acc[1][i] = fma2(f, v[i], acc[1][i]);
          p[i] = mul2(e, w[0][i]);
          q[i] = mul2(f, w[1][i]);
          dot = fma2(p[i], u[i], fma2(q[i], v[i], dot));
        }
        const float2 k = both(-group_sum<LANES>(dot.x + dot.y) * inv_d);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          p[i] = mul2(r2, fma2(u[i], k, p[i]));
          q[i] = mul2(r2, fma2(v[i], k, q[i]));
        }
        if (live) sl.store(yp + (int64_t)h * a.D, p, q);
      }
    };
    // the next head's values are on their way while one is worked on
    Run8<T> x0, x1, g0, g1;
    sl.fetch(xp + h0 * sh, x0, x1);
    if (BWD) sl.fetch(gp + h0 * gh, g0, g1);
    for (int z = 0; z < hb; ++z) {
      const int h = min(h0 + z, H - 1), next = min(h0 + z + 1, H - 1);
      float2 u[N / 2], v[N / 2], p[N / 2], q[N / 2];
      sl.unpack(xp + h * sh, x0, x1, u, v);
      if (BWD) sl.unpack(gp + h * gh, g0, g1, p, q);
      if (z + 1 < hb) {
        sl.fetch(xp + next * sh, x0, x1);
        if (BWD) sl.fetch(gp + next * gh, g0, g1);
      }
      one(h, on && h0 + z < H, u, v, p, q);
    }
  }
  if constexpr (BWD) {  // this block's part of the weight gradient, groups in order
    const int grp = threadIdx.x / LANES;
    constexpr int NG = kThreads / LANES;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (sl.element(i, 0) >= 0) {
        red[grp * a.D + sl.element(i, 0)] = i & 1 ? acc[0][i / 2].y : acc[0][i / 2].x;
        red[grp * a.D + sl.element(i, 1)] = i & 1 ? acc[1][i / 2].y : acc[1][i / 2].x;
      }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += kThreads) {
      float t = 0.f;
      for (int n = 0; n < NG; ++n) t += red[n * a.D + d];
      a.part[(long long)blockIdx.x * a.D + d] = t;
    }
  }
}

// dw[d] = sum over the blocks of a side: one warp per value, in 64 bits.
__global__ void rope_dw_kernel(const float* __restrict__ part, int q_blocks, int blocks, int D, int wtype, void* dwq,
                               void* dwk) {
  const int e = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (e >= 2 * D) return;
  void* dst = e < D ? dwq : dwk;
  if (!dst) return;  // no keys
  const int d = e % D, lo = e < D ? 0 : q_blocks, hi = e < D ? q_blocks : blocks;
  double s = 0.0;
#pragma unroll 4
  for (int b = lo + lane; b < hi; b += 32) s += part[(long long)b * D + d];
#pragma unroll
  for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
  if (lane) return;
  if (wtype == kF32) static_cast<float*>(dst)[d] = (float)s;
  else if (wtype == kBf16) static_cast<__nv_bfloat16*>(dst)[d] = __float2bfloat16_rn((float)s);
  else static_cast<__half*>(dst)[d] = __float2half_rn((float)s);
}

bool run8(const RopeArgs& a, const void* p, const int64_t* s) {
  const int64_t e = 16 / type_size(a.type);
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % e == 0 && s[1] % e == 0 && s[2] % e == 0;
}

// Runs of eight: both halves of the rotated and of the plain values come in
// eights, and the rows of the tables start on 16 bytes.
bool vec_ok(const RopeArgs& a, bool backward) {
  const auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  return a.R % 16 == 0 && a.D % 16 == 0 && al(a.cos) && al(a.sin) && al(a.oq) && al(a.ok) && run8(a, a.q, a.qs) &&
         (a.Hk == 0 || run8(a, a.k, a.ks)) &&
         (!backward || (run8(a, a.gq, a.gqs) && (a.Hk == 0 || run8(a, a.gk, a.gks))));
}

int lanes_of(const RopeArgs& a, bool vec) {
  if (!vec) return 32;
  int n = 2;
  while (n * 16 < a.D) n *= 2;
  return n;
}

// Heads of one item: all of a token's where the tokens alone fill the GPU, else
// fewer, so that the groups are many (the angles are then read again).  Blocks
// are shared out by the heads of either side.
int share_out(RopeArgs& a, int lanes, int per_sm, int sms) {
  const int H = std::max(a.Hq, a.Hk);
  int hb = H;
  while (hb > 1 && (long long)a.B * a.L * ((H + hb - 1) / hb) * lanes < (long long)sms * 1024) hb = (hb + 1) / 2;
  a.head_block = hb;
  const int groups = kThreads / lanes;
  const auto need = [&](int h) {
    const int x = std::min(hb, h);
    return h == 0 ? 0ll : ((long long)a.B * a.L * ((h + x - 1) / x) + groups - 1) / groups;
  };
  const long long most = (long long)sms * per_sm, nq = need(a.Hq), nk = need(a.Hk);
  const long long kb = std::min(nk, std::max(nk > 0 ? 1ll : 0ll, most * a.Hk / (a.Hq + a.Hk)));
  a.q_blocks = (int)std::min(nq, most - kb);
  return a.q_blocks + (int)kb;
}

constexpr int kFwdPerSm = 6, kBwdPerSm = 4;

template <typename T, bool BWD>
void launch_t(const RopeArgs& a, bool vec, int lanes, int blocks, cudaStream_t st) {
  const size_t smem = BWD ? sizeof(float) * a.D * (kThreads / lanes) : 0;
  if (!vec) rope_kernel<T, false, 32, BWD><<<blocks, kThreads, smem, st>>>(a);
  else if (lanes == 2) rope_kernel<T, true, 2, BWD><<<blocks, kThreads, smem, st>>>(a);
  else if (lanes == 4) rope_kernel<T, true, 4, BWD><<<blocks, kThreads, smem, st>>>(a);
  else if (lanes == 8) rope_kernel<T, true, 8, BWD><<<blocks, kThreads, smem, st>>>(a);
  else rope_kernel<T, true, 16, BWD><<<blocks, kThreads, smem, st>>>(a);
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

int64_t rope_backward_workspace(const RopeArgs& a, int sms) { return (int64_t)sms * kBwdPerSm * a.D * 4; }

void rope_forward(RopeArgs a, int sms, cudaStream_t st) {
  const bool vec = vec_ok(a, false);
  const int lanes = lanes_of(a, vec);
  launch<false>(a, vec, lanes, share_out(a, lanes, kFwdPerSm, sms), st);
}

void rope_backward(RopeArgs a, void* ws, int sms, cudaStream_t st) {
  const bool vec = vec_ok(a, true);
  const int lanes = lanes_of(a, vec);
  a.part = static_cast<float*>(ws);
  const int blocks = share_out(a, lanes, kBwdPerSm, sms);
  launch<true>(a, vec, lanes, blocks, st);
  rope_dw_kernel<<<(2 * a.D + 7) / 8, 256, 0, st>>>(a.part, a.q_blocks, blocks, a.D, a.wtype, a.dwq, a.dwk);
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
}

}  // namespace rvc
