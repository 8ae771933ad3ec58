// Attention and its gradient on warp-level matrix instructions: the kernels
// that take every type, stride, length and head dimension (<= 128), and the
// fast ones where rows are few (one new token against long states) or the
// type is fp32.
//
// 16-bit inputs go through m16n8k16 with fp32 accumulators.  fp32 inputs are
// split into three bf16 parts (24 bits) when they are staged, and a product is
// the six of their products that are above 2^-24, smallest first; the tensor
// cores cut their sums off instead of rounding them, so every 16 values' worth
// is formed in an accumulator of its own and added in fp32 with rounding (a
// chain in one accumulator was off by 6e-6 over 1500 keys).  Where rows are few
// and the reading of the states counts, fp32 stays as it is in shared memory and
// goes through m16n8k8 TF32 as hi + lo with three products (2^-22).  Weights P
// and dS enter their second product rounded to the inputs' type (16-bit inputs:
// the rounding of the output itself) or split the same way (fp32).
//
// Layout: a block stages a tile of keys and values in shared memory (16-bit
// types by cp.async in two stages, fp32 through registers) with 16 bytes of
// padding per row, so that both the row-wise and the transposed fragment reads
// are free of bank conflicts.  Dead keys (past the length or masked out) are
// staged as zeros: whatever the caller's buffer holds there, NaN included, never
// meets a product.
//
// Measured: one row, 12 heads, 499 keys of 64, bf16: 8.8 us alone and cold (the
// call is 17 to 18, its host part); 32 x 4 key heads of 128, ragged to 8192 keys:
// 89 to 95 us (3.6 TB/s; 580 instructions per 16 keys of a warp); fp32 gradients of
// 4 x 2 x 1000 x 1000 x 96 with a bias: 417 us (tensor pipe busy 23 and 30 % of the
// two kernels: eight warps to an SM, which load, split and multiply in turn).
#include "attn_common.cuh"
#include "context.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <atomic>

namespace rvc {

namespace {

constexpr int kT = 128;   // threads of a forward block (4 warps)
constexpr int kBN = 64;   // keys per tile (16-bit types)
constexpr int kBM = 64;   // query rows per block (4 warps x 16) where rows are many

// ------------------------------------------------------------ fragment helpers
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo: hi rounded to TF32's 11 bits on the integer form (half away from
// zero; a carry runs into the exponent as it should, infinities and NaN stay
// themselves or become NaN), the rest exact, and cut to 11 bits by the tensor
// core, which reads no more.  The conversion instruction runs at a fraction of
// this rate.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
struct Split4 {
  uint32_t hi[4], lo[4];
};
__device__ __forceinline__ void mma8x3(float (&c)[4], const Split4& a, float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split_tf32(b0, h0, l0);
  split_tf32(b1, h1, l1);
  // The tensor cores cut their sums off instead of rounding them: a chain of
  // products in one accumulator drifts (6e-6 over 1500 keys).  Each product of
  // eight values is formed alone and added in fp32 with rounding.
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  mma8(t, a.lo, h0, h1);
  mma8(t, a.hi, l0, l1);
  mma8(t, a.hi, h0, h1);
#pragma unroll
  for (int x = 0; x < 4; ++x) c[x] += t[x];
}
__device__ __forceinline__ float lds_f(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T> constexpr int kParts = sizeof(T) == 4 ? 3 : 1;  // bf16 parts of a value
// Bytes of a staged row (of one part): D 16-bit values and 16 bytes, so rows
// start 4 banks apart.
template <int DP> constexpr int pitch() { return DP * 2 + 16; }
template <typename T, int DP> constexpr int tile_bytes(int rows) { return kParts<T> * rows * pitch<DP>(); }
// Staged rows: the first row of the first part, and the distance of the parts.
struct Rows {
  uint32_t at, part;
};

// x = hi + mid + lo in bf16 for two values at once, each rounded from what is left.
__device__ __forceinline__ void split3(float a, float b, uint32_t (&w)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    w[i] = pack2<__nv_bfloat16>(a, b);
    a -= __uint_as_float(w[i] << 16);
    b -= __uint_as_float(w[i] & 0xffff0000u);
  }
}
// c0, c1 += the six products of three parts each that count, smallest first.
__device__ __forceinline__ void mma_parts(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[3][4],
                                          const uint32_t (&b)[3][4]) {
  constexpr int pa[6] = {2, 1, 0, 1, 0, 0}, pb[6] = {0, 1, 2, 0, 1, 0};
  float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    mma16(t0, a[pa[i]], b[pb[i]][0], b[pb[i]][1], __nv_bfloat16());
    mma16(t1, a[pa[i]], b[pb[i]][2], b[pb[i]][3], __nv_bfloat16());
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) c0[x] += t0[x], c1[x] += t1[x];
}

// C[16][8 NT] (+)= A[16][DP] . B[8 NT][DP]^T; A and B staged rows.
template <typename T, int DP, int NT>
__device__ __forceinline__ void mma_abt(float (&c)[NT][4], Rows a, Rows b, int lane) {
  constexpr int P = pitch<DP>(), N = kParts<T>;
  const int mi = lane >> 3, r8 = lane & 7;
  const uint32_t ra = a.at + ((mi & 1) * 8 + r8) * P + (mi >> 1) * 16, rb = b.at + ((mi >> 1) * 8 + r8) * P + (mi & 1) * 16;
#pragma unroll(N == 1 ? DP / 16 : 1)
  for (int kk = 0; kk < DP / 16; ++kk) {
    uint32_t af[N][4];
#pragma unroll
    for (int i = 0; i < N; ++i) ldsm4(af[i], ra + i * a.part + kk * 32);
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t bf[N][4];
#pragma unroll
      for (int i = 0; i < N; ++i) ldsm4(bf[i], rb + i * b.part + n * 8 * P + kk * 32);
      if constexpr (N == 1) {
        mma16(c[n], af[0], bf[0][0], bf[0][1], T());
        mma16(c[n + 1], af[0], bf[0][2], bf[0][3], T());
      } else {
        mma_parts(c[n], c[n + 1], af, bf);
      }
    }
  }
}

// C[16][DP] += A[16][8 NT] . B[8 NT][DP]: A are accumulator fragments (weights),
// B staged rows.
template <typename T, int DP, int NT>
__device__ __forceinline__ void mma_pb(float (&c)[DP / 8][4], const float (&p)[NT][4], Rows b, int lane) {
  constexpr int P = pitch<DP>(), N = kParts<T>;
  const int mi = lane >> 3, r8 = lane & 7;
  const uint32_t rb = b.at + ((mi & 1) * 8 + r8) * P + (mi >> 1) * 16;
#pragma unroll
  for (int n = 0; n < NT; n += 2) {
    uint32_t af[N][4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float u = p[n + (x >> 1)][2 * (x & 1)], v = p[n + (x >> 1)][2 * (x & 1) + 1];
      if constexpr (N == 1) {
        af[0][x] = pack2<T>(u, v);
      } else {
        uint32_t w[3];
        split3(u, v, w);
#pragma unroll
        for (int i = 0; i < 3; ++i) af[i][x] = w[i];
      }
    }
#pragma unroll
    for (int d = 0; d < DP / 8; d += 2) {
      uint32_t bf[N][4];
#pragma unroll
      for (int i = 0; i < N; ++i) ldsm4t(bf[i], rb + i * b.part + n * 8 * P + d * 16);
      if constexpr (N == 1) {
        mma16(c[d], af[0], bf[0][0], bf[0][1], T());
        mma16(c[d + 1], af[0], bf[0][2], bf[0][3], T());
      } else {
        mma_parts(c[d], c[d + 1], af, bf);
      }
    }
  }
}

// Stages `rows` rows into `dst`; row r comes from src(r), a null source is
// staged as zeros.  Columns past D are zeros.
template <typename T, int DP, int THREADS, typename F>
__device__ __forceinline__ void stage_rows(Rows dst, int rows, int D, bool vec, int tid, F src) {
  constexpr int P = pitch<DP>();
  if constexpr (sizeof(T) == 2) {
    if (vec) {
      constexpr int CH = DP / 8;
      for (int e = tid; e < rows * CH; e += THREADS) {
        const int r = e / CH, c = e % CH;
        const T* s = src(r);
        const bool on = s != nullptr && c * 8 < D;
        cp16(dst.at + r * P + c * 16, on ? s + c * 8 : nullptr, on ? 16u : 0u);
      }
    } else {
      for (int e = tid; e < rows * DP; e += THREADS) {
        const int r = e / DP, c = e % DP;
        const T* s = src(r);
        const T v = (s != nullptr && c < D) ? s[c] : from_f<T>(0.f);
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst.at + r * P + c * 2), "h"(*reinterpret_cast<const uint16_t*>(&v))
                     : "memory");
      }
    }
  } else {
    constexpr int CH = DP / 4;
#pragma unroll 4
    for (int e = tid; e < rows * CH; e += THREADS) {
      const int r = e / CH, c = e % CH * 4;
      const T* s = src(r);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s != nullptr) {
        if (vec) {
          if (c < D) v = *reinterpret_cast<const float4*>(s + c);
        } else {
          if (c < D) v.x = s[c];
          if (c + 1 < D) v.y = s[c + 1];
          if (c + 2 < D) v.z = s[c + 2];
          if (c + 3 < D) v.w = s[c + 3];
        }
      }
      uint32_t lo[3], hi[3];
      split3(v.x, v.y, lo);
      split3(v.z, v.w, hi);
#pragma unroll
      for (int i = 0; i < 3; ++i) ptx::sts64(dst.at + i * dst.part + r * P + c * 2, lo[i], hi[i]);
    }
  }
}

// ------------------------------------- fp32 as it is, for few rows (TF32 hi + lo)
template <typename T, int DP> constexpr int raw_pitch() { return DP * (int)sizeof(T) + 16; }

template <int DP>
__device__ __forceinline__ void tf32_abt(float (&c)[2][4], uint32_t a, uint32_t b, int lane) {
  constexpr int P = raw_pitch<float, DP>();
  const int g = lane >> 2, t = lane & 3;
#pragma unroll 2
  for (int kk = 0; kk < DP / 8; ++kk) {
    Split4 af;
    const uint32_t ar = a + g * P + (kk * 8 + t) * 4;
    split_tf32(lds_f(ar), af.hi[0], af.lo[0]);
    split_tf32(lds_f(ar + 8 * P), af.hi[1], af.lo[1]);
    split_tf32(lds_f(ar + 16), af.hi[2], af.lo[2]);
    split_tf32(lds_f(ar + 8 * P + 16), af.hi[3], af.lo[3]);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const uint32_t br = b + (n * 8 + g) * P + (kk * 8 + t) * 4;
      mma8x3(c[n], af, lds_f(br), lds_f(br + 16));
    }
  }
}
// The contraction runs over the columns in the order 2t, 2t + 1, which is the
// accumulators' own, so no value changes lanes.
template <int DP>
__device__ __forceinline__ void tf32_pb(float (&c)[DP / 8][4], const float (&p)[2][4], uint32_t b, int lane) {
  constexpr int P = raw_pitch<float, DP>();
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    Split4 af;
    split_tf32(p[n][0], af.hi[0], af.lo[0]);
    split_tf32(p[n][2], af.hi[1], af.lo[1]);
    split_tf32(p[n][1], af.hi[2], af.lo[2]);
    split_tf32(p[n][3], af.hi[3], af.lo[3]);
    const uint32_t br = b + (n * 8 + 2 * t) * P + g * 4;
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) mma8x3(c[d], af, lds_f(br + d * 32), lds_f(br + P + d * 32));
  }
}

// The A operand held in registers over many calls (16-bit types).
template <typename T, int DP>
struct FragA {
  uint32_t f[DP / 16][4];
  __device__ __forceinline__ void load(uint32_t a, int lane) {
    const int mi = lane >> 3, r8 = lane & 7;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) ldsm4(f[kk], a + ((mi & 1) * 8 + r8) * pitch<DP>() + (kk * 16 + (mi >> 1) * 8) * 2);
  }
  // C[16][16] += A . B[16][DP]^T
  __device__ __forceinline__ void abt(float (&c)[2][4], uint32_t b, int lane) const {
    const int mi = lane >> 3, r8 = lane & 7;
    const uint32_t at = b + ((mi >> 1) * 8 + r8) * pitch<DP>() + (mi & 1) * 16;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      uint32_t bf[4];
      ldsm4(bf, at + kk * 32);
      mma16(c[0], f[kk], bf[0], bf[1], T());
      mma16(c[1], f[kk], bf[2], bf[3], T());
    }
  }
};

// ------------------------------------------------- forward, many query rows
// One block: one KV head of one batch entry, 64 (fp32: 128) rows of the (query head in the
// group, query) plane - every warp has 16 of its own - and the key tiles of one
// split.
// fp32: 128 rows share a staged tile of 32 keys (one stage: two blocks to an SM
// cover each other's loads), as the splitting costs what a warp's products do.
template <typename T> constexpr int kFwdRows = sizeof(T) == 4 ? 128 : kBM;
template <typename T> constexpr int kFwdKeys = sizeof(T) == 4 ? 32 : kBN;
template <typename T> constexpr int kFwdStages = sizeof(T) == 4 ? 1 : 2;

template <typename T, int DP>
__global__ void __launch_bounds__(kFwdRows<T> * 2, sizeof(T) == 4 && DP <= 64 ? 2 : 1) attn_mma_fwd_kernel(const __grid_constant__ AttnArgs a, int vec_q, int vec_kv) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int P = pitch<DP>(), BN = kFwdKeys<T>, ST = kFwdStages<T>;
  constexpr int NT = BN / 8, BM = kFwdRows<T>, TH = 2 * BM;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.Hq / a.Hkv;
  const long long rows = (long long)G * a.Lq;
  const unsigned ntile = (unsigned)((rows + BM - 1) / BM);
  const int b = blockIdx.x / ntile / a.Hkv, kh = blockIdx.x / ntile % a.Hkv;
  const long long r0 = (long long)(blockIdx.x % ntile) * BM;
  const uint32_t sm = ptx::smem_u32(smem);
  constexpr uint32_t TB = tile_bytes<T, DP>(BN);
  const Rows sQ = {sm, BM * P};
  const auto kv = [&](int st, int v) { return Rows{sm + (uint32_t)tile_bytes<T, DP>(BM) + (2 * st + v) * TB, BN * P}; };
  const int len = kv_len(a, b);

  // the furthest key that a row of this block may meet
  long long kend = len;
  if (a.causal) {
    const long long last = min(rows, r0 + BM) - 1;
    const long long imax = (r0 / a.Lq != last / a.Lq) ? a.Lq - 1 : last % a.Lq;
    kend = max(0ll, min(kend, imax + a.q_off + 1));
  }
  const int tiles = (int)((kend + BN - 1) / BN);
  const int t0 = (int)((long long)tiles * blockIdx.y / a.nsplit), t1 = (int)((long long)tiles * (blockIdx.y + 1) / a.nsplit);

  const T* qb = static_cast<const T*>(a.q) + (int64_t)b * a.qs[0];
  const T* kb = static_cast<const T*>(a.k) + (int64_t)b * a.ks[0] + (int64_t)kh * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + (int64_t)b * a.vs[0] + (int64_t)kh * a.vs[2];
  const uint8_t* mb = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
  stage_rows<T, DP, TH>(sQ, BM, a.D, vec_q, tid, [&](int r) -> const T* {
    const long long x = r0 + r;
    return x < rows ? qb + (x % a.Lq) * a.qs[1] + (kh * G + x / a.Lq) * a.qs[2] : nullptr;
  });
  auto load = [&](int tile, int st) {
    const int j0 = tile * BN;
    auto alive = [&](int r) { return j0 + r < len && (!mb || mb[(int64_t)(j0 + r) * a.mask_k]); };
    stage_rows<T, DP, TH>(kv(st, 0), BN, a.D, vec_kv, tid,
                      [&](int r) -> const T* { return alive(r) ? kb + (int64_t)(j0 + r) * a.ks[1] : nullptr; });
    stage_rows<T, DP, TH>(kv(st, 1), BN, a.D, vec_kv, tid,
                      [&](int r) -> const T* { return alive(r) ? vb + (int64_t)(j0 + r) * a.vs[1] : nullptr; });
    cp_commit();
  };
  if (ST == 2 && t0 < t1) load(t0, 0);

  // the two rows of this thread
  const int wr = warp * 16;
  long long qi[2];
  const float* bias[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const long long r = min(r0 + wr + g + 8 * x, rows - 1);
    qi[x] = r % a.Lq;
    bias[x] = a.diag ? a.diag + (kh * G + r / a.Lq) * a.diag_ld + a.diag0 - qi[x] : nullptr;
  }
  const float sc = a.scale * kLog2e;
  float o[DP / 8][4];
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x) o[d][x] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  for (int tile = t0; tile < t1; ++tile) {
    const int st = ST == 2 ? (tile - t0) & 1 : 0;
    if (ST == 1) {
      load(tile, 0);
    } else if (tile + 1 < t1) {
      load(tile + 1, st ^ 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[n][x] = 0.f;
    mma_abt<T, DP, NT>(s, Rows{sQ.at + wr * P, sQ.part}, kv(st, 0), lane);
    const int j0 = tile * BN;
    const bool whole = !mb && j0 + BN <= len && (!a.causal || j0 + BN <= min(qi[0], qi[1]) + a.q_off + 1);
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int j = j0 + n * 8 + 2 * t + (x & 1), y = x >> 1;
        float v = s[n][x] * sc;
        if (a.diag && j < a.Lk) v += __ldg(bias[y] + j);
        if (!whole) {
          const bool on = j < len && (!mb || mb[(int64_t)j * a.mask_k]) && (!a.causal || j <= qi[y] + a.q_off);
          v = on ? v : -INFINITY;
        }
        s[n][x] = v;
        mx[y] = fmaxf(mx[y], v);
      }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      mx[y] = fmaxf(mx[y], __shfl_xor_sync(0xffffffffu, mx[y], 1));
      mx[y] = fmaxf(mx[y], __shfl_xor_sync(0xffffffffu, mx[y], 2));
    }
    const float base[2] = {mx[0] == -INFINITY ? 0.f : mx[0], mx[1] == -INFINITY ? 0.f : mx[1]};
    const float f[2] = {exp2_approx(m[0] - base[0]), exp2_approx(m[1] - base[1])};
    l[0] *= f[0];
    l[1] *= f[1];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[n][x] = exp2_approx(s[n][x] - base[x >> 1]);
        l[x >> 1] += s[n][x];
      }
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[d][x] *= f[x >> 1];
    m[0] = mx[0];
    m[1] = mx[1];
    mma_pb<T, DP, NT>(o, s, kv(st, 1), lane);
    __syncthreads();
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
    l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const long long x = r0 + wr + g + 8 * y;
    if (x >= rows) continue;
    const long long i = x % a.Lq, h = kh * G + x / a.Lq;
    const long long row = ((long long)b * a.Hq + h) * a.Lq + i;
    if (a.nsplit > 1) {
      const long long pr = (long long)blockIdx.y * a.B * a.Hq * a.Lq + row;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d)
#pragma unroll
        for (int z = 0; z < 2; ++z)
          if (d * 8 + 2 * t + z < a.D) a.po[pr * a.D + d * 8 + 2 * t + z] = o[d][2 * y + z];
      if (t == 0) {
        a.pml[2 * pr] = m[y];
        a.pml[2 * pr + 1] = l[y];
      }
    } else {
      const float inv = row_inv(l[y]);
      T* dst = static_cast<T*>(a.out) + (((long long)b * a.Lq + i) * a.Hq + h) * a.D;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d)
#pragma unroll
        for (int z = 0; z < 2; ++z)
          if (d * 8 + 2 * t + z < a.D) dst[d * 8 + 2 * t + z] = from_f<T>(o[d][2 * y + z] * inv);
      if (t == 0) a.lse[row] = row_lse(m[y], l[y]);
    }
  }
}

// -------------------------------------------------- forward, few query rows
// At most 16 rows to a KV head (one or a few new tokens): bound by reading the
// keys and values once.  Every warp streams 16 keys at a time through a ring of
// its own in shared memory (cp.async, no barrier between warps) with all rows in
// one fragment; the running maximum is raised, and the output rescaled, only
// when it grows by more than 2^8.  The warps join through shared memory, and
// the splits of a row through the shared memory of their cluster (nsplit <=
// kCluster), so that one launch does it; more splits go through the workspace.
constexpr int kCluster = 8;

// Three stages of 128 16-bit values leave room for two blocks to an SM.
template <typename T, int DP> constexpr int few_stages() { return DP * sizeof(T) > 256 ? 2 : DP * sizeof(T) > 192 ? 3 : 4; }
template <typename T, int DP> constexpr size_t few_smem() {
  return std::max((size_t)4 * few_stages<T, DP>() * 2 * 16 * raw_pitch<T, DP>() + (size_t)16 * raw_pitch<T, DP>(),
                  (size_t)(5 * 16 * (DP + 4) + 5 * 32) * 4);
}

__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile(
      "{\n\t.reg .b32 r;\n\t"
      "mapa.shared::cluster.u32 r, %1, %2;\n\t"
      "ld.shared::cluster.f32 %0, [r];\n\t}"
      : "=f"(v)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, int DP, bool CLUSTER>
__global__ void __launch_bounds__(kT) attn_mma_few_kernel(const __grid_constant__ AttnArgs a, int vec_q, int vec_kv) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int P = raw_pitch<T, DP>(), S = few_stages<T, DP>();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.Hq / a.Hkv, rows = G * a.Lq;  // <= 16
  const int b = blockIdx.x / a.Hkv, kh = blockIdx.x % a.Hkv;
  const uint32_t sm = ptx::smem_u32(smem);
  const uint32_t sQ = sm, ring = sm + 16 * P + warp * S * 2 * 16 * P;
  const int len = kv_len(a, b);
  long long kend = len;
  if (a.causal) kend = max(0ll, min(kend, (long long)a.Lq + a.q_off));
  // steps of 16 keys of this split, dealt to the warps in turn
  const int steps = (int)((kend + 15) / 16);
  const int s0 = (int)((long long)steps * blockIdx.y / a.nsplit), s1 = (int)((long long)steps * (blockIdx.y + 1) / a.nsplit);
  const int n = max(0, s1 - s0 - warp + 3) / 4;  // of this warp: s0 + warp + 4 x

  const T* qb = static_cast<const T*>(a.q) + (int64_t)b * a.qs[0];
  const T* kb = static_cast<const T*>(a.k) + (int64_t)b * a.ks[0] + (int64_t)kh * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + (int64_t)b * a.vs[0] + (int64_t)kh * a.vs[2];
  const uint8_t* mb = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
  constexpr int E = 16 / (int)sizeof(T), CH = DP / E;
  constexpr bool POW2 = (CH & (CH - 1)) == 0;
  // a lane's chunk of a row and its rows: lane / CH, then every 32 / CH
  const int lr = lane / CH, lc = lane % CH;
  const T* kp = kb + (int64_t)((s0 + warp) * 16 + lr) * a.ks[1] + lc * E;
  const T* vp = vb + (int64_t)((s0 + warp) * 16 + lr) * a.vs[1] + lc * E;
  const uint32_t cols = lc * E < a.D ? 16u : 0u;
  auto load = [&](int x) {  // the warp's x-th step; always one group, so that counts agree
    if (x < n) {
      const int j0 = (s0 + warp + 4 * x) * 16;
      const uint32_t dk = ring + (x % S) * 2 * 16 * P, dv = dk + 16 * P;
      if (vec_kv && POW2) {
        const T *k = kp + (int64_t)(64 * x) * a.ks[1], *v = vp + (int64_t)(64 * x) * a.vs[1];
        const bool whole = !mb && j0 + 16 <= len;
        const uint32_t at = dk + lr * P + lc * 16;
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
          const int r = i * (32 / CH);
          uint32_t on = cols;
          if (!whole && !(j0 + lr + r < len && (!mb || mb[(int64_t)(j0 + lr + r) * a.mask_k]))) on = 0;
          cp16(at + r * P, on ? k : kb, on);
          cp16(at + 16 * P + r * P, on ? v : vb, on);
          k += (32 / CH) * a.ks[1];
          v += (32 / CH) * a.vs[1];
        }
      } else if (vec_kv) {
#pragma unroll
        for (int e = lane; e < 16 * CH; e += 32) {
          const int r = e / CH, c = e % CH, j = j0 + r;
          const bool on = c * E < a.D && j < len && (!mb || mb[(int64_t)j * a.mask_k]);
          cp16(dk + r * P + c * 16, on ? kb + (int64_t)j * a.ks[1] + c * E : kb, on ? 16u : 0u);
          cp16(dv + r * P + c * 16, on ? vb + (int64_t)j * a.vs[1] + c * E : vb, on ? 16u : 0u);
        }
      } else {
        for (int e = lane; e < 16 * DP; e += 32) {
          const int r = e / DP, c = e % DP, j = j0 + r;
          const bool on = c < a.D && j < len && (!mb || mb[(int64_t)j * a.mask_k]);
          T* pk = reinterpret_cast<T*>(smem + (dk - sm) + r * P) + c;
          T* pv = reinterpret_cast<T*>(smem + (dv - sm) + r * P) + c;
          *pk = on ? kb[(int64_t)j * a.ks[1] + c] : from_f<T>(0.f);
          *pv = on ? vb[(int64_t)j * a.vs[1] + c] : from_f<T>(0.f);
        }
      }
    }
    cp_commit();
  };
  const auto row_of = [&](int r) { return qb + (int64_t)(r % a.Lq) * a.qs[1] + (int64_t)(kh * G + r / a.Lq) * a.qs[2]; };
  if (vec_q) {
    for (int e = tid; e < 16 * CH; e += kT) {
      const int r = e / CH, c = e % CH;
      const bool on = r < rows && c * E < a.D;
      cp16(sQ + r * P + c * 16, on ? row_of(r) + c * E : qb, on ? 16u : 0u);
    }
  } else {
    for (int e = tid; e < 16 * DP; e += kT) {
      const int r = e / DP, c = e % DP;
      *(reinterpret_cast<T*>(smem + r * P) + c) = r < rows && c < a.D ? row_of(r)[c] : from_f<T>(0.f);
    }
  }
  cp_commit();
#pragma unroll
  for (int x = 0; x < S - 1; ++x) load(x);
  cp_wait<S - 1>();
  __syncthreads();  // Q is there for every warp
  FragA<T, sizeof(T) == 2 ? DP : 16> fq;
  if constexpr (sizeof(T) == 2) fq.load(sQ, lane);

  int qi[2];
  const float* bias[2];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const int r = min(g + 8 * y, rows - 1);
    qi[y] = r % a.Lq;
    bias[y] = a.diag ? a.diag + (kh * G + r / a.Lq) * a.diag_ld + a.diag0 - qi[y] : nullptr;
  }
  const float sc = a.scale * kLog2e;
  float o[DP / 8][4];
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x) o[d][x] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  for (int x = 0; x < n; ++x) {
    load(x + S - 1);
    cp_wait<S - 1>();
    __syncwarp();
    const uint32_t sK = ring + (x % S) * 2 * 16 * P, sV = sK + 16 * P;
    float s[2][4];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int z = 0; z < 4; ++z) s[c][z] = 0.f;
    if constexpr (sizeof(T) == 2) fq.abt(s, sK, lane);
    else tf32_abt<DP>(s, sQ, sK, lane);
    const int j0 = (s0 + warp + 4 * x) * 16;
    const bool whole = !mb && j0 + 16 <= len && (!a.causal || j0 + 16 <= min(qi[0], qi[1]) + a.q_off + 1);
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const int j = j0 + c * 8 + 2 * t + (z & 1), y = z >> 1;
        float v = s[c][z] * sc;
        if (a.diag && j < a.Lk) v += __ldg(bias[y] + j);
        if (!whole) {
          const bool on = j < len && (!mb || mb[(int64_t)j * a.mask_k]) && (!a.causal || j <= qi[y] + a.q_off);
          v = on ? v : -INFINITY;
        }
        s[c][z] = v;
        mx[y] = fmaxf(mx[y], v);
      }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      mx[y] = fmaxf(mx[y], __shfl_xor_sync(0xffffffffu, mx[y], 1));
      mx[y] = fmaxf(mx[y], __shfl_xor_sync(0xffffffffu, mx[y], 2));
    }
    const bool up[2] = {mx[0] > m[0] + 8.f, mx[1] > m[1] + 8.f};
    if (__any_sync(0xffffffffu, up[0] || up[1])) {
      float f[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        f[y] = up[y] ? (m[y] == -INFINITY ? 0.f : exp2_approx(m[y] - mx[y])) : 1.f;
        m[y] = up[y] ? mx[y] : m[y];
        l[y] *= f[y];
      }
#pragma unroll
      for (int d = 0; d < DP / 8; ++d)
#pragma unroll
        for (int z = 0; z < 4; ++z) o[d][z] *= f[z >> 1];
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        s[c][z] = exp2_approx(s[c][z] - base[z >> 1]);
        l[z >> 1] += s[c][z];
      }
    if constexpr (sizeof(T) == 2) mma_pb<T, DP, 2>(o, s, Rows{sV, 0}, lane);
    else tf32_pb<DP>(o, s, sV, lane);
    __syncwarp();  // the ring's place is read before it is written again
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
    l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
  }
  cp_wait<0>();
  __syncthreads();
  // parts of the four warps [4][16][DP + 4], this block's [16][DP + 4] behind, then (max, sum) of each
  constexpr int LD = DP + 4;
  float* part = reinterpret_cast<float*>(smem);
  float* mine = part + 4 * 16 * LD;
  float* ml = mine + 16 * LD;   // [4][16][2]
  float* bml = ml + 4 * 32;     // [16][2]
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int z = 0; z < 4; ++z) part[(warp * 16 + g + 8 * (z >> 1)) * LD + d * 8 + 2 * t + (z & 1)] = o[d][z];
  if (t == 0)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      ml[2 * (warp * 16 + g + 8 * y)] = m[y];
      ml[2 * (warp * 16 + g + 8 * y) + 1] = l[y];
    }
  __syncthreads();
  for (int e = tid; e < rows * DP; e += kT) {
    const int r = e / DP, d = e % DP;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, ml[2 * (w * 16 + r)]);
    float L = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = ml[2 * (w * 16 + r)] == -INFINITY ? 0.f : exp2_approx(ml[2 * (w * 16 + r)] - M);
      L = fmaf(f, ml[2 * (w * 16 + r) + 1], L);
      v = fmaf(f, part[(w * 16 + r) * LD + d], v);
    }
    mine[r * LD + d] = v;
    if (d == 0) {
      bml[2 * r] = M;
      bml[2 * r + 1] = L;
    }
  }
  if (!CLUSTER && a.nsplit > 1) {
    __syncthreads();
    for (int e = tid; e < rows * a.D; e += kT) {
      const int r = e / a.D, d = e % a.D;
      const long long row = ((long long)b * a.Hq + kh * G + r / a.Lq) * a.Lq + r % a.Lq;
      const long long pr = (long long)blockIdx.y * a.B * a.Hq * a.Lq + row;
      a.po[pr * a.D + d] = mine[r * LD + d];
      if (d == 0) {
        a.pml[2 * pr] = bml[2 * r];
        a.pml[2 * pr + 1] = bml[2 * r + 1];
      }
    }
    return;
  }
  if (CLUSTER) cluster_sync();
  else __syncthreads();
  // the blocks of the cluster take the values in turn
  const int ranks = CLUSTER ? a.nsplit : 1, rank = CLUSTER ? (int)blockIdx.y : 0;
  const uint32_t at_o = ptx::smem_u32(mine), at_ml = ptx::smem_u32(bml);
  for (int e = rank * kT + tid; e < rows * a.D; e += ranks * kT) {
    const int r = e / a.D, d = e % a.D;
    float M, L, v;
    if (CLUSTER) {
      float ms[kCluster];
      M = -INFINITY;
#pragma unroll
      for (int c = 0; c < kCluster; ++c) {
        ms[c] = c < ranks ? ld_cluster(at_ml + 8 * r, c) : -INFINITY;
        M = fmaxf(M, ms[c]);
      }
      L = v = 0.f;
#pragma unroll
      for (int c = 0; c < kCluster; ++c)
        if (c < ranks) {
          const float f = ms[c] == -INFINITY ? 0.f : exp2_approx(ms[c] - M);
          L = fmaf(f, ld_cluster(at_ml + 8 * r + 4, c), L);
          v = fmaf(f, ld_cluster(at_o + 4 * (r * LD + d), c), v);
        }
    } else {
      M = bml[2 * r], L = bml[2 * r + 1], v = mine[r * LD + d];
    }
    const int i = r % a.Lq, h = kh * G + r / a.Lq;
    static_cast<T*>(a.out)[(((long long)b * a.Lq + i) * a.Hq + h) * a.D + d] = from_f<T>(L == 0.f ? 0.f : v / L);
    if (d == 0) a.lse[((long long)b * a.Hq + h) * a.Lq + i] = row_lse(M, L);
  }
  if (CLUSTER) cluster_sync();  // no block leaves while another reads its memory
}

// Joins the splits of a row: one warp per row, lanes over the head dimension.
template <typename T>
__global__ void attn_join_kernel(const __grid_constant__ AttnArgs a, long long rows) {
  const long long row = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  float M = -INFINITY, L = 0.f;
  for (int s = lane; s < a.nsplit; s += 32) M = fmaxf(M, a.pml[2 * (s * rows + row)]);
#pragma unroll
  for (int x = 16; x; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.nsplit; ++s) {
    const long long pr = s * rows + row;
    const float ms = a.pml[2 * pr];
    const float ls = a.pml[2 * pr + 1];
    if (ls == 0.f) continue;  // no weight; a NaN sum has a maximum of -inf too where every score is NaN
    const float f = exp2_approx(ms - M);
    L = fmaf(f, ls, L);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (lane + 32 * x < a.D) o[x] = fmaf(f, a.po[pr * a.D + lane + 32 * x], o[x]);
  }
  const float inv = row_inv(L);
  const long long i = row % a.Lq, bh = row / a.Lq, b = bh / a.Hq, h = bh % a.Hq;
  T* dst = static_cast<T*>(a.out) + ((b * a.Lq + i) * a.Hq + h) * a.D;
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (lane + 32 * x < a.D) dst[lane + 32 * x] = from_f<T>(o[x] * inv);
  if (lane == 0) a.lse[row] = row_lse(M, L);
}

// --------------------------------------------------------------- backward
// delta_i = sum_j P dP.  For fp32 it is dout_i . out_i, one warp per row; a
// 16-bit out is too coarse for it (where the softmax is narrow, or a wide bucket
// of the bias is summed, dP - delta cancels), so there the dQ kernel runs once
// more before, for delta alone.
__global__ void attn_delta_kernel(const __grid_constant__ AttnArgs a, long long rows) {
  const long long row = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const long long i = row % a.Lq, bh = row / a.Lq, b = bh / a.Hq, h = bh % a.Hq;
  const float* x = static_cast<const float*>(a.dout) + b * a.dos[0] + i * a.dos[1] + h * a.dos[2];
  const float* y = static_cast<const float*>(a.fout) + b * a.os[0] + i * a.os[1] + h * a.os[2];
  float s = 0.f;
  for (int d = lane; d < a.D; d += 32) s = fmaf(x[d], y[d], s);
#pragma unroll
  for (int z = 16; z; z >>= 1) s += __shfl_xor_sync(0xffffffffu, s, z);
  if (lane == 0) a.delta[row] = s;
}

// The delta of a query with one key at most (lone_queries) is this NaN, whose bits
// no sum gives (an infinite delta is a result, which has to go on into the
// gradients).
constexpr uint32_t kLone = 0x7fc01ead;
__device__ __forceinline__ bool is_lone(float delta) { return __float_as_uint(delta) == kLone; }

// The second half's accumulators added to the first's, through shared memory
// that nobody reads any more; false for the second half, which is done.
template <int DP>
__device__ __forceinline__ bool add_halves(float (&acc)[DP / 8][4], float* mem, int warp, int half, int lane) {
  __syncthreads();
  float* at = mem + (warp * 32 + lane) * (DP / 2 + 1);
  if (half)
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x) at[d * 4 + x] = acc[d][x];
  __syncthreads();
  if (half) return false;
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[d][x] += at[d * 4 + x];
  return true;
}

// dQ = scale dS K for 64 queries of one query head, with the sums of dS along
// the diagonals of every tile when the table's gradient is wanted: thread u
// adds the entries (y, x) with x - y = u - 63, in the order of the rows; the
// upper half of a tile's diagonals goes on in the next tile.
//
// KS = 2 (fp32, whose blocks are few and long): eight warps, two to 16 rows, each
// half of a tile's keys; their sums are added at the end.
template <typename T, int DP, int BN, int KS, bool DELTA>
__global__ void __launch_bounds__(kT * KS) attn_mma_dq_kernel(const __grid_constant__ AttnArgs a, int vec_q, int vec_kv,
                                                         int vec_do) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int P = pitch<DP>(), TH = kT * KS;
  constexpr int NT = BN / 8 / KS;
  constexpr int ST = sizeof(T) == 4 ? 1 : 2;
  const int tid = threadIdx.x, warp = (tid >> 5) & 3, key0 = (tid >> 7) * NT * 8, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.Hq / a.Hkv;
  const unsigned ntile = (unsigned)((a.Lq + kBM - 1) / kBM);
  const int b = blockIdx.x / ntile / a.Hq, h = blockIdx.x / ntile % a.Hq, kh = h / G;
  const long long i0 = (long long)(blockIdx.x % ntile) * kBM;
  const uint32_t sm = ptx::smem_u32(smem);
  constexpr uint32_t TM = tile_bytes<T, DP>(kBM), TB = tile_bytes<T, DP>(BN);
  const Rows sQ = {sm, kBM * P}, sO = {sm + TM, kBM * P};
  const auto kv = [&](int st, int v) { return Rows{sm + 2 * TM + (2 * st + v) * TB, BN * P}; };
  constexpr int SL = BN + 1;
  float* sD = reinterpret_cast<float*>(smem + 2 * TM + 2 * ST * TB);  // dS tile [64][BN + 1], carry behind
  float* carry = sD + kBM * SL;
  const int len = kv_len(a, b);
  long long kend = len;
  if (a.causal) kend = max(0ll, min(kend, min((long long)a.Lq, i0 + kBM) - 1 + a.q_off + 1));
  const int tiles = (int)((kend + BN - 1) / BN);
  const T* qb = static_cast<const T*>(a.q) + (int64_t)b * a.qs[0] + (int64_t)h * a.qs[2];
  const T* ob = static_cast<const T*>(a.dout) + (int64_t)b * a.dos[0] + (int64_t)h * a.dos[2];
  const T* kb = static_cast<const T*>(a.k) + (int64_t)b * a.ks[0] + (int64_t)kh * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + (int64_t)b * a.vs[0] + (int64_t)kh * a.vs[2];
  const uint8_t* mb = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
  stage_rows<T, DP, TH>(sQ, kBM, a.D, vec_q, tid,
                    [&](int r) -> const T* { return i0 + r < a.Lq ? qb + (i0 + r) * a.qs[1] : nullptr; });
  stage_rows<T, DP, TH>(sO, kBM, a.D, vec_do, tid,
                    [&](int r) -> const T* { return i0 + r < a.Lq ? ob + (i0 + r) * a.dos[1] : nullptr; });
  auto load = [&](int tile, int st) {
    const int j0 = tile * BN;
    auto alive = [&](int r) { return j0 + r < len && (!mb || mb[(int64_t)(j0 + r) * a.mask_k]); };
    stage_rows<T, DP, TH>(kv(st, 0), BN, a.D, vec_kv, tid,
                      [&](int r) -> const T* { return alive(r) ? kb + (int64_t)(j0 + r) * a.ks[1] : nullptr; });
    stage_rows<T, DP, TH>(kv(st, 1), BN, a.D, vec_kv, tid,
                      [&](int r) -> const T* { return alive(r) ? vb + (int64_t)(j0 + r) * a.vs[1] : nullptr; });
    cp_commit();
  };
  if (ST == 2 && tiles > 0) load(0, 0);
  const int lone = DELTA ? 0 : lone_queries(a, b, len);
  long long qi[2];
  float lse2[2], delta[2];
  const float* bias[2];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    qi[y] = min(i0 + warp * 16 + g + 8 * y, (long long)a.Lq - 1);
    const long long row = ((long long)b * a.Hq + h) * a.Lq + qi[y];
    const float z = a.lse[row];
    const bool live = z != -INFINITY && i0 + warp * 16 + g + 8 * y < a.Lq;
    lse2[y] = live ? z * kLog2e : INFINITY;  // a row that is not there or has no key: P = 0
    delta[y] = DELTA ? 0.f : qi[y] < lone ? __uint_as_float(kLone) : a.delta[row];
    bias[y] = a.diag ? a.diag + h * a.diag_ld + a.diag0 - qi[y] : nullptr;
  }
  const float sc = a.scale * kLog2e;
  float acc[DP / 8][4];
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[d][x] = 0.f;
  float* dws = a.dws && !DELTA ? a.dws + (long long)blockIdx.x * a.dws_ld : nullptr;
  if (dws && tid < kBM) carry[tid] = 0.f;
  for (int tile = 0; tile < tiles; ++tile) {
    const int st = ST == 2 ? tile & 1 : 0;
    if (ST == 1) {
      load(tile, 0);
    } else if (tile + 1 < tiles) {
      load(tile + 1, st ^ 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    float s[NT][4], dp[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[n][x] = dp[n][x] = 0.f;
    const Rows k = {kv(st, 0).at + key0 * P, BN * P}, v = {kv(st, 1).at + key0 * P, BN * P};
    mma_abt<T, DP, NT>(s, Rows{sQ.at + warp * 16 * P, sQ.part}, k, lane);
    mma_abt<T, DP, NT>(dp, Rows{sO.at + warp * 16 * P, sO.part}, v, lane);
    const int j0 = tile * BN;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int j = j0 + key0 + n * 8 + 2 * t + (x & 1), y = x >> 1;
        float z = s[n][x] * sc;
        if (a.diag && j < a.Lk) z += __ldg(bias[y] + j);
        const bool on = j < len && (!mb || mb[(int64_t)j * a.mask_k]) && (!a.causal || j <= qi[y] + a.q_off);
        const float p = on ? exp2_approx(z - lse2[y]) : 0.f;
        s[n][x] = p != 0.f && (DELTA || !is_lone(delta[y])) ? p * (dp[n][x] - (DELTA ? 0.f : delta[y])) : 0.f;
        if (DELTA) delta[y] += s[n][x];
        if (dws) sD[(warp * 16 + g + 8 * y) * SL + key0 + n * 8 + 2 * t + (x & 1)] = s[n][x];
      }
    if (!DELTA) mma_pb<T, DP, NT>(acc, s, k, lane);
    __syncthreads();
    if (dws) {  // diagonals u = x - y + 63 of this tile, 0 <= u < 63 + BN
      const int u = tid;
      float z = u < kBM - 1 ? carry[u] : 0.f;
      if (u < kBM - 1 + BN) {
        const int d = u - (kBM - 1);
        for (int y = max(0, -d); y < min(kBM, BN - d); ++y) z += sD[y * SL + y + d];
        if (u < BN) dws[(long long)tile * BN + u] = z;
      }
      __syncthreads();
      if (u >= BN && u < kBM - 1 + BN) carry[u - BN] = z;
      __syncthreads();
    }
  }
  if (DELTA) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      delta[y] += __shfl_xor_sync(0xffffffffu, delta[y], 1);
      delta[y] += __shfl_xor_sync(0xffffffffu, delta[y], 2);
      const long long i = i0 + warp * 16 + g + 8 * y;
      if (t == 0 && i < a.Lq) a.delta[((long long)b * a.Hq + h) * a.Lq + i] = delta[y];
    }
    return;
  }
  if (dws) {  // the last diagonals, and zeros where no tile was
    const long long at = (long long)tiles * BN;
    for (long long x = at + tid; x < a.dws_ld; x += TH) dws[x] = x - at < kBM - 1 ? carry[x - at] : 0.f;
  }
  if constexpr (KS == 2) {
    if (!add_halves<DP>(acc, reinterpret_cast<float*>(smem), warp, tid >> 7, lane)) return;
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const long long i = i0 + warp * 16 + g + 8 * y;
    if (i >= a.Lq) continue;
    T* dst = static_cast<T*>(a.dq) + (((long long)b * a.Lq + i) * a.Hq + h) * a.D;
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
      for (int z = 0; z < 2; ++z)
        if (d * 8 + 2 * t + z < a.D) dst[d * 8 + 2 * t + z] = from_f<T>(acc[d][2 * y + z] * a.scale);
  }
}

// dK = scale sum dS^T Q and dV = sum P^T dO for 64 keys of one KV head, over
// every query of every head of its group, BQ rows at a time.
// KS as above, over the rows.
template <typename T, int DP, int BQ, int KS>
__global__ void __launch_bounds__(kT * KS) attn_mma_dkv_kernel(const __grid_constant__ AttnArgs a, int vec_q, int vec_kv,
                                                          int vec_do) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int P = pitch<DP>(), TH = kT * KS;
  constexpr int NT = BQ / 8 / KS;
  constexpr int ST = sizeof(T) == 4 ? 1 : 2;
  const int tid = threadIdx.x, warp = (tid >> 5) & 3, row0 = (tid >> 7) * NT * 8, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.Hq / a.Hkv;
  const unsigned ntile = (unsigned)((a.Lk + kBN - 1) / kBN);
  const int b = blockIdx.x / ntile / a.Hkv, kh = blockIdx.x / ntile % a.Hkv;
  const int j0 = (int)(blockIdx.x % ntile) * kBN;
  const uint32_t sm = ptx::smem_u32(smem);
  constexpr uint32_t TM = tile_bytes<T, DP>(kBN), TB = tile_bytes<T, DP>(BQ);
  const Rows sK = {sm, kBN * P}, sV = {sm + TM, kBN * P};
  const auto qo = [&](int st, int o) { return Rows{sm + 2 * TM + (2 * st + o) * TB, BQ * P}; };
  float* stat = reinterpret_cast<float*>(smem + 2 * TM + 2 * ST * TB);  // [stages][2][BQ]: lse2, delta
  const int len = kv_len(a, b);
  const T* qb = static_cast<const T*>(a.q) + (int64_t)b * a.qs[0];
  const T* ob = static_cast<const T*>(a.dout) + (int64_t)b * a.dos[0];
  const T* kb = static_cast<const T*>(a.k) + (int64_t)b * a.ks[0] + (int64_t)kh * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + (int64_t)b * a.vs[0] + (int64_t)kh * a.vs[2];
  const uint8_t* mb = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
  auto alive = [&](int j) { return j < len && (!mb || mb[(int64_t)j * a.mask_k]); };
  stage_rows<T, DP, TH>(sK, kBN, a.D, vec_kv, tid,
                    [&](int r) -> const T* { return alive(j0 + r) ? kb + (int64_t)(j0 + r) * a.ks[1] : nullptr; });
  stage_rows<T, DP, TH>(sV, kBN, a.D, vec_kv, tid,
                    [&](int r) -> const T* { return alive(j0 + r) ? vb + (int64_t)(j0 + r) * a.vs[1] : nullptr; });
  // rows of one head at a time, so a tile never holds two heads; with a causal
  // mask only queries with i + q_off >= j0 meet these keys
  long long ifirst = 0;
  if (a.causal) ifirst = max(0ll, (long long)j0 - a.q_off) / BQ * BQ;
  const int per = j0 < len && ifirst < a.Lq ? (int)((a.Lq - ifirst + BQ - 1) / BQ) : 0;
  const long long tiles = (long long)per * G;
  const int lone = tiles > 0 ? lone_queries(a, b, len) : 0;
  auto load = [&](long long tile, int st) {
    const int h = kh * G + (int)(tile / per);
    const long long i0 = ifirst + (tile % per) * BQ;
    stage_rows<T, DP, TH>(qo(st, 0), BQ, a.D, vec_q, tid, [&](int r) -> const T* {
      return i0 + r < a.Lq ? qb + (i0 + r) * a.qs[1] + (int64_t)h * a.qs[2] : nullptr;
    });
    stage_rows<T, DP, TH>(qo(st, 1), BQ, a.D, vec_do, tid, [&](int r) -> const T* {
      return i0 + r < a.Lq ? ob + (i0 + r) * a.dos[1] + (int64_t)h * a.dos[2] : nullptr;
    });
    if (tid < BQ) {
      const bool in = i0 + tid < a.Lq;
      const long long row = ((long long)b * a.Hq + h) * a.Lq + i0 + tid;
      const float z = in ? a.lse[row] : -INFINITY;
      stat[(st * 2) * BQ + tid] = z != -INFINITY ? z * kLog2e : INFINITY;
      stat[(st * 2 + 1) * BQ + tid] = !in ? 0.f : i0 + tid < lone ? __uint_as_float(kLone) : a.delta[row];
    }
    cp_commit();
  };
  if (ST == 2 && tiles > 0) load(0, 0);
  int key[2];
  bool on[2];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    key[y] = j0 + warp * 16 + g + 8 * y;
    on[y] = alive(key[y]);
  }
  const float sc = a.scale * kLog2e;
  float dk[DP / 8][4], dv[DP / 8][4];
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x) dk[d][x] = dv[d][x] = 0.f;
  for (long long tile = 0; tile < tiles; ++tile) {
    const int st = ST == 2 ? (int)(tile & 1) : 0;
    if (ST == 1) {
      load(tile, 0);
    } else if (tile + 1 < tiles) {
      load(tile + 1, st ^ 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    const int h = kh * G + (int)(tile / per);
    const long long i0 = ifirst + (tile % per) * BQ;
    const float* bias = a.diag ? a.diag + h * a.diag_ld + a.diag0 : nullptr;
    float s[NT][4], dp[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[n][x] = dp[n][x] = 0.f;
    const Rows q = {qo(st, 0).at + row0 * P, BQ * P}, o = {qo(st, 1).at + row0 * P, BQ * P};
    mma_abt<T, DP, NT>(s, Rows{sK.at + warp * 16 * P, sK.part}, q, lane);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int c = row0 + n * 8 + 2 * t + (x & 1), y = x >> 1;
        const long long i = i0 + c;
        float v = s[n][x] * sc;
        if (bias && i < a.Lq && key[y] < a.Lk) v += __ldg(bias + key[y] - i);
        const bool live = on[y] && (!a.causal || key[y] <= i + a.q_off);
        s[n][x] = live ? exp2_approx(v - stat[st * 2 * BQ + c]) : 0.f;
      }
    mma_pb<T, DP, NT>(dv, s, o, lane);
    mma_abt<T, DP, NT>(dp, Rows{sV.at + warp * 16 * P, sV.part}, o, lane);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float de = stat[(st * 2 + 1) * BQ + row0 + n * 8 + 2 * t + (x & 1)];
        s[n][x] = s[n][x] != 0.f && !is_lone(de) ? s[n][x] * (dp[n][x] - de) : 0.f;
      }
    mma_pb<T, DP, NT>(dk, s, q, lane);
    __syncthreads();
  }
  if constexpr (KS == 2) {
    const bool on1 = add_halves<DP>(dk, reinterpret_cast<float*>(smem), warp, tid >> 7, lane);
    if (!add_halves<DP>(dv, reinterpret_cast<float*>(smem), warp, tid >> 7, lane) || !on1) return;
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    if (key[y] >= a.Lk) continue;
    const long long at = (((long long)b * a.Lk + key[y]) * a.Hkv + kh) * a.D;
    T* pk = static_cast<T*>(a.dk) + at;
    T* pv = static_cast<T*>(a.dv) + at;
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
      for (int z = 0; z < 2; ++z)
        if (d * 8 + 2 * t + z < a.D) {
          pk[d * 8 + 2 * t + z] = from_f<T>(dk[d][2 * y + z] * a.scale);
          pv[d * 8 + 2 * t + z] = from_f<T>(dv[d][2 * y + z]);
        }
  }
}

// Lifts a kernel's limit of dynamic shared memory once per device.
template <auto K>
void allow_smem(size_t smem) {
  static std::atomic<uint64_t> done{0};
  if (smem <= 48 * 1024) return;
  int dev = 0;
  RVC_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 64 && (done.load(std::memory_order_relaxed) & (1ull << dev))) return;
  RVC_CUDA_TRY(cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
  if (dev < 64) done.fetch_or(1ull << dev);
}

bool few_rows(const AttnArgs& a) { return (long long)(a.Hq / a.Hkv) * a.Lq <= 16; }

template <typename T, int DP>
void few_dp(const AttnArgs& a, cudaStream_t st) {
  const int vq = aligned16(a, a.q, a.qs), vkv = aligned16(a, a.k, a.ks) && aligned16(a, a.v, a.vs);
  constexpr size_t smem = few_smem<T, DP>();
  const dim3 grid((unsigned)(a.B * a.Hkv), a.nsplit);
  if (a.nsplit > 1 && a.nsplit <= kCluster) {
    allow_smem<attn_mma_few_kernel<T, DP, true>>(smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1;
    at[0].val.clusterDim.y = a.nsplit;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    RVC_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn_mma_few_kernel<T, DP, true>, a, vq, vkv));
  } else {
    allow_smem<attn_mma_few_kernel<T, DP, false>>(smem);
    attn_mma_few_kernel<T, DP, false><<<grid, kT, smem, st>>>(a, vq, vkv);
  }
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
}

template <typename T, int DP>
void fwd_dp(const AttnArgs& a, cudaStream_t st) {
  if (few_rows(a)) {
    few_dp<T, DP>(a, st);
  } else {
    const int vq = aligned16(a, a.q, a.qs), vkv = aligned16(a, a.k, a.ks) && aligned16(a, a.v, a.vs);
    const long long rows = (long long)(a.Hq / a.Hkv) * a.Lq;
    constexpr size_t smem = tile_bytes<T, DP>(kFwdRows<T>) + 2 * kFwdStages<T> * tile_bytes<T, DP>(kFwdKeys<T>);
    constexpr int BM = kFwdRows<T>;
    const dim3 grid((unsigned)((rows + BM - 1) / BM * a.B * a.Hkv), a.nsplit);
    allow_smem<attn_mma_fwd_kernel<T, DP>>(smem);
    attn_mma_fwd_kernel<T, DP><<<grid, 2 * BM, smem, st>>>(a, vq, vkv);
    note_launch();
    RVC_CUDA_TRY(cudaGetLastError());
  }
  attn_join(a, st);
}

template <typename T, int DP>
void bwd_dp(const AttnArgs& a, cudaStream_t st) {
  const int vq = aligned16(a, a.q, a.qs), vkv = aligned16(a, a.k, a.ks) && aligned16(a, a.v, a.vs),
            vdo = aligned16(a, a.dout, a.dos);
  // fp32: tiles of 32 rows in one stage, eight warps to a block
  constexpr int BN = sizeof(T) == 4 ? 32 : 64, KS = sizeof(T) == 4 ? 2 : 1, ST = sizeof(T) == 4 ? 1 : 2;
  constexpr size_t tiles = 2 * tile_bytes<T, DP>(kBM) + 2 * ST * tile_bytes<T, DP>(BN);
  constexpr size_t halves = KS == 2 ? (size_t)128 * (DP / 2 + 1) * 4 : 0;
  const long long n = (long long)a.B * a.Hq * a.Lq;
  if (n > 0) {
    const size_t smem = std::max(halves, tiles + (a.dws ? (size_t)(kBM * (BN + 1) + kBM) * 4 : 0));
    const unsigned grid = (unsigned)((a.Lq + kBM - 1ll) / kBM * a.B * a.Hq);
    if constexpr (sizeof(T) == 4) {
      attn_delta_kernel<<<(unsigned)((n + 7) / 8), 256, 0, st>>>(a, n);
    } else {
      allow_smem<attn_mma_dq_kernel<T, DP, BN, KS, true>>(smem);
      attn_mma_dq_kernel<T, DP, BN, KS, true><<<grid, kT * KS, smem, st>>>(a, vq, vkv, vdo);
    }
    note_launch();
    RVC_CUDA_TRY(cudaGetLastError());
    allow_smem<attn_mma_dq_kernel<T, DP, BN, KS, false>>(smem);
    attn_mma_dq_kernel<T, DP, BN, KS, false><<<grid, kT * KS, smem, st>>>(a, vq, vkv, vdo);
    note_launch();
    RVC_CUDA_TRY(cudaGetLastError());
  }
  if (a.Lk > 0) {
    constexpr size_t smem = std::max(halves, tiles + (size_t)2 * ST * BN * 4);
    allow_smem<attn_mma_dkv_kernel<T, DP, BN, KS>>(smem);
    attn_mma_dkv_kernel<T, DP, BN, KS>
        <<<(unsigned)((a.Lk + kBN - 1ll) / kBN * a.B * a.Hkv), kT * KS, smem, st>>>(a, vq, vkv, vdo);
    note_launch();
    RVC_CUDA_TRY(cudaGetLastError());
  }
}

template <typename T>
void fwd_t(const AttnArgs& a, cudaStream_t st) {
  if (a.D <= 32) fwd_dp<T, 32>(a, st);
  else if (a.D <= 64) fwd_dp<T, 64>(a, st);
  else if (a.D <= 96) fwd_dp<T, 96>(a, st);
  else fwd_dp<T, 128>(a, st);
}
template <typename T>
void bwd_t(const AttnArgs& a, cudaStream_t st) {
  if (a.D <= 32) bwd_dp<T, 32>(a, st);
  else if (a.D <= 64) bwd_dp<T, 64>(a, st);
  else if (a.D <= 96) bwd_dp<T, 96>(a, st);
  else bwd_dp<T, 128>(a, st);
}

}  // namespace

// Splits of the keys.  Many rows: enough blocks for two to an SM, at least two
// key tiles each.  Few rows: 64 keys at least (a step for each warp), no more
// than four blocks to an SM, a power of two up to kCluster (a GPU cluster's
// blocks share a group of 16 to 18 SMs); where that leaves SMs without work (a
// single long sequence), as many as fill the GPU, through the workspace.
int attn_mma_splits(const AttnArgs& a, int sms, bool* workspace) {
  const long long rows = (long long)(a.Hq / a.Hkv) * a.Lq;
  *workspace = false;
  if (rows == 0 || a.B == 0) return 1;
  if (few_rows(a)) {
    const long long blocks = (long long)a.B * a.Hkv;
    const long long n = std::min((a.Lk + 63ll) / 64, (4ll * sms + blocks - 1) / blocks);
    if (n > kCluster && blocks * kCluster < sms) {
      *workspace = true;
      return (int)std::min<long long>({n, (sms + blocks - 1) / blocks, 128ll});
    }
    int p = 1;
    while (p < n && p < kCluster) p *= 2;
    return p;
  }
  const int BM = a.type == kF32 ? kFwdRows<float> : kBM;
  const long long blocks = (rows + BM - 1) / BM * a.B * a.Hkv;
  const int tiles = (a.Lk + kBN - 1) / kBN;
  const long long want = (2ll * sms + blocks - 1) / blocks;
  const int n = (int)std::max(1ll, std::min({want, (long long)(tiles / 2), 64ll}));
  *workspace = n > 1;
  return n;
}

void attn_join(const AttnArgs& a, cudaStream_t st) {
  if (!a.po) return;
  const long long n = (long long)a.B * a.Hq * a.Lq;
  const unsigned grid = (unsigned)((n + 7) / 8);
  if (a.type == kF32) attn_join_kernel<float><<<grid, 256, 0, st>>>(a, n);
  else if (a.type == kBf16) attn_join_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a, n);
  else attn_join_kernel<__half><<<grid, 256, 0, st>>>(a, n);
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
}

void attn_mma_forward(const AttnArgs& a, cudaStream_t st) {
  switch (a.type) {
    case kF32: return fwd_t<float>(a, st);
    case kBf16: return fwd_t<__nv_bfloat16>(a, st);
    default: return fwd_t<__half>(a, st);
  }
}

void attn_mma_backward(const AttnArgs& a, cudaStream_t st) {
  switch (a.type) {
    case kF32: return bwd_t<float>(a, st);
    case kBf16: return bwd_t<__nv_bfloat16>(a, st);
    default: return bwd_t<__half>(a, st);
  }
}

}  // namespace rvc
