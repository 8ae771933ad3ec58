// Attention on the fifth-generation tensor cores (16-bit inputs, many queries).
//
// One block takes 256 queries of one head, as two tiles of 128, and walks over
// the keys in tiles of 128:
//   warp 8    loads Q once and K, V (and the bias of the tile's diagonals) per
//             key tile by TMA into 128-byte swizzled slabs, two stages each;
//   warp 9    issues S = Q K^T (fp32 in tensor memory) and O += P V with P read
//             from tensor memory, in the order S0 S1 | O0 S0' | O1 S1' ..., so
//             that one tile's products run while the other's softmax does;
//   warps 0-3 and 4-7: the softmax of one query tile each, one row to a thread,
//             so that row maxima and sums need no exchange.  P = 2^(s - m) is
//             written back as 16-bit pairs over the columns of S.
// The output stays in tensor memory over all key tiles.  It is rescaled only
// when a row's maximum has grown by more than 2^8 over the one in use (P then
// stays below 256, far inside either 16-bit type, and the sums are fp32).
// P is rounded to the inputs' type: the same relative step as the output's own.
//
// A tile's dead keys get s = -inf; their rows of V are zeroed in shared memory
// first, so that nothing a padded buffer holds reaches a product.
//
// Every wait is bounded; one that gives up sets the context's error word, lets the
// block wind down and leaves NaN in the rows that are not finished.
//
// Measured: 2 x 16/4 heads x 2048 x 16384 x 128, bf16: 485 to 555 us from run to
// run, 0.99 to 1.13 PFLOP/s of 1.70; the same pipeline with the softmax taken out
// takes 433, so the products and their two waves of blocks bound it.  4 x 16 x 2047
// x 2047 x 64 with the bias, fp16: 159 us, of which 38 are the look-ups of the bias.
// Sixteen softmax warps (two to a row) took 895 us for the first, exponentials by
// polynomial for one pair in eight 588 against 511.
#include "attn_tc.cuh"
#include "context.cuh"

#include <algorithm>
#include <atomic>
#include <mutex>

namespace rvc {

namespace atc {

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  if (!fn) throw Error{kErrCuda, "cuTensorMapEncodeTiled is not available from the driver"};
  return fn;
}

// TMA wants 16-byte aligned starts and strides; a stride of a dimension that
// has one entry is never used, any other must be positive and below 2^40 bytes.
bool map_ok(const AttnArgs& a, const void* p, const int64_t* s, int L, int H) {
  const int64_t n[3] = {a.B, L, H};
  if (reinterpret_cast<uintptr_t>(p) % 16 || a.D * 2 % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] <= 0 || s[i] * 2 % 16 || s[i] * 2 >= (1ll << 40))) return false;
  return true;
}

void make_map(CUtensorMap* m, int type, const void* p, const int64_t* s, int B, int L, int H, int D, int rows) {
  const cuuint64_t row = (cuuint64_t)(D * 2 + 15) / 16 * 16;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)L, (cuuint64_t)B};
  cuuint64_t strides[3] = {H > 1 ? (cuuint64_t)s[2] * 2 : row, L > 1 ? (cuuint64_t)s[1] * 2 : row,
                           B > 1 ? (cuuint64_t)s[0] * 2 : row};
  cuuint32_t box[4] = {64, 1, (cuuint32_t)rows, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  CUresult r = encode_fn()(m, type == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                           const_cast<void*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error{kErrCuda, "cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")"};
}

}  // namespace atc

namespace {

using namespace atc;

constexpr int kFwdThreads = 384;  // three warpgroups: two of softmax, one of loader and issuer
constexpr float kGrow = 8.f;  // log2 of the growth of a maximum that is taken without rescaling
// Largest bias that a whole tile may keep beside its products, x mul + (add - m):
// up to here add and m are exact to 2^-12, beyond (and for -inf, which masks) the
// bias is added pair by pair, so that a row's maximum holds it as its scores do.
constexpr float kFlatMost = 4096.f;

struct FwdMaps {
  CUtensorMap q, k, v;
};

// Key tiles under way: a load takes about as long as a tile of 128 values does,
// two tiles of 64 and more.
template <int NS> constexpr int kRing = NS == 1 ? 4 : 2;
// shared memory: Q [2 tiles][NS], K [stages][NS], V [stages][NS] slabs, bias [stages][384], barriers
template <int NS> constexpr uint32_t fwd_smem() {
  return (2 + 2 * kRing<NS>) * NS * kSlab + kRing<NS> * 384 * 4 + 512 + 1024;
}

// FULL: the head dimension is 64 NS, its steps are known to the compiler.
template <typename T, int NS, bool FULL>
__global__ void __launch_bounds__(kFwdThreads, 1)
    attn_tc_fwd_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ FwdMaps maps) {
  constexpr int R = kRing<NS>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (ptx::smem_u32(raw) + 1023) & ~1023u;
  uint8_t* gen = raw + (base - ptx::smem_u32(raw));
  const uint32_t sQ = base, sK = sQ + 2 * NS * kSlab, sV = sK + R * NS * kSlab;
  const uint32_t oB = (2 + 2 * R) * NS * kSlab, oBar = oB + R * 384 * 4;
  const float* bias_s = reinterpret_cast<const float*>(gen + oB);
  const uint32_t bar = base + oBar;
  const uint32_t Q_FULL = bar, K_FULL = bar + 8, V_FULL = K_FULL + 8 * R, K_EMPTY = V_FULL + 8 * R,
                 V_EMPTY = K_EMPTY + 8 * R, S_FULL = V_EMPTY + 8 * R, P_FULL = S_FULL + 16 /* [2 tiles][2 halves] */,
                 O_DONE = P_FULL + 32, DRAIN = O_DONE + 16;
  uint32_t* slot = reinterpret_cast<uint32_t*>(gen + oBar + 248);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int npair = (a.Lq + 255) / 256;
  const int pair = a.causal ? npair - 1 - (int)(blockIdx.x % npair) : (int)(blockIdx.x % npair);
  const int bh = blockIdx.x / npair, b = bh / a.Hq, h = bh % a.Hq, kh = h / (a.Hq / a.Hkv);
  const int q0 = pair * 256;
  const int len = kv_len(a, b);
  long long kend = len;
  if (a.causal) kend = max(0ll, min(kend, (long long)min(a.Lq, q0 + 256) + a.q_off));
  // the key tiles of this split: from key k0 on
  const int all = (int)((kend + 127) / 128), t0 = (int)((long long)all * blockIdx.y / a.nsplit);
  const int tiles = (int)((long long)all * (blockIdx.y + 1) / a.nsplit) - t0, k0 = t0 * 128;

  if (threadIdx.x == 0) {
    ptx::mbar_init(Q_FULL, 1);
    for (int s = 0; s < R; ++s) {
      ptx::mbar_init(K_FULL + 8 * s, 1);
      ptx::mbar_init(V_FULL + 8 * s, 1);
      ptx::mbar_init(K_EMPTY + 8 * s, a.diag ? 9 : 1);  // the softmax warps read the bias of the stage
      ptx::mbar_init(V_EMPTY + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(S_FULL + 8 * s, 1);
      ptx::mbar_init(P_FULL + 16 * s, 4);
      ptx::mbar_init(P_FULL + 16 * s + 8, 4);
      ptx::mbar_init(O_DONE + 8 * s, 1);
    }
    ptx::mbar_init(DRAIN, 1);
    ptx::fence_mbar_init();
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(slot), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *slot;
  // S0 S1 (128 columns each, P over them), O0 O1 (64 NS each)
  const uint32_t tS = tmem, tO = tmem + 256;

  // 3 x 168 registers a thread at the launch: 216 + 216 + 72 (the issuer must not spill)
  if (warp >= 8) {
    regs_down<72>();
    if (warp == 8) {
      if (lane == 0 && tiles > 0) {
        ptx::mbar_expect_tx(Q_FULL, 2 * NS * kSlab);
        for (int w = 0; w < 2; ++w)
          for (int s = 0; s < NS; ++s)
            ptx::tma_load_4d(sQ + (w * NS + s) * kSlab, &maps.q, 64 * s, h, q0 + 128 * w, b, Q_FULL);
        bool ok = true;
        int nk = 0, nv = 0;  // tiles asked for
        for (int t = 0; t < tiles && ok; ++t) {
          const int st = t % R;
          const uint32_t ph = ((t / R) & 1) ^ 1;
          if (!bar_wait(K_EMPTY + 8 * st, ph)) {
            ok = false;
            break;
          }
          ptx::mbar_expect_tx(K_FULL + 8 * st, NS * kSlab + (a.diag ? 384 * 4 : 0));
          for (int s = 0; s < NS; ++s)
            ptx::tma_load_4d(sK + (st * NS + s) * kSlab, &maps.k, 64 * s, kh, k0 + t * 128, b, K_FULL + 8 * st);
          nk = t + 1;
          if (a.diag)
            ptx::bulk_g2s(base + oB + st * 384 * 4, a.diag + h * a.diag_ld + (k0 + t * 128 - q0 - 256 + a.diag0), 384 * 4,
                          K_FULL + 8 * st);
          if (!bar_wait(V_EMPTY + 8 * st, ph)) {
            ok = false;
            break;
          }
          ptx::mbar_expect_tx(V_FULL + 8 * st, NS * kSlab);
          for (int s = 0; s < NS; ++s)
            ptx::tma_load_4d(sV + (st * NS + s) * kSlab, &maps.v, 64 * s, kh, k0 + t * 128, b, V_FULL + 8 * st);
          nv = t + 1;
        }
        if (!ok) atomicExch(a.err, 41);
        // no copy left in flight when the block ends
        bar_wait(Q_FULL, 0);
        for (int x = max(0, nk - R); x < nk; ++x) bar_wait(K_FULL + 8 * (x % R), (x / R) & 1);
        for (int x = max(0, nv - R); x < nv; ++x) bar_wait(V_FULL + 8 * (x % R), (x / R) & 1);
      }
      __syncwarp();
    } else if (warp == 9) {
      if (lane == 0 && tiles > 0) {
        const uint32_t id_s = idesc<T>(128, false, false);
        const int DK = FULL ? 4 * NS : (a.D + 15) / 16;
        const uint32_t id_o = idesc<T>(16 * DK, false, true);
        bool ok = bar_wait(Q_FULL, 0);
        auto issue_s = [&](int w, int t) {
          const int st = t % R;
          if (ok) ok = bar_wait(K_FULL + 8 * st, (t / R) & 1);
          if (!ok) return;
          ptx::tc_fence_after();
          const uint64_t dq = desc_k(sQ + w * NS * kSlab), dk = desc_k(sK + st * NS * kSlab);
#pragma unroll
          for (int kk = 0; kk < 4 * NS; ++kk) {
            if (kk >= DK) break;
            const uint64_t off = (uint64_t)(((kk >> 2) * kSlab + (kk & 3) * 32) >> 4);
            mma_ss(tS + 128 * w, dq + off, dk + off, id_s, kk > 0);
          }
          ptx::mma_commit(S_FULL + 8 * w);
          if (w == 1) ptx::mma_commit(K_EMPTY + 8 * st);
        };
        auto issue_o = [&](int w, int t) {
          const int st = t % R;
          if (ok) ok = bar_wait(V_FULL + 8 * st, (t / R) & 1);
          const uint64_t dv = desc_mn(sV + st * NS * kSlab);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (ok) ok = bar_wait(P_FULL + 16 * w + 8 * x, t & 1);
            if (!ok) return;
            ptx::tc_fence_after();
#pragma unroll
            for (int kk = 4 * x; kk < 4 * x + 4; ++kk)
              mma_ts(tO + 64 * NS * w, tS + 128 * w + 8 * kk, dv + (uint64_t)(kk * 2048 >> 4), id_o, t > 0 || kk > 0);
          }
          ptx::mma_commit(O_DONE + 8 * w);
          if (w == 1) ptx::mma_commit(V_EMPTY + 8 * st);
        };
        issue_s(0, 0);
        issue_s(1, 0);
        for (int t = 0; t < tiles && ok; ++t) {
          issue_o(0, t);
          if (t + 1 < tiles) issue_s(0, t + 1);
          issue_o(1, t);
          if (t + 1 < tiles) issue_s(1, t + 1);
        }
        if (!ok) atomicExch(a.err, 42);
        ptx::mma_commit(DRAIN);
        bar_wait(DRAIN, 0);  // every product done before tensor memory is freed
      }
      __syncwarp();
    }
  } else {
    regs_up<216>();
    const int w = warp >> 2;  // query tile
    const int row = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tS + 128 * w + lanes, o_col = tO + 64 * NS * w + lanes;
    const long long i = (long long)q0 + 128 * w + row;
    const float sc = a.scale * kLog2e;
    // keys that this row may meet: [0, lim)
    const long long lim = a.causal ? min((long long)len, i + a.q_off + 1) : (long long)len;
    // the smallest limit of the warp: tiles below it need no comparison
    const long long wlim =
        a.causal ? min((long long)len, (long long)q0 + 128 * w + (warp & 3) * 32 + a.q_off + 1) : (long long)len;
    const uint8_t* mb = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    uint8_t bytes[4] = {0, 0, 0, 0};  // mask of keys `lane`, 32 + `lane`, ... of the next tile
    auto fetch = [&](int j0) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int j = j0 + 32 * x + lane;
        bytes[x] = j < len ? mb[(int64_t)j * a.mask_k] : 0;
      }
    };
    if (mb) fetch(k0);
    for (int t = 0; t < tiles && ok; ++t) {
      const int st = t % R, j0 = k0 + t * 128;
      uint32_t alive[4] = {~0u, ~0u, ~0u, ~0u};  // the mask's bytes came with the last tile
      if (mb) {
#pragma unroll
        for (int x = 0; x < 4; ++x) alive[x] = __ballot_sync(0xffffffffu, bytes[x] != 0);
        fetch(j0 + 128);
      }
      if (mb || j0 + 128 > len) {  // zero the dead rows of V (both query tiles do, with the same result)
        const uint32_t word = (warp & 3) == 0 ? alive[0] : (warp & 3) == 1 ? alive[1] : (warp & 3) == 2 ? alive[2] : alive[3];
        const bool dead = j0 + row >= len || !((word >> lane) & 1);
        if (!warp_wait(V_FULL + 8 * st, (t / R) & 1)) {
          ok = false;
          break;
        }
        if (dead) {
          uint4* z = reinterpret_cast<uint4*>(gen + (2 + R + st) * NS * kSlab + row * 128);
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int x = 0; x < 8; ++x) z[s * (kSlab / 16) + x] = make_uint4(0, 0, 0, 0);
        }
        ptx::fence_proxy_async_smem();
      }
      // relative positions of this query tile and the key tile: [hi - 254, hi].  Where
      // they lie whole in the last bucket the bias is one value.
      const long long hi = (long long)j0 + 127 - (q0 + 128 * w) - a.q_off;
      const bool flat = !a.diag || hi <= -(long long)a.far || hi - 254 >= (a.far_both ? (long long)a.far : 0ll);
      if (a.diag && !warp_wait(K_FULL + 8 * st, (t / R) & 1)) {
        ok = false;
        break;
      }
      if (!warp_wait(S_FULL + 8 * w, t & 1)) {
        ok = false;
        break;
      }
      ptx::tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int x = 0; x < 4; ++x) ptx::tmem_ld32_async(s_col + 32 * x, s[x]);
#pragma unroll
      for (int x = 0; x < 4; ++x) ptx::tmem_wait_ld(s[x]);
      // exponents are s x + c - m; without a bias by pair the products stay as they are
      float mul = 1.f, add = 0.f;
      bool plain = flat && sc > 0.f;
      if (a.diag) {
        const float* bb = bias_s + st * 384 + 256 - 128 * w - row;
        plain = plain && fabsf(bb[0]) <= kFlatMost;
        if (plain) {
          add = bb[0];
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int c = 0; c < 32; ++c) s[x][c] = __float_as_uint(fmaf(__uint_as_float(s[x][c]), sc, bb[32 * x + c]));
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(K_EMPTY + 8 * st);
      } else if (!plain) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int c = 0; c < 32; ++c) s[x][c] = __float_as_uint(__uint_as_float(s[x][c]) * sc);
      }
      if (plain) mul = sc;
      const bool cut = mb || j0 + 128 > wlim;
      if (cut) {
        const int n = (int)max(0ll, min(128ll, lim - j0));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          alive[x] &= low_bits(n - 32 * x);
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (!(alive[x] & (1u << c))) s[x][c] = 0xff800000u;
        }
      }
      float mx = -INFINITY, my = -INFINITY;
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          mx = fmaxf(fmaxf(mx, __uint_as_float(s[x][c])), __uint_as_float(s[x][c + 1]));
          my = fmaxf(fmaxf(my, __uint_as_float(s[x][c + 2])), __uint_as_float(s[x][c + 3]));
        }
      mx = fmaf(fmaxf(mx, my), mul, add);
      const bool up = mx > m + kGrow;  // always on a row's first live key
      if (__any_sync(0xffffffffu, up)) {
        const float m_new = up ? mx : m;
        const float f = m == -INFINITY ? 0.f : exp2_approx(m - m_new);
        if (t > 0) {
          if (!warp_wait(O_DONE + 8 * w, (t - 1) & 1)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
#pragma unroll 1
          for (int x = 0; x < 64 * NS; x += 16) {
            float o[16];
            ptx::tmem_ld16(o_col + x, o);
            uint32_t r[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) r[c] = __float_as_uint(o[c] * (up ? f : 1.f));
            tmem_st16(o_col + x, r);
          }
        }
        if (up) l *= f;
        m = m_new;
      }
      const float off = m == -INFINITY ? 0.f : add - m;
      const uint64_t mul2 = f32x2(mul, mul), off2 = f32x2(off, off);
      uint64_t l2 = f32x2(0.f, 0.f), l3 = l2;
      // in two halves of 64 keys, so that the product of the first starts early
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t p[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const uint32_t(&v)[32] = s[2 * x + (c >> 4)];
          const uint64_t y =
              fma2(f32x2(__uint_as_float(v[(2 * c) & 31]), __uint_as_float(v[(2 * c + 1) & 31])), mul2, off2);
          float e0, e1;
          split2(y, e0, e1);
          e0 = exp2_approx(e0);
          e1 = exp2_approx(e1);
          if (c & 1) l2 = add2(l2, f32x2(e0, e1));
          else l3 = add2(l3, f32x2(e0, e1));
          p[c] = pack2<T>(e0, e1);
        }
        tmem_st32(s_col + 32 * x, p);
        tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(P_FULL + 16 * w + 8 * x);
      }
      float la, lb;
      split2(add2(l2, l3), la, lb);
      l += la + lb;
    }
    if (ok && tiles > 0) {
      ok = warp_wait(O_DONE + 8 * w, (tiles - 1) & 1);
      ptx::tc_fence_after();
    }
    if (!ok && lane == 0) atomicExch(a.err, 43);
    {
      const bool part = a.nsplit > 1;  // the row as it stands, for attn_join_kernel
      const float inv = part || !ok ? 1.f : row_inv(l);
      T* dst = static_cast<T*>(a.out) + (((long long)b * a.Lq + i) * a.Hq + h) * a.D;
      const long long row_at = ((long long)b * a.Hq + h) * a.Lq + i;
      const long long pr = (long long)blockIdx.y * a.B * a.Hq * a.Lq + row_at;
#pragma unroll 1
      for (int x = 0; x < 64 * NS; x += 16) {
        if (x >= a.D) break;
        float o[16];
        if (ok && tiles > 0) {
          ptx::tmem_ld16(o_col + x, o);
        } else {
#pragma unroll
          for (int c = 0; c < 16; ++c) o[c] = ok ? 0.f : no_result();
        }
        if (i < a.Lq && part) {
#pragma unroll
          for (int c = 0; c < 16; c += 4)
            if (x + c < a.D)
              *reinterpret_cast<float4*>(a.po + pr * a.D + x + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
        } else if (i < a.Lq) {
#pragma unroll
          for (int c = 0; c < 16; c += 8)
            if (x + c < a.D)  // D is a multiple of 8
              *reinterpret_cast<uint4*>(dst + x + c) =
                  make_uint4(pack2<T>(o[c] * inv, o[c + 1] * inv), pack2<T>(o[c + 2] * inv, o[c + 3] * inv),
                             pack2<T>(o[c + 4] * inv, o[c + 5] * inv), pack2<T>(o[c + 6] * inv, o[c + 7] * inv));
        }
      }
      if (i < a.Lq && part) {
        a.pml[2 * pr] = m;
        a.pml[2 * pr + 1] = ok ? l : no_result();
      } else if (i < a.Lq) {
        a.lse[row_at] = ok ? row_lse(m, l) : no_result();
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 9) ptx::tmem_dealloc(tmem, 512);
}

template <typename T, int NS, bool FULL>
void fwd(const AttnArgs& a, cudaStream_t st) {
  FwdMaps maps;
  make_map(&maps.q, a.type, a.q, a.qs, a.B, a.Lq, a.Hq, a.D, 128);
  make_map(&maps.k, a.type, a.k, a.ks, a.B, a.Lk, a.Hkv, a.D, 128);
  make_map(&maps.v, a.type, a.v, a.vs, a.B, a.Lk, a.Hkv, a.D, 128);
  static std::atomic<uint64_t> done{0};  // one bit per device
  int dev = 0;
  RVC_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !(done.load() & (1ull << dev))) {
    RVC_CUDA_TRY(cudaFuncSetAttribute(attn_tc_fwd_kernel<T, NS, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)fwd_smem<NS>()));
    if (dev < 64) done.fetch_or(1ull << dev);
  }
  const unsigned grid = (unsigned)((a.Lq + 255ll) / 256 * a.B * a.Hq);
  attn_tc_fwd_kernel<T, NS, FULL><<<dim3(grid, a.nsplit), kFwdThreads, fwd_smem<NS>(), st>>>(a, maps);
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
}

template <typename T>
void fwd_t(const AttnArgs& a, cudaStream_t st) {
  if (a.D == 64) fwd<T, 1, true>(a, st);
  else if (a.D < 64) fwd<T, 1, false>(a, st);
  else if (a.D == 128) fwd<T, 2, true>(a, st);
  else fwd<T, 2, false>(a, st);
}

}  // namespace

// 16-bit operands that TMA can address, and queries enough: the general kernel
// fills its tiles with the rows of a whole group, this one leaves them empty.
// Measured in us, general / tiles, at 20, 32 and 48 queries (6831 keys unless said):
//   heads of 128   8 x 16/4  191 / 107  181 / 107  235 / 107 (6 queries 98 / 107)
//                  4 x 64/8  233 / 211  308 / 211  450 / 211
//   12 heads of 64  33 / 26   34 / 27   35 / 27;  8 x 12  102 / 98 at 20 to 64
//   64, groups of 2 to 4   8 x 16/4  85 / 98  87 / 98  104 / 98;  1 x 16/4  35 / 26
//       35 / 27  36 / 27;  8 x 8/4  49 / 56  50 / 56  85 / 56;  8 x 16/4 on 499
//       keys  17 / 13  17 / 13  19 / 13;  on 1499 keys  28 / 27  28 / 27  32 / 27
//   64, groups of 8   4 x 64/8  103 / 193  136 / 193  198 / 193
// So for heads of up to 64 in groups of 2 to 4 the general kernel is ahead (12 to 15
// %) at 20 to 32 queries of large batches on thousands of keys, and the tiles
// elsewhere (by up to a third): they take the whole range.
bool attn_tc_fits(const AttnArgs& a) {
  const int least = a.D > 64 || a.Hq / a.Hkv <= 4 ? 20 : 48;
  return a.type != kF32 && a.Lq >= least && a.Lk >= 1 && atc::map_ok(a, a.q, a.qs, a.Lq, a.Hq) &&
         atc::map_ok(a, a.k, a.ks, a.Lk, a.Hkv) && atc::map_ok(a, a.v, a.vs, a.Lk, a.Hkv) &&
         reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
}

void attn_tc_forward(const AttnArgs& a, cudaStream_t st) {
  if (a.type == kBf16) fwd_t<__nv_bfloat16>(a, st);
  else fwd_t<__half>(a, st);
  attn_join(a, st);
}

// Splits of the keys where the query tiles leave half of the SMs or more without
// work: as many as there are idle SMs for, eight tiles of 128 keys each at least
// (the parts of a row are written and read once more, 4 D bytes each).
int attn_tc_splits(const AttnArgs& a, int sms) {
  const long long rows = a.type == kF32 ? 128 : 256;
  const long long blocks = (a.Lq + rows - 1) / rows * a.B * a.Hq;
  return (int)std::max(1ll, std::min({sms / std::max(1ll, blocks), a.Lk / 1024ll, 64ll}));
}

}  // namespace rvc
