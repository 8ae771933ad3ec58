// fp32 attention on the fifth-generation tensor cores, for heads of up to 64
// values and many queries.
//
// x = hi + mid + lo in bf16 carries the 24 bits of an fp32 value, and the six
// products of parts that are above 2^-24 give a product to fp32's accuracy at a
// sixth of the bf16 rate (a third of what TF32 would take with two parts' three
// products at half the rate - the same time - but with exact parts).  A first
// kernel writes the parts of q, k and v into the workspace, where dead keys become
// zeros, so that nothing a padded buffer holds reaches a product.
//
// One block takes 128 queries of one head and walks over the keys in tiles of 64,
// which two groups of four warps take in turn, one query to a thread.  A group has
// its own S, P (three parts) and O in tensor memory, its own running maximum, sum
// and output row in registers, and the two are joined at the end.  Per tile
//   S = the six products, smallest first (the tensor cores cut their sums off:
//       only the last four of 24 instructions add at full size),
//   P = 2^(s - m) in three parts,  O_t = P V in the same order,
//   o = (o + O_(t-2)) 2^(m_old - m) in registers, rounded as fp32.
//
// Measured: 8 x 12 x 499 x 1499 x 64, padded: 202 to 223 us, about 35 of them for
// the parts (the general kernel: 369; tensor pipe busy 26 %, captured alone); error
// 2e-7 of the output's norm.
#include "attn_tc.cuh"
#include "context.cuh"

#include <algorithm>
#include <atomic>

namespace rvc {

namespace {

using namespace atc;

constexpr int kThreads = 384;          // three warpgroups: two of softmax, one of loader and issuer
constexpr uint32_t kTile = kSlab / 2;  // one part of 64 rows
constexpr int R = 3;                   // key tiles under way
using B16 = __nv_bfloat16;

struct Maps {
  CUtensorMap q, k, v;
};

// Q [3 parts of 128 rows], K, V [R][3] tiles, bias [R][192], barriers
constexpr uint32_t kSmem = 3 * kSlab + 6 * R * kTile + R * 192 * 4 + 256 + 1024;

// x [B, L, H, D] with strides -> parts [3][B][L][H][D], dead rows of keys as
// zeros; rows past the last tile that anybody reads are left alone.
__global__ void __launch_bounds__(256) split_kernel(const __grid_constant__ AttnArgs a, const float* __restrict__ x,
                                                    int64_t sb, int64_t sl, int64_t sh, int L, int H, int keys, int vec,
                                                    uint2* __restrict__ out) {
  const int c4 = a.D / 4;
  const long long n = (long long)a.B * L * H * c4;
  for (long long e = blockIdx.x * 256ll + threadIdx.x; e < n; e += gridDim.x * 256ll) {
    const int c = (int)(e % c4);
    const long long r = e / c4;
    const int h = (int)(r % H), l = (int)(r / H % L), b = (int)(r / H / L);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    bool on = true;
    if (keys) {
      const int len = kv_len(a, b);
      if (l >= (len + 63) / 64 * 64) continue;
      on = l < len && (!a.mask || a.mask[b * a.mask_b + l * a.mask_k]);
    }
    if (on) {
      const float* p = x + b * sb + l * sl + h * sh + 4 * c;
      if (vec) v = *reinterpret_cast<const float4*>(p);
      else v = make_float4(p[0], p[1], p[2], p[3]);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const uint32_t w0 = pack2<B16>(v.x, v.y), w1 = pack2<B16>(v.z, v.w);
      out[i * n + e] = make_uint2(w0, w1);
      v.x -= __uint_as_float(w0 << 16), v.y -= __uint_as_float(w0 & 0xffff0000u);
      v.z -= __uint_as_float(w1 << 16), v.w -= __uint_as_float(w1 & 0xffff0000u);
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_f32_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Maps maps) {
  extern __shared__ uint8_t raw[];
  const uint32_t base = (ptx::smem_u32(raw) + 1023) & ~1023u;
  uint8_t* gen = raw + (base - ptx::smem_u32(raw));
  constexpr uint32_t oK = 3 * kSlab, oV = oK + 3 * R * kTile, oB = oV + 3 * R * kTile, oBar = oB + R * 192 * 4;
  const uint32_t sQ = base, sK = base + oK, sV = base + oV;
  const float* bias_s = reinterpret_cast<const float*>(gen + oB);
  const uint32_t bar = base + oBar;
  const uint32_t Q_FULL = bar, K_FULL = bar + 8, V_FULL = K_FULL + 8 * R, K_EMPTY = V_FULL + 8 * R,
                 V_EMPTY = K_EMPTY + 8 * R, S_FULL = V_EMPTY + 8 * R, P_READY = S_FULL + 16, O_FULL = P_READY + 16,
                 DRAIN = O_FULL + 16;
  uint32_t* slot = reinterpret_cast<uint32_t*>(gen + oBar + 248);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nq = (a.Lq + 127) / 128;
  const int qt = a.causal ? nq - 1 - (int)(blockIdx.x % nq) : (int)(blockIdx.x % nq);
  const int bh = blockIdx.x / nq, b = bh / a.Hq, h = bh % a.Hq, kh = h / (a.Hq / a.Hkv);
  const int q0 = qt * 128;
  const int len = kv_len(a, b);
  long long kend = len;
  if (a.causal) kend = max(0ll, min(kend, (long long)min(a.Lq, q0 + 128) + a.q_off));
  // the key tiles of this split: from key k0 on
  const int all = (int)((kend + 63) / 64), t0 = (int)((long long)all * blockIdx.y / a.nsplit);
  const int tiles = (int)((long long)all * (blockIdx.y + 1) / a.nsplit) - t0, k0 = t0 * 64;

  if (threadIdx.x == 0) {
    ptx::mbar_init(Q_FULL, 1);
    for (int s = 0; s < R; ++s) {
      ptx::mbar_init(K_FULL + 8 * s, 1);
      ptx::mbar_init(V_FULL + 8 * s, 1);
      ptx::mbar_init(K_EMPTY + 8 * s, a.diag ? 5 : 1);
      ptx::mbar_init(V_EMPTY + 8 * s, 1);
    }
    for (int w = 0; w < 2; ++w) {
      ptx::mbar_init(S_FULL + 8 * w, 1);
      ptx::mbar_init(P_READY + 8 * w, 4);
      ptx::mbar_init(O_FULL + 8 * w, 1);
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
  // a group's columns at 256 w: S 64, P 3 x 32, O 64
  const uint32_t tS = tmem, tP = tmem + 64, tO = tmem + 160;

  if (warp >= 8) {
    regs_down<72>();  // 216 + 216 + 72 of 3 x 168 at the launch
    if (warp == 8) {
      if (lane == 0 && tiles > 0) {
        ptx::mbar_expect_tx(Q_FULL, 3 * kSlab);
        for (int i = 0; i < 3; ++i) ptx::tma_load_4d(sQ + i * kSlab, &maps.q, 0, h, q0, i * a.B + b, Q_FULL);
        int nk = 0, nv = 0;  // tiles asked for
        bool ok = true;
        for (int t = 0; t < tiles; ++t) {
          const int st = t % R;
          const uint32_t ph = ((t / R) & 1) ^ 1;
          ok = bar_wait(K_EMPTY + 8 * st, ph);
          if (!ok) break;
          ptx::mbar_expect_tx(K_FULL + 8 * st, 3 * kTile + (a.diag ? 768 : 0));
          for (int i = 0; i < 3; ++i)
            ptx::tma_load_4d(sK + (st * 3 + i) * kTile, &maps.k, 0, kh, k0 + t * 64, i * a.B + b, K_FULL + 8 * st);
          if (a.diag)
            ptx::bulk_g2s(base + oB + st * 768, a.diag + h * a.diag_ld + (k0 + t * 64 - q0 - 128 + a.diag0), 768,
                          K_FULL + 8 * st);
          nk = t + 1;
          ok = bar_wait(V_EMPTY + 8 * st, ph);
          if (!ok) break;
          ptx::mbar_expect_tx(V_FULL + 8 * st, 3 * kTile);
          for (int i = 0; i < 3; ++i)
            ptx::tma_load_4d(sV + (st * 3 + i) * kTile, &maps.v, 0, kh, k0 + t * 64, i * a.B + b, V_FULL + 8 * st);
          nv = t + 1;
        }
        if (!ok) atomicExch(a.err, 61);
        bar_wait(Q_FULL, 0);  // no copy left in flight when the block ends
        for (int x = max(0, nk - R); x < nk; ++x) bar_wait(K_FULL + 8 * (x % R), (x / R) & 1);
        for (int x = max(0, nv - R); x < nv; ++x) bar_wait(V_FULL + 8 * (x % R), (x / R) & 1);
      }
      __syncwarp();
    } else if (warp == 9) {
      if (lane == 0 && tiles > 0) {
        const int DK = (a.D + 15) / 16;
        const uint32_t id_s = idesc<B16>(64, false, false), id_o = idesc<B16>(16 * DK, false, true);
        constexpr int pa[6] = {2, 1, 0, 1, 0, 0}, pb[6] = {0, 1, 2, 0, 1, 0};  // parts of the products, smallest first
        bool ok = bar_wait(Q_FULL, 0);
        auto issue_s = [&](int t) {
          const int st = t % R;
          if (ok) ok = bar_wait(K_FULL + 8 * st, (t / R) & 1);
          if (!ok) return;
          ptx::tc_fence_after();
          const uint64_t dq = desc_k(sQ), dk = desc_k(sK + st * 3 * kTile);
#pragma unroll
          for (int i = 0; i < 6; ++i)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              if (kk < DK)
                mma_ss(tS + 256 * (t & 1), dq + (uint64_t)((pa[i] * kSlab + kk * 32) >> 4),
                       dk + (uint64_t)((pb[i] * kTile + kk * 32) >> 4), id_s, i > 0 || kk > 0);
          ptx::mma_commit(S_FULL + 8 * (t & 1));
          ptx::mma_commit(K_EMPTY + 8 * st);
        };
        issue_s(0);
        if (tiles > 1) issue_s(1);
        for (int t = 0; t < tiles && ok; ++t) {
          const int st = t % R;
          ok = bar_wait(V_FULL + 8 * st, (t / R) & 1);
          if (ok) ok = bar_wait(P_READY + 8 * (t & 1), (t >> 1) & 1);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint64_t dv = desc_mn(sV + st * 3 * kTile);
#pragma unroll
          for (int i = 0; i < 6; ++i)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ts(tO + 256 * (t & 1), tP + 256 * (t & 1) + 32 * pa[i] + 8 * kk,
                     dv + (uint64_t)((pb[i] * kTile + kk * 2048) >> 4), id_o, i > 0 || kk > 0);
          ptx::mma_commit(O_FULL + 8 * (t & 1));
          ptx::mma_commit(V_EMPTY + 8 * st);
          if (t + 2 < tiles) issue_s(t + 2);
        }
        if (!ok) atomicExch(a.err, 62);
        ptx::mma_commit(DRAIN);
        bar_wait(DRAIN, 0);  // every product done before tensor memory is freed
      }
      __syncwarp();
    }
  } else {
    regs_up<216>();
    const int w = warp >> 2, row = threadIdx.x & 127;
    const uint32_t at = 256 * w + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_col = tS + at, p_col = tP + at, o_col = tO + at;
    const long long i = (long long)q0 + row;
    const float sc = a.scale * kLog2e;
    const long long lim = a.causal ? min((long long)len, i + a.q_off + 1) : (long long)len;
    const long long wlim =
        a.causal ? min((long long)len, (long long)q0 + (warp & 3) * 32 + a.q_off + 1) : (long long)len;
    const uint8_t* mb = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
    float m = -INFINITY, l = 0.f;
    uint64_t o[32];  // the output row, two values to a word
#pragma unroll
    for (int c = 0; c < 32; ++c) o[c] = f32x2(0.f, 0.f);
    bool ok = true;
    uint8_t byte0 = 0, byte1 = 0;  // mask of keys `lane` and 32 + `lane` of this group's next tile
    auto fetch = [&](int j0) {
      byte0 = j0 + lane < len ? mb[(int64_t)(j0 + lane) * a.mask_k] : 0;
      byte1 = j0 + 32 + lane < len ? mb[(int64_t)(j0 + 32 + lane) * a.mask_k] : 0;
    };
    // adds the group's last O to the row and multiplies by f
    auto fold = [&](float f) {
      const uint64_t f2 = f32x2(f, f);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t u[32];
        ptx::tmem_ld32_async(o_col + 32 * x, u);
        ptx::tmem_wait_ld(u);
#pragma unroll
        for (int c = 0; c < 16; ++c)
          o[16 * x + c] = mul2(add2(o[16 * x + c], f32x2(__uint_as_float(u[2 * c]), __uint_as_float(u[2 * c + 1]))), f2);
      }
    };
    if (mb) fetch(k0 + 64 * w);
    int last = -1;  // this group's last tile
    for (int t = w; t < tiles; t += 2) {
      const int st = t % R, j0 = k0 + t * 64;
      const uint32_t turn = (t >> 1) & 1;
      uint32_t alive[2] = {~0u, ~0u};
      if (mb) {
        alive[0] = __ballot_sync(0xffffffffu, byte0 != 0);
        alive[1] = __ballot_sync(0xffffffffu, byte1 != 0);
        fetch(j0 + 128);
      }
      // relative positions of the tile: [hi - 190, hi]; where they lie whole in the
      // last bucket the bias is one value
      const long long hi = (long long)j0 + 63 - q0 - a.q_off;
      const bool flat = !a.diag || hi <= -(long long)a.far || hi - 190 >= (a.far_both ? (long long)a.far : 0ll);
      if (a.diag && !(ok = warp_wait(K_FULL + 8 * st, (t / R) & 1))) break;
      if (!(ok = warp_wait(S_FULL + 8 * w, turn))) break;
      ptx::tc_fence_after();
      uint32_t s[2][32];
      ptx::tmem_ld32_async(s_col, s[0]);
      ptx::tmem_ld32_async(s_col + 32, s[1]);
      ptx::tmem_wait_ld(s[0]);
      ptx::tmem_wait_ld(s[1]);
      const float* bb = bias_s + st * 192 + 128 - row;
      const float add = a.diag && flat ? bb[0] : 0.f;
      const bool each = !flat;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int c = 0; c < 32; ++c)
          s[x][c] = __float_as_uint(fmaf(__uint_as_float(s[x][c]), sc, each ? bb[32 * x + c] : add));
      if (a.diag) {
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(K_EMPTY + 8 * st);
      }
      if (mb || j0 + 64 > wlim) {
        const int n = (int)max(0ll, min(64ll, lim - j0));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          alive[x] &= low_bits(n - 32 * x);
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (!(alive[x] & (1u << c))) s[x][c] = 0xff800000u;
        }
      }
      float mx = m, my = m;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          mx = fmaxf(fmaxf(mx, __uint_as_float(s[x][c])), __uint_as_float(s[x][c + 1]));
          my = fmaxf(fmaxf(my, __uint_as_float(s[x][c + 2])), __uint_as_float(s[x][c + 3]));
        }
      mx = fmaxf(mx, my);
      const float off = mx == -INFINITY ? 0.f : mx;
      const float f = exp2_approx(m - off);
      // the last O and P of this group are free: fold the one, overwrite the other
      if (last >= 0) {
        if (!(ok = warp_wait(O_FULL + 8 * w, (last >> 1) & 1))) break;
        ptx::tc_fence_after();
        fold(f);
      }
      m = mx;
      l *= f;
      uint64_t l2 = f32x2(0.f, 0.f);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t p[3][16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          float e0 = exp2_approx(__uint_as_float(s[x][2 * c]) - off), e1 = exp2_approx(__uint_as_float(s[x][2 * c + 1]) - off);
          l2 = add2(l2, f32x2(e0, e1));
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            p[k][c] = pack2<B16>(e0, e1);
            e0 -= __uint_as_float(p[k][c] << 16);
            e1 -= __uint_as_float(p[k][c] & 0xffff0000u);
          }
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) tmem_st16(p_col + 32 * k + 16 * x, p[k]);
      }
      float la, lb;
      split2(l2, la, lb);
      l += la + lb;
      tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(P_READY + 8 * w);
      last = t;
    }
    if (ok && last >= 0) {
      ok = warp_wait(O_FULL + 8 * w, (last >> 1) & 1);
      if (ok) {
        ptx::tc_fence_after();
        fold(1.f);
      }
    }
    if (ok && tiles > 0) ok = warp_wait(DRAIN, 0);  // nobody reads the tiles any more
    // Joins the groups: the second leaves its row in shared memory (every warp
    // comes here, also after a wait that gave up).
    ok = ptx::named_bar_and(1, 256, ok);
    float* part = reinterpret_cast<float*>(gen) + row;  // [66][128]
    if (ok && w == 1) {
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        float u, v;
        split2(o[c], u, v);
        part[(2 * c) * 128] = u;
        part[(2 * c + 1) * 128] = v;
      }
      part[64 * 128] = m;
      part[65 * 128] = l;
    }
    ptx::named_bar(1, 256);
    if (!ok && lane == 0) atomicExch(a.err, 63);
    if (w == 0 && i < a.Lq) {
      const float m1 = part[64 * 128], M = fmaxf(m, m1), off = M == -INFINITY ? 0.f : M;
      const float f0 = exp2_approx(m - off), f1 = exp2_approx(m1 - off);
      const float L = f0 * l + f1 * part[65 * 128], inv = a.nsplit > 1 ? 1.f : row_inv(L);
      const long long row_at = ((long long)b * a.Hq + h) * a.Lq + i;
      const long long pr = (long long)blockIdx.y * a.B * a.Hq * a.Lq + row_at;
      float* dst = a.nsplit > 1 ? a.po + pr * a.D  // the row as it stands, for attn_join_kernel
                                : static_cast<float*>(a.out) + (((long long)b * a.Lq + i) * a.Hq + h) * a.D;
#pragma unroll
      for (int c = 0; c < 64; c += 4)
        if (c < a.D) {
          float u[4];
          split2(o[c / 2], u[0], u[1]);
          split2(o[c / 2 + 1], u[2], u[3]);
#pragma unroll
          for (int k = 0; k < 4; ++k) u[k] = ok ? (f0 * u[k] + f1 * part[(c + k) * 128]) * inv : no_result();
          *reinterpret_cast<float4*>(dst + c) = make_float4(u[0], u[1], u[2], u[3]);
        }
      if (a.nsplit > 1) {
        a.pml[2 * pr] = M;
        a.pml[2 * pr + 1] = ok ? L : no_result();
      } else {
        a.lse[row_at] = ok ? row_lse(M, L) : no_result();
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 9) ptx::tmem_dealloc(tmem, 512);
}

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

// Heads whose parts TMA can address and three of whose tiles fit shared memory,
// enough queries to fill a tile of 128 more than half, and keys enough to pay for
// the splitting.
bool attn_tc_f32_fits(const AttnArgs& a) {
  return a.type == kF32 && a.D <= 64 && a.D % 8 == 0 && a.Lq >= 64 && a.Lk >= 64 &&
         reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
}

int64_t attn_tc_f32_workspace(const AttnArgs& a) {
  return up256(6ll * a.B * a.Lq * a.Hq * a.D) + 2 * up256(6ll * a.B * a.Lk * a.Hkv * a.D);
}

void attn_tc_f32_forward(const AttnArgs& a, void* ws, int sms, cudaStream_t st) {
  char* parts[3];
  parts[0] = static_cast<char*>(ws);
  parts[1] = parts[0] + up256(6ll * a.B * a.Lq * a.Hq * a.D);
  parts[2] = parts[1] + up256(6ll * a.B * a.Lk * a.Hkv * a.D);
  const void* src[3] = {a.q, a.k, a.v};
  const int64_t* s[3] = {a.qs, a.ks, a.vs};
  Maps maps;
  CUtensorMap* m[3] = {&maps.q, &maps.k, &maps.v};
  for (int i = 0; i < 3; ++i) {
    const int L = i ? a.Lk : a.Lq, H = i ? a.Hkv : a.Hq;
    const long long n = (long long)a.B * L * H * (a.D / 4);
    split_kernel<<<(unsigned)std::min<long long>((n + 255) / 256, 16ll * sms), 256, 0, st>>>(
        a, static_cast<const float*>(src[i]), s[i][0], s[i][1], s[i][2], L, H, i > 0, aligned16(a, src[i], s[i]),
        reinterpret_cast<uint2*>(parts[i]));
    note_launch();
    RVC_CUDA_TRY(cudaGetLastError());
    const int64_t ps[3] = {(int64_t)L * H * a.D, (int64_t)H * a.D, a.D};
    make_map(m[i], kBf16, parts[i], ps, 3 * a.B, L, H, a.D, i ? 64 : 128);
  }
  static std::atomic<uint64_t> done{0};  // one bit per device
  int dev = 0;
  RVC_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !(done.load() & (1ull << dev))) {
    RVC_CUDA_TRY(cudaFuncSetAttribute(attn_tc_f32_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    if (dev < 64) done.fetch_or(1ull << dev);
  }
  attn_tc_f32_kernel<<<dim3((unsigned)((a.Lq + 127ll) / 128 * a.B * a.Hq), a.nsplit), kThreads, kSmem, st>>>(a, maps);
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
  attn_join(a, st);
}

}  // namespace rvc
