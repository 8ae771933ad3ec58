// Gradients of attention on the fifth-generation tensor cores (16-bit inputs).
//
// Two kernels of one build, each deterministic (no sum crosses blocks):
//   first   dQ of 128 queries, keys passing by;
//   second  dK, dV of 128 keys of one KV head, queries of its group passing by.
// Both hold a resident pair X1, X2 and stream pairs Y1, Y2 (first: X = Q, dO and
// Y = K, V; second: X = K, V and Y = Q, dO) and form, per tile of 128 x 128,
//   S = X1 Y1^T, dP = X2 Y2^T           (fp32 in tensor memory)
//   P = 2^(scale S + bias - lse), dS = P (dP - delta)   (eight warps)
//   first:  A1 += dS K, A2 += P K       second: A1 += dS^T Q, A2 += P^T dO
// with P and dS read from tensor memory as 16-bit pairs over the columns of S
// and dP.  The tensor pipe runs in the order S dP | A2 S' | A1 dP' ..., so the
// products of the next tile run while the warps work on this one.  Seven
// products instead of the five of a single kernel, against no atomics and no
// fp32 copy of dQ in memory.
//
// delta = sum_j P dP is wanted to more than the 16 bits that dO . out gives
// (where the softmax is narrow, or summed over a wide bucket of the bias, dP -
// delta cancels): the first kernel starts from t = dO . out and sums
// r = sum_j P (dP - t) beside its products.  As sum P = 1, delta = t + r and
// dQ = scale (A1 - r A2): exact to fp32 for one product more.  It leaves delta
// and lse, padded to whole tiles, for the second kernel.
//
// The table's gradient is taken in the second kernel from the fp32 dS: a lane
// holds one key, and the running sum of a diagonal moves one lane up with every
// query, so a diagonal's part in a warp costs one shuffle and one addition per
// entry.  Tiles that lie whole in the last bucket are summed without diagonals.
#include "attn_tc.cuh"
#include "context.cuh"

#include <algorithm>
#include <atomic>

namespace rvc {

namespace {

using namespace atc;

constexpr int kBwdThreads = 320;
constexpr int kDiagLd = 96;  // diagonals of one warp's 32 x 64 part: 95

struct BwdMaps {
  CUtensorMap x1, x2, y1, y2;
};

// Tiles that pass by under way: as in the forward pass.
template <int NS> constexpr int kRing = NS == 1 ? 4 : 2;

// X1 X2 [NS], Y1 Y2 [stages][NS] slabs; per stage bias [256], lse [128],
// delta [128]; diagonals [8][96], carry [128]; row exchange [2][128]; barriers
template <int NS> constexpr uint32_t bwd_smem() {
  return (2 + 2 * kRing<NS>) * NS * kSlab + kRing<NS> * 512 * 4 + 8 * kDiagLd * 4 + 128 * 4 + 256 * 4 + 256 + 1024;
}

template <typename T, int NS, bool KV>
__global__ void __launch_bounds__(kBwdThreads, 1)
    attn_tc_bwd_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ BwdMaps maps) {
  constexpr int R = kRing<NS>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (ptx::smem_u32(raw) + 1023) & ~1023u;
  uint8_t* gen = raw + (base - ptx::smem_u32(raw));
  const uint32_t sX1 = base, sX2 = sX1 + NS * kSlab, sY1 = sX2 + NS * kSlab, sY2 = sY1 + R * NS * kSlab;
  const uint32_t oE = (2 + 2 * R) * NS * kSlab;  // extras of the stages
  float* ext = reinterpret_cast<float*>(gen + oE);
  float* diag_s = ext + R * 512;
  float* carry = diag_s + 8 * kDiagLd;
  float* red = carry + 128;
  const uint32_t oBar = oE + (R * 512 + 8 * kDiagLd + 128 + 256) * 4;
  const uint32_t bar = base + oBar;
  const uint32_t X_FULL = bar, Y1_FULL = bar + 8, Y2_FULL = Y1_FULL + 8 * R, Y1_EMPTY = Y2_FULL + 8 * R,
                 Y2_EMPTY = Y1_EMPTY + 8 * R, S_FULL = Y2_EMPTY + 8 * R, DP_FULL = S_FULL + 8, P_READY = S_FULL + 16,
                 DS_READY = S_FULL + 24, DONE = S_FULL + 32;
  uint32_t* slot = reinterpret_cast<uint32_t*>(gen + oBar + 192);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int G = a.Hq / a.Hkv;
  const int nq = (a.Lq + 127) / 128;
  const int ntile = KV ? (a.Lk + 127) / 128 : nq;
  const int heads = KV ? a.Hkv : a.Hq;
  // with a causal limit the longest walks come first: late queries, early keys
  const int xt = a.causal && !KV ? ntile - 1 - (int)(blockIdx.x % ntile) : (int)(blockIdx.x % ntile);
  const int bh = blockIdx.x / ntile, b = bh / heads, hx = bh % heads;
  const int kh = KV ? hx : hx / G;
  const int x0 = xt * 128;
  const int len = kv_len(a, b);
  // tiles that pass by: first: keys [0, kend); second: queries from `first` on, head by head
  int first = 0, per = 0, tiles = 0;
  if (KV) {
    if (a.causal) first = (int)(max(0ll, min((long long)a.Lq, (long long)x0 - a.q_off)) / 128);
    per = x0 < len ? max(0, nq - first) : 0;
    tiles = per * G;
  } else {
    long long kend = len;
    if (a.causal) kend = max(0ll, min(kend, (long long)min(a.Lq, x0 + 128) + a.q_off));
    tiles = (int)((kend + 127) / 128);
  }
  const bool extras = KV || a.diag;

  if (threadIdx.x == 0) {
    ptx::mbar_init(X_FULL, 1);
    for (int s = 0; s < R; ++s) {
      ptx::mbar_init(Y1_FULL + 8 * s, 1);
      ptx::mbar_init(Y2_FULL + 8 * s, 1);
      ptx::mbar_init(Y1_EMPTY + 8 * s, extras ? 9 : 1);
      ptx::mbar_init(Y2_EMPTY + 8 * s, 1);
    }
    ptx::mbar_init(S_FULL, 1);
    ptx::mbar_init(DP_FULL, 1);
    ptx::mbar_init(P_READY, 8);
    ptx::mbar_init(DS_READY, 8);
    ptx::mbar_init(DONE, 1);
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
  const uint32_t tS = tmem, tD = tmem + 128, tA1 = tmem + 256, tA2 = tA1 + 64 * NS;
  const int Lp = nq * 128;  // padded rows of lse and delta

  if (warp == 8) {
    if (lane == 0 && tiles > 0) {
      ptx::mbar_expect_tx(X_FULL, 2 * NS * kSlab);
      for (int s = 0; s < NS; ++s) {
        ptx::tma_load_4d(sX1 + s * kSlab, &maps.x1, 64 * s, hx, x0, b, X_FULL);
        ptx::tma_load_4d(sX2 + s * kSlab, &maps.x2, 64 * s, hx, x0, b, X_FULL);
      }
      int n1 = 0, n2 = 0;  // tiles asked for
      bool ok = true;
      for (int t = 0; t < tiles; ++t) {
        const int st = t % R;
        const uint32_t ph = ((t / R) & 1) ^ 1;
        const int hy = KV ? kh * G + t / per : kh;
        const int y0 = KV ? (first + t % per) * 128 : t * 128;
        ok = bar_wait(Y1_EMPTY + 8 * st, ph);
        if (!ok) break;
        ptx::mbar_expect_tx(Y1_FULL + 8 * st, NS * kSlab + (a.diag ? 1024 : 0) + (KV ? 1024 : 0));
        for (int s = 0; s < NS; ++s)
          ptx::tma_load_4d(sY1 + (st * NS + s) * kSlab, &maps.y1, 64 * s, hy, y0, b, Y1_FULL + 8 * st);
        const uint32_t e = base + oE + st * 2048;
        if (a.diag) {
          const int h = KV ? hy : hx;
          const int d = KV ? x0 - y0 - 128 : y0 - x0 - 128;
          ptx::bulk_g2s(e, a.diag + h * a.diag_ld + (d + a.diag0), 1024, Y1_FULL + 8 * st);
        }
        if (KV) {
          const int64_t r = ((int64_t)b * a.Hq + hy) * Lp + y0;
          ptx::bulk_g2s(e + 1024, a.lse2 + r, 512, Y1_FULL + 8 * st);
          ptx::bulk_g2s(e + 1536, a.delta + r, 512, Y1_FULL + 8 * st);
        }
        n1 = t + 1;
        ok = bar_wait(Y2_EMPTY + 8 * st, ph);
        if (!ok) break;
        ptx::mbar_expect_tx(Y2_FULL + 8 * st, NS * kSlab);
        for (int s = 0; s < NS; ++s)
          ptx::tma_load_4d(sY2 + (st * NS + s) * kSlab, &maps.y2, 64 * s, hy, y0, b, Y2_FULL + 8 * st);
        n2 = t + 1;
      }
      if (!ok) atomicExch(a.err, 51);
      bar_wait(X_FULL, 0);  // no copy left in flight when the block ends
      for (int x = max(0, n1 - R); x < n1; ++x) bar_wait(Y1_FULL + 8 * (x % R), (x / R) & 1);
      for (int x = max(0, n2 - R); x < n2; ++x) bar_wait(Y2_FULL + 8 * (x % R), (x / R) & 1);
    }
    __syncwarp();
  } else if (warp == 9) {
    if (lane == 0 && tiles > 0) {
      const int DK = (a.D + 15) / 16;
      const uint32_t id_s = idesc<T>(128, false, false), id_a = idesc<T>(16 * DK, false, true);
      bool ok = bar_wait(X_FULL, 0);
      auto abt = [&](uint32_t d, uint32_t x, uint32_t y) {
        const uint64_t dx = desc_k(x), dy = desc_k(y);
#pragma unroll
        for (int kk = 0; kk < 4 * NS; ++kk) {
          if (kk >= DK) break;
          const uint64_t off = (uint64_t)(((kk >> 2) * kSlab + (kk & 3) * 32) >> 4);
          mma_ss(d, dx + off, dy + off, id_s, kk > 0);
        }
      };
      auto pb = [&](uint32_t d, uint32_t p, uint32_t y, bool acc) {
        const uint64_t dy = desc_mn(y);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          mma_ts(d, p + 64 * (kk >> 2) + 8 * (kk & 3), dy + (uint64_t)(kk * 2048 >> 4), id_a, acc || kk > 0);
      };
      auto issue_s = [&](int t) {
        const int st = t % R;
        if (ok) ok = bar_wait(Y1_FULL + 8 * st, (t / R) & 1);
        if (!ok) return;
        ptx::tc_fence_after();
        abt(tS, sX1, sY1 + st * NS * kSlab);
        ptx::mma_commit(S_FULL);
      };
      auto issue_dp = [&](int t) {
        const int st = t % R;
        if (ok) ok = bar_wait(Y2_FULL + 8 * st, (t / R) & 1);
        if (!ok) return;
        ptx::tc_fence_after();
        abt(tD, sX2, sY2 + st * NS * kSlab);
        ptx::mma_commit(DP_FULL);
        if (!KV) ptx::mma_commit(Y2_EMPTY + 8 * st);
      };
      issue_s(0);
      issue_dp(0);
      for (int t = 0; t < tiles && ok; ++t) {
        const int st = t % R;
        if (ok) ok = bar_wait(P_READY, t & 1);
        if (!ok) break;
        ptx::tc_fence_after();
        pb(tA2, tS, (KV ? sY2 : sY1) + st * NS * kSlab, t > 0);
        if (KV) ptx::mma_commit(Y2_EMPTY + 8 * st);
        if (t + 1 < tiles) issue_s(t + 1);
        if (ok) ok = bar_wait(DS_READY, t & 1);
        if (!ok) break;
        ptx::tc_fence_after();
        pb(tA1, tD, sY1 + st * NS * kSlab, t > 0);
        ptx::mma_commit(Y1_EMPTY + 8 * st);
        if (t + 1 < tiles) issue_dp(t + 1);
      }
      if (!ok) atomicExch(a.err, 52);
      ptx::mma_commit(DONE);
      bar_wait(DONE, 0);  // every product done before tensor memory is freed
    }
    __syncwarp();
  } else {
    const int hf = warp >> 2, row = threadIdx.x & 127;  // columns 64 hf .. 64 hf + 63 of row `row`
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tS + 64 * hf + lanes, d_col = tD + 64 * hf + lanes;
    const float sc = a.scale * kLog2e;
    const uint8_t* mb = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
    const long long x = (long long)x0 + row;  // this row's query (first) or key (second)
    bool ok = true;
    // first: this row's lse and t = dO . out, each half sums half of the values
    float lse2 = INFINITY, t0 = 0.f, r = 0.f;
    bool dead = false;  // second: this row's key
    if (!KV) {
      const bool in = x < a.Lq;
      const T* go = static_cast<const T*>(a.dout) + (int64_t)b * a.dos[0] + x * a.dos[1] + (int64_t)hx * a.dos[2];
      const T* fo = static_cast<const T*>(a.fout) + (int64_t)b * a.os[0] + x * a.os[1] + (int64_t)hx * a.os[2];
      if (in) {
        const float z = a.lse[((int64_t)b * a.Hq + hx) * a.Lq + x];
        lse2 = z == -INFINITY ? INFINITY : z * kLog2e;
        for (int d = 8 * hf; d < a.D; d += 16) {
          const uint4 u = *reinterpret_cast<const uint4*>(go + d), v = *reinterpret_cast<const uint4*>(fo + d);
          const T *pu = reinterpret_cast<const T*>(&u), *pv = reinterpret_cast<const T*>(&v);
#pragma unroll
          for (int c = 0; c < 8; ++c) t0 = fmaf(to_f(pu[c]), to_f(pv[c]), t0);
        }
      }
      red[128 * hf + row] = t0;
      ptx::named_bar(1, 256);
      t0 = red[row] + red[128 + row];
      ptx::named_bar(1, 256);
    } else {
      dead = x >= len || (mb && !mb[x * a.mask_k]);
      if (a.dws && threadIdx.x < 128) carry[threadIdx.x] = 0.f;
    }
    float far_behind = 0.f, far_ahead = 0.f;
    for (int t = 0; t < tiles; ++t) {
      const int st = t % R;
      const int y0 = KV ? (first + t % per) * 128 : t * 128;
      const float* e = ext + st * 512;
      uint32_t alive[2] = {~0u, ~0u};  // first: keys of this half
      if (!KV && mb) {
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int j = y0 + 64 * hf + 32 * z + lane;
          alive[z] = __ballot_sync(0xffffffffu, j < len && mb[(int64_t)j * a.mask_k] != 0);
        }
      }
      float p[64];
      do {  // a wait that gives up leaves the tile; the warps meet again below
        if (extras && !(ok = warp_wait(Y1_FULL + 8 * st, (t / R) & 1))) break;
        if (!(ok = warp_wait(S_FULL, t & 1))) break;
        ptx::tc_fence_after();
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          uint32_t s[32];
          ptx::tmem_ld32_async(s_col + 32 * z, s);
          ptx::tmem_wait_ld(s);
          if (KV) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 l4 = *reinterpret_cast<const float4*>(e + 256 + 64 * hf + 32 * z + c);
              p[32 * z + c] = -l4.x, p[32 * z + c + 1] = -l4.y, p[32 * z + c + 2] = -l4.z, p[32 * z + c + 3] = -l4.w;
            }
            if (a.diag) {
              const float* bb = e + 128 + row - 64 * hf - 32 * z;
#pragma unroll
              for (int c = 0; c < 32; ++c) p[32 * z + c] += bb[-c];
            }
          } else if (a.diag) {
            const float* bb = e + 128 - row + 64 * hf + 32 * z;
#pragma unroll
            for (int c = 0; c < 32; ++c) p[32 * z + c] = bb[c] - lse2;
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) p[32 * z + c] = -lse2;
          }
#pragma unroll
          for (int c = 0; c < 32; ++c) p[32 * z + c] = exp2_approx(fmaf(__uint_as_float(s[c]), sc, p[32 * z + c]));
        }
        if (KV) {
          // causal: queries c of this half with y0 + 64 hf + c + q_off < key are out
          const long long lo = a.causal ? x - a.q_off - y0 - 64 * hf : 0;
          if (dead || lo > 0) {
            const int n = dead ? 64 : (int)min(64ll, lo);
#pragma unroll
            for (int c = 0; c < 64; ++c) p[c] = c < n ? 0.f : p[c];
          }
        } else {
          const long long lim = (a.causal ? min((long long)len, x + a.q_off + 1) : (long long)len) - y0 - 64 * hf;
          if (mb || lim < 64) {
            const int n = (int)max(0ll, min(64ll, lim));
#pragma unroll
            for (int c = 0; c < 64; ++c) p[c] = c < n && ((alive[c >> 5] >> (c & 31)) & 1) ? p[c] : 0.f;
          }
          if (mb || y0 + 128 > len) {  // zero the dead rows of K: both halves' threads take half of the slabs
            const int j = y0 + row;
            if (j >= len || (mb && !mb[(int64_t)j * a.mask_k])) {
              uint4* zr = reinterpret_cast<uint4*>(gen + 2 * NS * kSlab + st * NS * kSlab + row * 128);
#pragma unroll
              for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int c = 0; c < 4; ++c) zr[s * (kSlab / 16) + 4 * hf + c] = make_uint4(0, 0, 0, 0);
            }
            ptx::fence_proxy_async_smem();
          }
        }
        {
          uint32_t w[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) w[c] = pack2<T>(p[2 * c], p[2 * c + 1]);
          tmem_st32(s_col, w);
        }
        tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(P_READY);

        if (!(ok = warp_wait(DP_FULL, t & 1))) break;
        ptx::tc_fence_after();
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          uint32_t s[32];
          ptx::tmem_ld32_async(d_col + 32 * z, s);
          ptx::tmem_wait_ld(s);
          if (KV) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 d4 = *reinterpret_cast<const float4*>(e + 384 + 64 * hf + 32 * z + c);
              const float dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                float& q = p[32 * z + c + k];
                q = q != 0.f ? q * (__uint_as_float(s[c + k]) - dd[k]) : 0.f;
              }
            }
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              float& q = p[32 * z + c];
              q = q != 0.f ? q * (__uint_as_float(s[c]) - t0) : 0.f;
              r += q;
            }
          }
        }
        {
          uint32_t w[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) w[c] = pack2<T>(p[2 * c], p[2 * c + 1]);
          tmem_st32(d_col, w);
        }
        tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(DS_READY);
          if (extras) ptx::mbar_arrive(Y1_EMPTY + 8 * st);
        }
      } while (false);
      // the named barriers below are taken by all warps or by none
      if (KV && a.dws) ok = ptx::named_bar_and(1, 256, ok);
      if (!ok) break;
      if (KV && a.dws) {
        const int hy = kh * G + t / per, tq = t % per;
        float* dws = a.dws + (((int64_t)b * a.Hq + hy) * ntile + xt) * a.dws_ld;
        // relative positions of the tile: [hi - 254, hi]
        const long long hi = (long long)x0 + 127 - y0 - a.q_off;
        const bool behind = hi <= -(long long)a.far, ahead = hi - 254 >= (a.far_both ? (long long)a.far : 0ll);
        const int u = threadIdx.x;  // diagonal key - query = 127 - u within the tile, u < 255
        float v = 0.f;
        if (behind || ahead) {
          float s = 0.f;
#pragma unroll
          for (int c = 0; c < 64; ++c) s += p[c];
          if (behind) far_behind += s;
          else far_ahead += s;
        } else {
          float acc = 0.f;
          float* mine = diag_s + warp * kDiagLd;
#pragma unroll
          for (int c = 0; c < 64; ++c) {
            acc += p[c];
            if (lane == 31) mine[c] = acc;  // diagonal lane - column = 31 - c is whole
            const float up = __shfl_up_sync(0xffffffffu, acc, 1);
            if (c < 63) acc = lane == 0 ? 0.f : up;
          }
          if (lane < 31) mine[94 - lane] = acc;  // lane - 63
          ptx::named_bar(1, 256);
          if (u < 255) {
#pragma unroll
            for (int w = 0; w < 8; ++w) {
              // rows 32 (w & 3) + lane, columns 64 (w >> 2) + c: entry 31 - (lane - c)
              const int k = 31 - ((127 - u) - 32 * (w & 3) + 64 * (w >> 2));
              if (k >= 0 && k < 95) v += diag_s[w * kDiagLd + k];
            }
          }
        }
        // u <= 127 (key - query >= 0) is whole with this tile, the others go on in the next
        if (u < 128) dws[(int64_t)(first + tq) * 128 + u] = v + carry[u];
        ptx::named_bar(1, 256);
        if (u >= 128 && u < 256) carry[u - 128] = u < 255 ? v : 0.f;
        ptx::named_bar(1, 256);
        if (tq + 1 == per) {  // a head ends: its open diagonals, and zeros where no tile was
          const int64_t end = (int64_t)(first + per) * 128;
          for (int64_t z = u; z < a.dws_ld - 2; z += 256)
            if (z < (int64_t)first * 128 || z >= end) dws[z] = z >= end && z < end + 128 ? carry[z - end] : 0.f;
          const float fb = far_behind, fa = far_ahead;
          red[u] = fb;
          ptx::named_bar(1, 256);
          if (u == 0) {
            float s = 0.f;
            for (int z = 0; z < 256; ++z) s += red[z];
            dws[a.dws_ld - 2] = s;
          }
          ptx::named_bar(1, 256);
          red[u] = fa;
          ptx::named_bar(1, 256);
          if (u == 0) {
            float s = 0.f;
            for (int z = 0; z < 256; ++z) s += red[z];
            dws[a.dws_ld - 1] = s;
          }
          far_behind = far_ahead = 0.f;
          if (u < 128) carry[u] = 0.f;
          ptx::named_bar(1, 256);
        }
      }
    }
    if (KV && a.dws && tiles == 0) {
      for (int g = 0; g < G; ++g) {
        float* dws = a.dws + (((int64_t)b * a.Hq + kh * G + g) * ntile + xt) * a.dws_ld;
        for (int64_t z = threadIdx.x; z < a.dws_ld; z += 256) dws[z] = 0.f;
      }
    }
    if (ok && tiles > 0) ok = warp_wait(DONE, 0);
    ptx::tc_fence_after();
    if (!ok) {
      if (lane == 0) atomicExch(a.err, 53);
    }
    float rr = 0.f;
    if (!KV) {
      // every warp comes here, also after a wait that gave up
      red[128 * hf + row] = r;
      ptx::named_bar(1, 256);
      rr = red[row] + red[128 + row];
      if (hf == 0) {
        const int64_t at = ((int64_t)b * a.Hq + hx) * Lp + x;
        a.lse2[at] = lse2;
        a.delta[at] = lse2 == INFINITY ? 0.f : t0 + rr;
      }
    }
    if (ok) {
      const int L = KV ? a.Lk : a.Lq;
      const int64_t at = (((int64_t)b * L + x) * heads + hx) * a.D;
      T* d1 = static_cast<T*>(KV ? a.dk : a.dq) + at;
      T* d2 = static_cast<T*>(a.dv) + at;
#pragma unroll 1
      for (int c0 = 32 * NS * hf; c0 < 32 * NS * (hf + 1); c0 += 16) {
        if (c0 >= a.D) break;
        float u[16], v[16];
        if (tiles > 0) {
          ptx::tmem_ld16(tA1 + lanes + c0, u);
          ptx::tmem_ld16(tA2 + lanes + c0, v);
        } else {
#pragma unroll
          for (int c = 0; c < 16; ++c) u[c] = v[c] = 0.f;
        }
        if (x >= L) continue;
#pragma unroll
        for (int c = 0; c < 16; ++c) u[c] = a.scale * (KV ? u[c] : u[c] - rr * v[c]);
#pragma unroll
        for (int c = 0; c < 16; c += 8)
          if (c0 + c < a.D) {
            *reinterpret_cast<uint4*>(d1 + c0 + c) = make_uint4(pack2<T>(u[c], u[c + 1]), pack2<T>(u[c + 2], u[c + 3]),
                                                                pack2<T>(u[c + 4], u[c + 5]), pack2<T>(u[c + 6], u[c + 7]));
            if (KV)
              *reinterpret_cast<uint4*>(d2 + c0 + c) = make_uint4(pack2<T>(v[c], v[c + 1]), pack2<T>(v[c + 2], v[c + 3]),
                                                                  pack2<T>(v[c + 4], v[c + 5]), pack2<T>(v[c + 6], v[c + 7]));
          }
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 9) ptx::tmem_dealloc(tmem, 512);
}

template <typename T, int NS, bool KV>
void launch(const AttnArgs& a, const BwdMaps& maps, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};  // one bit per device
  int dev = 0;
  RVC_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !(done.load() & (1ull << dev))) {
    RVC_CUDA_TRY(cudaFuncSetAttribute(attn_tc_bwd_kernel<T, NS, KV>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)bwd_smem<NS>()));
    if (dev < 64) done.fetch_or(1ull << dev);
  }
  const unsigned grid = KV ? (unsigned)((a.Lk + 127ll) / 128 * a.B * a.Hkv) : (unsigned)((a.Lq + 127ll) / 128 * a.B * a.Hq);
  attn_tc_bwd_kernel<T, NS, KV><<<grid, kBwdThreads, bwd_smem<NS>(), st>>>(a, maps);
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
}

template <typename T, int NS>
void bwd(const AttnArgs& a, cudaStream_t st) {
  BwdMaps m;
  make_map(&m.x1, a.type, a.q, a.qs, a.B, a.Lq, a.Hq, a.D, 128);
  make_map(&m.x2, a.type, a.dout, a.dos, a.B, a.Lq, a.Hq, a.D, 128);
  make_map(&m.y1, a.type, a.k, a.ks, a.B, a.Lk, a.Hkv, a.D, 128);
  make_map(&m.y2, a.type, a.v, a.vs, a.B, a.Lk, a.Hkv, a.D, 128);
  launch<T, NS, false>(a, m, st);
  std::swap(m.x1, m.y1);
  std::swap(m.x2, m.y2);
  launch<T, NS, true>(a, m, st);
}

}  // namespace

bool attn_tc_bwd_fits(const AttnArgs& a) {
  const auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  return a.type != kF32 && a.Lq >= 64 && a.Lk >= 64 && map_ok(a, a.q, a.qs, a.Lq, a.Hq) &&
         map_ok(a, a.k, a.ks, a.Lk, a.Hkv) && map_ok(a, a.v, a.vs, a.Lk, a.Hkv) &&
         map_ok(a, a.dout, a.dos, a.Lq, a.Hq) && map_ok(a, a.fout, a.os, a.Lq, a.Hq) && al(a.dq) && al(a.dk) && al(a.dv);
}

void attn_tc_backward(const AttnArgs& a, cudaStream_t st) {
  if (a.type == kBf16) {
    if (a.D <= 64) bwd<__nv_bfloat16, 1>(a, st);
    else bwd<__nv_bfloat16, 2>(a, st);
  } else {
    if (a.D <= 64) bwd<__half, 1>(a, st);
    else bwd<__half, 2>(a, st);
  }
}

}  // namespace rvc
