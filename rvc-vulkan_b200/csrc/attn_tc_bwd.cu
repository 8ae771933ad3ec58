// Gradients of attention on the fifth-generation tensor cores (16-bit inputs).
//
// Two kernels of one build, each with its sums in a fixed order:
//   first   dQ of 128 queries, keys passing by;
//   second  dK, dV of 128 keys of one KV head, queries of its group passing by;
//           where key tiles are few, the group's heads are shared out to blocks
//           and kv_join_kernel adds the shares in order.
// Both hold a resident pair X1, X2 and stream pairs Y1, Y2 (first: X = Q, dO and
// Y = K, V; second: X = K, V and Y = Q, dO) and form, per tile of 128 rows of X
// and 64 of Y,
//   S = X1 Y1^T, dP = X2 Y2^T           (fp32 in tensor memory)
//   P = 2^(scale S + bias - lse), dS = P (dP - delta)
//   first:  A1 += dS K, A2 += P K       second: A1 += dS^T Q, A2 += P^T dO
// with P and dS read from tensor memory as 16-bit pairs over the columns of S
// and dP, one row to a thread of a group of four warps.  The tensor pipe runs in
// the order
//   A2(t) S(t + GR) | A1(t - GR + 1) dP(t + 1)
// where GR = 1 or 2 groups take the tiles in turn, each with its own S and dP.
// Heads of up to 64 values have one group and half of the tensor memory, so that
// two blocks share an SM: one's start and end (5 to 8 us, as long as four tiles)
// and its exponentials go on beside the other's products.  Longer heads fill the
// tensor memory and have two groups.  Seven products instead of the five of a
// single kernel, against no atomics and no fp32 copy of dQ in memory.
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
//
// Measured: 8 x 12 x 251 x 1499 x 64 with a mask, bf16: 123 us; causal 4 x 16 x 2048
// x 64 with the table's gradient: 412 us.  The chain S, P, dS of a tile and the
// start and end of short blocks bound it: captured alone, the tensor pipe is busy
// 19 % (first kernel) and 15 % (second) of the one, 26 and 18 % of the other.
#include "attn_tc.cuh"
#include "context.cuh"

#include <algorithm>
#include <atomic>

namespace rvc {

namespace {

using namespace atc;

template <int NS> constexpr int kGroups = NS == 1 ? 1 : 2;
template <int NS> constexpr int kBwdThreads = 128 * kGroups<NS> + 64;
constexpr int kDiagLd = 96;          // diagonals of one warp's 32 x 64 part: 95
constexpr uint32_t kHalf = kSlab / 2;  // a slab of 64 rows
constexpr int R = 4;                 // Y tiles under way

struct BwdMaps {
  CUtensorMap x1, x2, y1, y2;
};

// X1 X2 [NS] slabs, Y1 Y2 [R][NS] slabs of 64 rows; per stage bias [192], -lse
// [64], -delta [64]; diagonals [4 GR warps][96], open diagonals [128]; barriers
constexpr uint32_t kExt = 320;
template <int NS> constexpr uint32_t bwd_smem() {
  return 2 * NS * kSlab + 2 * R * NS * kHalf + (R * kExt + 4 * kGroups<NS> * kDiagLd + 128) * 4 + 512 + 1024;
}

template <typename T, int NS, bool KV, bool FULL>
__global__ void __launch_bounds__(kBwdThreads<NS>, NS == 1 ? 2 : 1)
    attn_tc_bwd_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ BwdMaps maps) {
  constexpr int GR = kGroups<NS>;
  constexpr int kLoad = 4 * GR, kIssue = 4 * GR + 1;  // warps
  constexpr int kStep = 64 * GR, kOpen = 192 - kStep;  // diagonals that a group's tile closes, and leaves open
  extern __shared__ uint8_t raw[];
  const uint32_t base = (ptx::smem_u32(raw) + 1023) & ~1023u;
  uint8_t* gen = raw + (base - ptx::smem_u32(raw));
  constexpr uint32_t oY1 = 2 * NS * kSlab, oY2 = oY1 + R * NS * kHalf, oE = oY2 + R * NS * kHalf;
  constexpr uint32_t oBar = oE + (R * kExt + 4 * kGroups<NS> * kDiagLd + 128) * 4;
  const uint32_t sX1 = base, sX2 = sX1 + NS * kSlab, sY1 = base + oY1, sY2 = base + oY2;
  float* ext = reinterpret_cast<float*>(gen + oE);
  float* diag_s = ext + R * kExt;
  float* carry = diag_s + 4 * GR * kDiagLd;
  const uint32_t bar = base + oBar;
  const uint32_t X_FULL = bar, Y1_FULL = bar + 8, Y2_FULL = Y1_FULL + 8 * R, Y1_EMPTY = Y2_FULL + 8 * R,
                 Y2_EMPTY = Y1_EMPTY + 8 * R, S_FULL = Y2_EMPTY + 8 * R /* [2 groups] each from here */,
                 DP_FULL = S_FULL + 16, P_READY = S_FULL + 32, DS_READY = S_FULL + 48, DONE = S_FULL + 64;
  uint32_t* slot = reinterpret_cast<uint32_t*>(gen + oBar + 504);
  volatile uint32_t* undone = slot + 1;  // products that were not issued, set before DONE
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int group = a.Hq / a.Hkv;
  const int ny = KV ? (a.Lq + 63) / 64 : 0;  // second: query tiles of a head
  const int ntile = KV ? (a.Lk + 127) / 128 : (a.Lq + 127) / 128;
  const int heads = KV ? a.Hkv : a.Hq;
  // with a causal limit the longest walks come first: late queries, early keys
  const int xt = a.causal && !KV ? ntile - 1 - (int)(blockIdx.x % ntile) : (int)(blockIdx.x % ntile);
  const int bh = blockIdx.x / ntile, b = bh / heads, hx = bh % heads;
  const int kh = KV ? hx : hx / group;
  // second: the query heads of this share of the group, h0 .. h0 + G - 1
  const int g0 = KV ? group * (int)blockIdx.y / a.nsplit : 0;
  const int G = KV ? group * ((int)blockIdx.y + 1) / a.nsplit - g0 : 1, h0 = kh * group + g0;
  const int x0 = xt * 128;
  const int len = kv_len(a, b);
  // tiles that pass by: first: keys [0, kend); second: queries from `first` on, head by head
  int first = 0, per = 0, tiles = 0;
  if (KV) {
    if (a.causal) first = (int)(max(0ll, min((long long)a.Lq, (long long)x0 - a.q_off)) / 64);
    per = x0 < len ? max(0, ny - first) : 0;
    tiles = per * G;
  } else {
    long long kend = len;
    if (a.causal) kend = max(0ll, min(kend, (long long)min(a.Lq, x0 + 128) + a.q_off));
    tiles = (int)((kend + 63) / 64);
  }
  const bool extras = KV || a.diag;

  if (threadIdx.x == 0) {
    ptx::mbar_init(X_FULL, 1);
    for (int s = 0; s < R; ++s) {
      ptx::mbar_init(Y1_FULL + 8 * s, 1);
      ptx::mbar_init(Y2_FULL + 8 * s, 1);
      ptx::mbar_init(Y1_EMPTY + 8 * s, extras ? 5 : 1);
      ptx::mbar_init(Y2_EMPTY + 8 * s, 1);
    }
    for (int w = 0; w < GR; ++w) {
      ptx::mbar_init(S_FULL + 8 * w, 1);
      ptx::mbar_init(DP_FULL + 8 * w, 1);
      ptx::mbar_init(P_READY + 8 * w, 4);
      ptx::mbar_init(DS_READY + 8 * w, 4);
    }
    ptx::mbar_init(DONE, 2);
    *undone = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kIssue) {
    ptx::tmem_alloc(ptx::smem_u32(slot), 256 * GR);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *slot;
  // S and dP of a group: 64 columns each at 128 w; A1, A2: 64 NS columns each
  const uint32_t tS = tmem, tD = tmem + 64, tA1 = tmem + 128 * GR, tA2 = tA1 + 64 * NS;
  const int Lp = (a.Lq + 127) / 128 * 128;  // padded rows of lse and delta

  if (warp == kLoad) {
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
        const int hy = KV ? h0 + t / per : kh;
        const int y0 = KV ? (first + t % per) * 64 : t * 64;
        ok = bar_wait(Y1_EMPTY + 8 * st, ph);
        if (!ok) break;
        ptx::mbar_expect_tx(Y1_FULL + 8 * st, NS * kHalf + (a.diag ? 768 : 0) + (KV ? 512 : 0));
        for (int s = 0; s < NS; ++s)
          ptx::tma_load_4d(sY1 + (st * NS + s) * kHalf, &maps.y1, 64 * s, hy, y0, b, Y1_FULL + 8 * st);
        const uint32_t e = base + oE + st * kExt * 4;
        if (a.diag) {
          const int h = KV ? hy : hx;
          const int d = KV ? x0 - y0 - 64 : y0 - x0 - 128;
          ptx::bulk_g2s(e, a.diag + h * a.diag_ld + (d + a.diag0), 768, Y1_FULL + 8 * st);
        }
        if (KV) {
          const int64_t r = ((int64_t)b * a.Hq + hy) * Lp + y0;
          ptx::bulk_g2s(e + 768, a.lse2 + r, 256, Y1_FULL + 8 * st);
          ptx::bulk_g2s(e + 1024, a.delta + r, 256, Y1_FULL + 8 * st);
        }
        n1 = t + 1;
        ok = bar_wait(Y2_EMPTY + 8 * st, ph);
        if (!ok) break;
        ptx::mbar_expect_tx(Y2_FULL + 8 * st, NS * kHalf);
        for (int s = 0; s < NS; ++s)
          ptx::tma_load_4d(sY2 + (st * NS + s) * kHalf, &maps.y2, 64 * s, hy, y0, b, Y2_FULL + 8 * st);
        n2 = t + 1;
      }
      if (!ok) atomicExch(a.err, 51);
      bar_wait(X_FULL, 0);  // no copy left in flight when the block ends
      for (int x = max(0, n1 - R); x < n1; ++x) bar_wait(Y1_FULL + 8 * (x % R), (x / R) & 1);
      for (int x = max(0, n2 - R); x < n2; ++x) bar_wait(Y2_FULL + 8 * (x % R), (x / R) & 1);
    }
    __syncwarp();
  } else if (warp == kIssue) {
    if (lane == 0 && tiles > 0) {
      const int DK = FULL ? 4 * NS : (a.D + 15) / 16;
      const uint32_t id_s = idesc<T>(64, false, false), id_a = idesc<T>(16 * DK, false, true);
      bool ok = bar_wait(X_FULL, 0);
      auto abt = [&](uint32_t d, uint32_t x, uint32_t y) {
        const uint64_t dx = desc_k(x), dy = desc_k(y);
#pragma unroll
        for (int kk = 0; kk < 4 * NS; ++kk) {
          if (kk >= DK) break;
          mma_ss(d, dx + (uint64_t)(((kk >> 2) * kSlab + (kk & 3) * 32) >> 4),
                 dy + (uint64_t)(((kk >> 2) * kHalf + (kk & 3) * 32) >> 4), id_s, kk > 0);
        }
      };
      auto pb = [&](uint32_t d, uint32_t p, uint32_t y, bool acc) {
        const uint64_t dy = desc_mn(y, kHalf);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) mma_ts(d, p + 8 * kk, dy + (uint64_t)(kk * 2048 >> 4), id_a, acc || kk > 0);
      };
      auto issue_s = [&](int t) {
        const int st = t % R;
        if (ok) ok = bar_wait(Y1_FULL + 8 * st, (t / R) & 1);
        if (!ok) return;
        ptx::tc_fence_after();
        abt(tS + 128 * (t % GR), sX1, sY1 + st * NS * kHalf);
        ptx::mma_commit(S_FULL + 8 * (t % GR));
      };
      auto issue_dp = [&](int t) {
        const int st = t % R;
        if (ok) ok = bar_wait(Y2_FULL + 8 * st, (t / R) & 1);
        if (!ok) return;
        ptx::tc_fence_after();
        abt(tD + 128 * (t % GR), sX2, sY2 + st * NS * kHalf);
        ptx::mma_commit(DP_FULL + 8 * (t % GR));
        if (!KV) ptx::mma_commit(Y2_EMPTY + 8 * st);
      };
      for (int t = 0; t < GR && t < tiles; ++t) issue_s(t);
      issue_dp(0);
      for (int t = 0; t < tiles + GR - 1 && ok; ++t) {
        if (t < tiles) {
          const int st = t % R;
          ok = bar_wait(P_READY + 8 * (t % GR), (t / GR) & 1);
          if (!ok) break;
          ptx::tc_fence_after();
          pb(tA2, tS + 128 * (t % GR), (KV ? sY2 : sY1) + st * NS * kHalf, t > 0);
          if (KV) ptx::mma_commit(Y2_EMPTY + 8 * st);
          if (t + GR < tiles) issue_s(t + GR);
        }
        const int u = t - (GR - 1);
        if (u >= 0) {
          const int st = u % R;
          if (ok) ok = bar_wait(DS_READY + 8 * (u % GR), (u / GR) & 1);
          if (!ok) break;
          ptx::tc_fence_after();
          pb(tA1, tD + 128 * (u % GR), sY1 + st * NS * kHalf, u > 0);
          ptx::mma_commit(Y1_EMPTY + 8 * st);
        }
        if (t + 1 < tiles) issue_dp(t + 1);
      }
      if (!ok) {
        atomicExch(a.err, 52);
        *undone = 1;
      }
      ptx::mma_commit(DONE);
      ptx::mbar_arrive(DONE);
      bar_wait(DONE, 0);  // every product done before tensor memory is freed
    }
    __syncwarp();
  } else {
    const int w = warp >> 2, row = threadIdx.x & 127;  // group, row of X
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tS + 128 * w + lanes, d_col = tD + 128 * w + lanes;
    const float sc = a.scale * kLog2e;
    const uint64_t sc2 = f32x2(sc, sc);
    const uint8_t* mb = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
    const long long x = (long long)x0 + row;  // this row's query (first) or key (second)
    bool ok = true;
    // first: this row's -lse and -t, t = dO . out (both groups form them)
    float nl = -INFINITY, nt = 0.f, r = 0.f;
    bool dead = false;  // second: this row's key
    if (!KV) {
      const T* go = static_cast<const T*>(a.dout) + (int64_t)b * a.dos[0] + x * a.dos[1] + (int64_t)hx * a.dos[2];
      const T* fo = static_cast<const T*>(a.fout) + (int64_t)b * a.os[0] + x * a.os[1] + (int64_t)hx * a.os[2];
      if (x < a.Lq) {
        const float z = a.lse[((int64_t)b * a.Hq + hx) * a.Lq + x];
        nl = z == -INFINITY ? -INFINITY : -z * kLog2e;  // a row without a key: P = 0
#pragma unroll 4
        for (int d = 0; d < a.D; d += 8) {
          const uint4 u = *reinterpret_cast<const uint4*>(go + d), v = *reinterpret_cast<const uint4*>(fo + d);
          const T *pu = reinterpret_cast<const T*>(&u), *pv = reinterpret_cast<const T*>(&v);
#pragma unroll
          for (int c = 0; c < 8; ++c) nt = fmaf(-to_f(pu[c]), to_f(pv[c]), nt);
        }
      }
    } else {
      dead = x >= len || (mb && !mb[x * a.mask_k]);
      if (a.dws && row < kOpen) carry[64 * w + row] = 0.f;
    }
    float far_behind = 0.f, far_ahead = 0.f;
    int64_t at = 0;  // second: first diagonal of this group's array that is not written yet
    // second: writes the end of a head's diagonals (the array of this group)
    auto end_head = [&](int hy) {
      float* dws = a.dws + ((((int64_t)b * a.Hq + hy) * ntile + xt) * GR + w) * a.dws_ld;
      ptx::named_bar(1 + w, 128);  // the last open diagonals are there
      for (int64_t z = at + row; z < a.dws_ld - 2; z += 128) dws[z] = z - at < kOpen ? carry[64 * w + (z - at)] : 0.f;
      // sums of the tiles whole in a last bucket: lanes, then the four warps in order
      float fb = far_behind, fa = far_ahead;
#pragma unroll
      for (int z = 16; z; z >>= 1) {
        fb += __shfl_xor_sync(0xffffffffu, fb, z);
        fa += __shfl_xor_sync(0xffffffffu, fa, z);
      }
      ptx::named_bar(1 + w, 128);
      if (lane == 0) {
        diag_s[warp * kDiagLd] = fb;
        diag_s[warp * kDiagLd + 1] = fa;
      }
      if (row < kOpen) carry[64 * w + row] = 0.f;
      ptx::named_bar(1 + w, 128);
      if (row < 2) {
        const float* f = diag_s + 4 * w * kDiagLd + row;
        dws[a.dws_ld - 2 + row] = ((f[0] + f[kDiagLd]) + f[2 * kDiagLd]) + f[3 * kDiagLd];
      }
      ptx::named_bar(1 + w, 128);
      far_behind = far_ahead = 0.f;
      at = 0;
    };
    int head = 0;  // second: heads of the group whose diagonals are written
    uint8_t byte0 = 0, byte1 = 0;  // first: mask of keys `lane` and 32 + `lane` of this group's next tile
    auto fetch = [&](int y0) {
      byte0 = y0 + lane < len ? mb[(int64_t)(y0 + lane) * a.mask_k] : 0;
      byte1 = y0 + 32 + lane < len ? mb[(int64_t)(y0 + 32 + lane) * a.mask_k] : 0;
    };
    if (!KV && mb) fetch(64 * w);
    const int lone = tiles > 0 ? lone_queries(a, b, len) : 0;  // queries whose dS is zero: the first ones
    for (int t = w; t < tiles; t += GR) {
      const int st = t % R;
      const uint32_t turn = (t / GR) & 1;
      const int y0 = KV ? (first + t % per) * 64 : t * 64;
      const float* e = ext + st * kExt;
      if (KV && a.dws)
        for (; head < t / per; ++head) end_head(h0 + head);
      uint32_t alive[2] = {~0u, ~0u};  // first: keys of the tile; the mask's bytes came with the last one
      if (!KV && mb) {
        alive[0] = __ballot_sync(0xffffffffu, byte0 != 0);
        alive[1] = __ballot_sync(0xffffffffu, byte1 != 0);
        fetch(y0 + 64 * GR);
      }
      // relative positions of the tile: [hi - 190, hi]; where they lie whole in the
      // last bucket the bias is one value, and so is the gradient's bucket
      const long long hi = (KV ? (long long)x0 + 127 - y0 : (long long)y0 + 63 - x0) - a.q_off;
      const bool behind = hi <= -(long long)a.far, ahead = hi - 190 >= (a.far_both ? (long long)a.far : 0ll);
      const bool flat = behind || ahead;
      float p[64];
      do {  // a wait that gives up leaves the tile; the warps of a group meet again below
        if (extras && !(ok = warp_wait(Y1_FULL + 8 * st, (t / R) & 1))) break;
        if (!(ok = warp_wait(S_FULL + 8 * w, turn))) break;
        ptx::tc_fence_after();
        const float* bb = KV ? e + 64 + row : e + 128 - row;
        const float whole = KV ? (a.diag && flat ? bb[0] : 0.f) : nl + (a.diag && flat ? bb[0] : 0.f);
        const bool each = a.diag && !flat;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          uint32_t s[32];
          ptx::tmem_ld32_async(s_col + 32 * z, s);
          ptx::tmem_wait_ld(s);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            uint64_t o0 = f32x2(whole, whole), o1 = o0;
            if (KV) {
              const float4 l4 = *reinterpret_cast<const float4*>(e + 192 + 32 * z + c);
              o0 = add2(o0, f32x2(l4.x, l4.y));
              o1 = add2(o1, f32x2(l4.z, l4.w));
            }
            if (each) {
              const int k = 32 * z + c;
              o0 = add2(o0, KV ? f32x2(bb[-k], bb[-k - 1]) : f32x2(bb[k], bb[k + 1]));
              o1 = add2(o1, KV ? f32x2(bb[-k - 2], bb[-k - 3]) : f32x2(bb[k + 2], bb[k + 3]));
            }
            float v0, v1, v2, v3;
            split2(fma2(f32x2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sc2, o0), v0, v1);
            split2(fma2(f32x2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), sc2, o1), v2, v3);
            p[32 * z + c] = exp2_approx(v0);
            p[32 * z + c + 1] = exp2_approx(v1);
            p[32 * z + c + 2] = exp2_approx(v2);
            p[32 * z + c + 3] = exp2_approx(v3);
          }
        }
        bool cut = false;  // pairs that do not take part: their P is 0, whatever dP is
        if (KV) {
          // causal: queries c with y0 + c + q_off < key are out
          const long long lo = a.causal ? x - a.q_off - y0 : 0;
          const int rest = a.Lq - y0;  // rows past the last query are out too: they may meet any entry of the table
          cut = dead || lo > 0 || rest < 64;
          if (cut) {
            const int n = dead ? 64 : (int)min(64ll, lo);
            alive[0] = ~low_bits(n) & low_bits(rest), alive[1] = ~low_bits(n - 32) & low_bits(rest - 32);
          }
        } else {
          const long long lim = (a.causal ? min((long long)len, x + a.q_off + 1) : (long long)len) - y0;
          if (mb || y0 + 64 > len) {  // zero the dead rows of K: two threads to a key, half of its bytes each
            const int k = row >> 1;
            if (y0 + k >= len || !(((warp & 2 ? alive[1] : alive[0]) >> (k & 31)) & 1)) {
              uint4* zr = reinterpret_cast<uint4*>(gen + oY1 + st * NS * kHalf + k * 128) + 4 * (row & 1);
#pragma unroll
              for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int c = 0; c < 4; ++c) zr[s * (kHalf / 16) + c] = make_uint4(0, 0, 0, 0);
            }
            ptx::fence_proxy_async_smem();
          }
          cut = mb || lim < 64;
          if (cut) {
            const int n = (int)max(0ll, min(64ll, lim));
            alive[0] &= low_bits(n), alive[1] &= low_bits(n - 32);
          }
        }
        if (cut) {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (!(alive[c >> 5] & (1u << (c & 31)))) p[c] = 0.f;
        }
        {
          uint32_t q[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) q[c] = pack2<T>(p[2 * c], p[2 * c + 1]);
          tmem_st32(s_col, q);
        }
        tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(P_READY + 8 * w);

        if (KV ? lone > y0 : x < lone) {
          const int n = KV ? lone - y0 : 64;
          alive[0] &= ~low_bits(n), alive[1] &= ~low_bits(n - 32);
          cut = true;
        }
        if (!(ok = warp_wait(DP_FULL + 8 * w, turn))) break;
        ptx::tc_fence_after();
        uint64_t sum = f32x2(0.f, 0.f);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          uint32_t s[32];
          ptx::tmem_ld32_async(d_col + 32 * z, s);
          ptx::tmem_wait_ld(s);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            uint64_t n0 = f32x2(nt, nt), n1 = n0;
            if (KV) {
              const float4 d4 = *reinterpret_cast<const float4*>(e + 256 + 32 * z + c);
              n0 = f32x2(d4.x, d4.y), n1 = f32x2(d4.z, d4.w);
            }
            float* q = p + 32 * z + c;
            const uint64_t u0 = mul2(f32x2(q[0], q[1]), add2(f32x2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), n0));
            const uint64_t u1 =
                mul2(f32x2(q[2], q[3]), add2(f32x2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), n1));
            float v[4];
            split2(u0, v[0], v[1]);
            split2(u1, v[2], v[3]);
            if (cut) {
#pragma unroll
              for (int k = 0; k < 4; ++k) q[k] = alive[z] & (1u << (c + k)) ? v[k] : 0.f;
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) q[k] = v[k];
            }
            if (!KV) sum = add2(sum, add2(f32x2(q[0], q[1]), f32x2(q[2], q[3])));
          }
        }
        if (!KV) {
          float u, v;
          split2(sum, u, v);
          r += u + v;
        }
        {
          uint32_t q[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) q[c] = pack2<T>(p[2 * c], p[2 * c + 1]);
          tmem_st32(d_col, q);
        }
        tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(DS_READY + 8 * w);
          if (extras) ptx::mbar_arrive(Y1_EMPTY + 8 * st);
        }
      } while (false);
      // the named barriers below are taken by all warps of a group or by none
      if (KV && a.dws) ok = ptx::named_bar_and(1 + w, 128, ok);
      if (!ok) break;
      if (KV && a.dws) {
        float* dws = a.dws + ((((int64_t)b * a.Hq + h0 + head) * ntile + xt) * GR + w) * a.dws_ld;
        // Diagonal u < 191 of the tile: key - query = 127 - u; it is entry y0 + u of
        // the array.  The first kStep are whole with this tile (the group's next is
        // kStep queries on), the others stay open.
        for (int64_t z = at + row; z < y0; z += 128) dws[z] = z - at < kOpen ? carry[64 * w + (z - at)] : 0.f;
        const bool joins = at == y0;  // the open diagonals are the first of this tile
        float v0 = 0.f, v1 = 0.f;     // diagonals row and 128 + row
        if (flat) {
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
          ptx::named_bar(1 + w, 128);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            // rows 32 y + lane, columns c: entry 31 - (lane - c) = 31 - (127 - u - 32 y)
            const float* part = diag_s + (4 * w + y) * kDiagLd;
            const int k = 31 - (127 - row - 32 * y);
            if (k >= 0 && k < 95) v0 += part[k];
            if (row < 63 && k + 128 < 95) v1 += part[k + 128];
          }
        }
        if (joins && row < kOpen) v0 += carry[64 * w + row];
        if (row < kStep) dws[(int64_t)y0 + row] = v0;
        ptx::named_bar(1 + w, 128);
        if (row >= kStep) carry[64 * w + row - kStep] = v0;
        if (row < 64) carry[64 * w + 128 - kStep + row] = row < 63 ? v1 : 0.f;
        at = (int64_t)y0 + kStep;
        ptx::named_bar(1 + w, 128);
      }
    }
    if (KV && a.dws && ok)
      for (; head < G; ++head) end_head(h0 + head);
    if (ok && tiles > 0) ok = warp_wait(DONE, 0) && *undone == 0;
    ptx::tc_fence_after();
    if (KV && a.dws) ok = ptx::named_bar_and(1 + w, 128, ok);
    if (!ok) {  // a wait gave up: NaN in what this block was to write
      if (lane == 0) atomicExch(a.err, 53);
      if (KV && a.dws)
        for (int hy = h0; hy < h0 + G; ++hy) {
          float* dws = a.dws + ((((int64_t)b * a.Hq + hy) * ntile + xt) * GR + w) * a.dws_ld;
          for (int64_t z = row; z < a.dws_ld; z += 128) dws[z] = no_result();
        }
    }
    float rr = 0.f;
    if (!KV) {
      // the groups' sums of a row (every warp comes here, also after a wait that gave up)
      rr = r;
      if (GR == 2) {
        ext[128 * w + row] = r;
        ptx::named_bar(3, 256);
        rr = ext[row] + ext[128 + row];
      }
      if (w == 0) {
        const int64_t to = ((int64_t)b * a.Hq + hx) * Lp + x;
        a.lse2[to] = ok ? nl : no_result();
        a.delta[to] = nl == -INFINITY ? 0.f : nt - rr;
      }
    }
    {
      const int L = KV ? a.Lk : a.Lq;
      const int64_t to = (((int64_t)b * L + x) * heads + hx) * a.D;
      T* d1 = static_cast<T*>(KV ? a.dk : a.dq) + to;
      T* d2 = static_cast<T*>(a.dv) + to;
#pragma unroll 1
      for (int c0 = 64 * NS / GR * w; c0 < 64 * NS / GR * (w + 1); c0 += 16) {  // each group its share of the values
        if (c0 >= a.D) break;
        float u[16], v[16];
        if (ok && tiles > 0) {
          ptx::tmem_ld16(tA1 + lanes + c0, u);
          ptx::tmem_ld16(tA2 + lanes + c0, v);
        } else {
#pragma unroll
          for (int c = 0; c < 16; ++c) u[c] = v[c] = ok ? 0.f : no_result();
        }
        if (x >= L) continue;
        if (KV && a.nsplit > 1) {  // this share's part, for kv_join_kernel
          const int64_t part = (int64_t)blockIdx.y * a.B * a.Lk * a.Hkv * a.D + to + c0;
#pragma unroll
          for (int c = 0; c < 16; c += 4)
            if (c0 + c < a.D) {
              *reinterpret_cast<float4*>(a.po + part + c) = make_float4(u[c], u[c + 1], u[c + 2], u[c + 3]);
              *reinterpret_cast<float4*>(a.pml + part + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
            }
          continue;
        }
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
  if (warp == kIssue) ptx::tmem_dealloc(tmem, 256 * GR);
}

// dK and dV from the shares of the query heads, added in order.
template <typename T>
__global__ void __launch_bounds__(256) kv_join_kernel(const __grid_constant__ AttnArgs a, long long n) {
  const long long e = blockIdx.x * 256ll + threadIdx.x;
  if (e >= n) return;
  float k = 0.f, v = 0.f;
  for (int s = 0; s < a.nsplit; ++s) {
    k += a.po[s * n + e];
    v += a.pml[s * n + e];
  }
  static_cast<T*>(a.dk)[e] = from_f<T>(a.scale * k);
  static_cast<T*>(a.dv)[e] = from_f<T>(v);
}

template <typename T, int NS, bool KV, bool FULL>
void launch(const AttnArgs& a, const BwdMaps& maps, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};  // one bit per device
  int dev = 0;
  RVC_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !(done.load() & (1ull << dev))) {
    RVC_CUDA_TRY(cudaFuncSetAttribute(attn_tc_bwd_kernel<T, NS, KV, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)bwd_smem<NS>()));
    if (dev < 64) done.fetch_or(1ull << dev);
  }
  const unsigned grid = KV ? (unsigned)((a.Lk + 127ll) / 128 * a.B * a.Hkv) : (unsigned)((a.Lq + 127ll) / 128 * a.B * a.Hq);
  attn_tc_bwd_kernel<T, NS, KV, FULL><<<dim3(grid, KV ? a.nsplit : 1), kBwdThreads<NS>, bwd_smem<NS>(), st>>>(a, maps);
  note_launch();
  RVC_CUDA_TRY(cudaGetLastError());
  if (KV && a.nsplit > 1) {
    const long long n = (long long)a.B * a.Lk * a.Hkv * a.D;
    kv_join_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a, n);
    note_launch();
    RVC_CUDA_TRY(cudaGetLastError());
  }
}

template <typename T, int NS, bool FULL>
void bwd(const AttnArgs& a, cudaStream_t st) {
  BwdMaps m;
  make_map(&m.x1, a.type, a.q, a.qs, a.B, a.Lq, a.Hq, a.D, 128);
  make_map(&m.x2, a.type, a.dout, a.dos, a.B, a.Lq, a.Hq, a.D, 128);
  make_map(&m.y1, a.type, a.k, a.ks, a.B, a.Lk, a.Hkv, a.D, 64);
  make_map(&m.y2, a.type, a.v, a.vs, a.B, a.Lk, a.Hkv, a.D, 64);
  launch<T, NS, false, FULL>(a, m, st);
  make_map(&m.x1, a.type, a.k, a.ks, a.B, a.Lk, a.Hkv, a.D, 128);
  make_map(&m.x2, a.type, a.v, a.vs, a.B, a.Lk, a.Hkv, a.D, 128);
  make_map(&m.y1, a.type, a.q, a.qs, a.B, a.Lq, a.Hq, a.D, 64);
  make_map(&m.y2, a.type, a.dout, a.dos, a.B, a.Lq, a.Hq, a.D, 64);
  launch<T, NS, true, FULL>(a, m, st);
}

template <typename T>
void bwd_t(const AttnArgs& a, cudaStream_t st) {
  if (a.D == 64) bwd<T, 1, true>(a, st);
  else if (a.D < 64) bwd<T, 1, false>(a, st);
  else if (a.D == 128) bwd<T, 2, true>(a, st);
  else bwd<T, 2, false>(a, st);
}

}  // namespace

// Shares of a group's query heads for the second kernel, where its key tiles
// leave half of the SMs' places or more empty.
int attn_tc_bwd_shares(const AttnArgs& a, int sms) {
  const long long blocks = (a.Lk + 127ll) / 128 * a.B * a.Hkv, places = (a.D <= 64 ? 2ll : 1ll) * sms;
  return (int)std::max(1ll, std::min((long long)(a.Hq / a.Hkv), places / std::max(1ll, blocks)));
}

int attn_tc_bwd_arrays(const AttnArgs& a) { return a.D <= 64 ? kGroups<1> : kGroups<2>; }

// Many queries, or keys enough to pay for a query tile that is mostly empty: for 1
// to 48 queries the general kernels take 53 us against 39 at 256 keys (12 heads of
// 64), 1434 against 307 at 8 x 6831 (16/4 heads of 128).
bool attn_tc_bwd_fits(const AttnArgs& a) {
  const auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  return a.type != kF32 && a.Lk >= 64 && (a.Lq >= 64 || a.Lk >= 256) && map_ok(a, a.q, a.qs, a.Lq, a.Hq) &&
         map_ok(a, a.k, a.ks, a.Lk, a.Hkv) && map_ok(a, a.v, a.vs, a.Lk, a.Hkv) &&
         map_ok(a, a.dout, a.dos, a.Lq, a.Hq) && map_ok(a, a.fout, a.os, a.Lq, a.Hq) && al(a.dq) && al(a.dk) && al(a.dv);
}

void attn_tc_backward(const AttnArgs& a, cudaStream_t st) {
  if (a.type == kBf16) bwd_t<__nv_bfloat16>(a, st);
  else bwd_t<__half>(a, st);
}

}  // namespace rvc
