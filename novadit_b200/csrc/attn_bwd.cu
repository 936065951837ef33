// Attention backward (sm_100a). With P = 2^(S c - lse) recomputed from the saved log-sum-exp,
//   delta = rowsum(dO * O),  dP = dO V^T,  dS = P (dP - delta),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
// in two kernels. One holds a query tile and walks the keys (dQ, and delta on the way), the other holds a key tile and
// walks the queries of all heads that share it (dK, dV). Recomputing S and dP for both costs two products more than one
// kernel that adds dQ up in global memory, but every sum stays in tensor memory in one fixed order: no atomics, results
// do not change from run to run, and the second operand of every product is a tile that lies in shared memory already.
//
// Both: one persistent CTA per SM, 320 threads, warps 0-7 the elementwise part (two warps per TMEM lane quarter, each
// taking 64 of the tile's 128 columns), warp 8 copies, warp 9 issues the MMAs. P and dS are the A operands of the last
// products straight from tensor memory, in 16 bits (one rounding, unbiased, below that of the output); scores, dP,
// statistics and accumulators stay in 32 bits.
//
// dQ kernel, per key tile j:  S(j) = Q K^T, dP(j) = dO V^T, dQ += dS(j) K. S(j + 1) is issued as soon as S(j) is in
// registers, dP(j + 1) behind dQ(j).
// dK/dV kernel, per query tile i (everything transposed: lanes are keys):  S(i) = K Q^T, dP(i) = V dO^T,
// dV += P(i) dO, dK += dS(i) Q. P lies over S's columns and dS over dP's, each half of the columns in its own half; S(i+1)
// is issued behind dV(i) while dS(i) is computed, dP(i + 1) behind dK(i) while the next exponentials run.
#include "attn.cuh"

namespace nd {

constexpr int kBwdThreads = 320;

struct BwdArgs {
  AttnShape s;
  AttnMask mask;
  WaitSink sink;
  const float* lse;   // [batch, hb, rows_pad]
  float* delta;       // [batch, hb, rows_pad]
  const void* out;    // contiguous [B, Sq, Hq, D]
  const void* dout;   // strided
  long long do_b, do_s, do_h;
  float* part;        // dK/dV, splits > 1: [splits][2][B * Sk * Hkv][D]
  float c, scale;
  int items;
  int splits, steps, steps_per_split;  // dK/dV: query tiles of all head blocks of a key head
};

template <int NB> struct __align__(1024) BwdSmem {
  static constexpr int kRing = NB == 1 ? 8 : 4;
  uint8_t res[2][NB * kBlkBytes];        // dQ: Q, dO; dK/dV: K, V
  uint8_t ring[kRing][NB * kBlkBytes];   // dQ: K, V, K, V, ...; dK/dV: Q, dO, ...
  uint8_t out[8][2048];
  alignas(16) float stat[kRing / 2][2][kTile];  // dK/dV: log-sum-exp and delta of the query tile
  uint64_t res_full, res_empty;
  uint64_t full[kRing], empty[kRing];
  uint64_t s_full, dp_full;   // MMA -> elementwise
  uint64_t p_full, ds_full;   // elementwise -> MMA (dQ: p_full = "S is in registers")
  uint64_t ds_free, acc_done; // dQ: dS has been read; both: the accumulators are complete
  uint32_t tmem_base;
  int abort_flag;
};

template <int NB> __device__ __forceinline__ void bwd_init(BwdSmem<NB>& s) {
  mbar_init(&s.res_full, 1);
  mbar_init(&s.res_empty, 1);
  for (int i = 0; i < BwdSmem<NB>::kRing; ++i) {
    mbar_init(&s.full[i], 1);
    mbar_init(&s.empty[i], 1);
  }
  mbar_init(&s.s_full, 1);
  mbar_init(&s.dp_full, 1);
  mbar_init(&s.p_full, 8);
  mbar_init(&s.ds_full, 8);
  mbar_init(&s.ds_free, 1);
  mbar_init(&s.acc_done, 1);
  s.abort_flag = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

// ------------------------------------------------------------------ dQ
// TMEM columns: S 0, dP 128, dS 256 (64 columns of 16-bit pairs), dQ 384
template <int NB, typename T>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
               const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
               const __grid_constant__ CUtensorMap map_dq, const BwdArgs a) {
  constexpr int kRing = BwdSmem<NB>::kRing;
  constexpr int kTileBytes = NB * kBlkBytes;
  extern __shared__ uint8_t smem_raw[];
  BwdSmem<NB>& s = *reinterpret_cast<BwdSmem<NB>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort_flag;
  if (threadIdx.x == 0) bwd_init<NB>(s);
  if (warp == 9) tmem_alloc<512>(&s.tmem_base);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  griddep_launch_dependents();
  griddep_wait();

  const int group_blocks = a.s.hb / a.s.hkv;
  const int pos_per_tile = kTile / a.s.gp;
  constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  struct Item {
    int b, hb, qt, n_keys, n_t;
  };
  auto get = [&](int item) {
    Item w;
    w.qt = item % a.s.qtiles;
    const int r = item / a.s.qtiles;
    w.hb = r % a.s.hb;
    w.b = r / a.s.hb;
    w.n_keys = key_count(a.mask, w.b, a.s.sk, lane);
    w.n_t = (w.n_keys + kTile - 1) / kTile;
    return w;
  };

  if (warp == 8) {
    int it = 0, cnt = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const Item w = get(item);
      if (w.n_t == 0) continue;
      if (lane == 0) {
        ok = mbar_wait(&s.res_empty, (cnt & 1) ^ 1, abort_flag, a.sink, 121);
        if (ok) {
          mbar_expect_tx(&s.res_full, 2 * kTileBytes);
          load_tile<NB>(s.res[0], &map_q, &s.res_full, w.hb * a.s.gp, w.qt * pos_per_tile, w.b);
          load_tile<NB>(s.res[1], &map_do, &s.res_full, w.hb * a.s.gp, w.qt * pos_per_tile, w.b);
        }
        for (int j = 0; j < 2 * w.n_t && ok; ++j) {
          const int slot = (it + j) % kRing;
          ok = mbar_wait(&s.empty[slot], (((it + j) / kRing) & 1) ^ 1, abort_flag, a.sink, 122);
          if (!ok) break;
          mbar_expect_tx(&s.full[slot], kTileBytes);
          load_tile<NB>(s.ring[slot], (j & 1) ? &map_v : &map_k, &s.full[slot], w.hb / group_blocks, (j >> 1) * kTile, w.b);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      it += 2 * w.n_t;
      ++cnt;
    }
    if (!ok) settle();
  } else if (warp == 9) {
    const int ksteps = a.s.dn / 16;
    const uint32_t id_s = attn_idesc(kFmt, kTile, false), id_o = attn_idesc(kFmt, a.s.dn, true);
    const uint64_t res = desc_k(smem_u32(s.res[0])), ring = desc_k(smem_u32(s.ring[0])), ring_mn = desc_mn<>(smem_u32(s.ring[0]));
    constexpr uint32_t kStep = kTileBytes >> 4;
    int it = 0, cnt = 0;
    uint32_t done = 0;  // key tiles of the items before
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const Item w = get(item);
      if (w.n_t == 0) continue;
      if (elect_one()) {
        ok = mbar_wait(&s.res_full, cnt & 1, abort_flag, a.sink, 123);
        for (int j = -1; j < w.n_t && ok; ++j) {
          const int k_at = it + 2 * j, k_next = k_at + 2, v_next = k_at + 3;
          const bool more = j + 1 < w.n_t;
          // S(j + 1), once S(j) is in registers
          if (j >= 0) {
            ok = mbar_wait(&s.p_full, (done + j) & 1, abort_flag, a.sink, 124);
            if (!ok) break;
          }
          if (more) {
            ok = mbar_wait(&s.full[k_next % kRing], (k_next / kRing) & 1, abort_flag, a.sink, 125);
            if (!ok) break;
            tc_fence_after();
            issue_nt(tmem, res, ring + (k_next % kRing) * kStep, ksteps, id_s);
            mma_commit(&s.s_full);
          }
          if (j >= 0) {  // dQ += dS(j) K(j)
            ok = mbar_wait(&s.ds_full, (done + j) & 1, abort_flag, a.sink, 126);
            if (!ok) break;
            tc_fence_after();
            issue_tn(tmem + 384, tmem + 256, 32, ring_mn + (k_at % kRing) * kStep, 8, id_o, j > 0 ? 1u : 0u);
            mma_commit(&s.ds_free);
            mma_commit(&s.empty[k_at % kRing]);
            if (!more) mma_commit(&s.acc_done);
          }
          if (more) {  // dP(j + 1): dP(j) was in registers before dS(j) was ready
            ok = mbar_wait(&s.full[v_next % kRing], (v_next / kRing) & 1, abort_flag, a.sink, 127);
            if (!ok) break;
            tc_fence_after();
            issue_nt(tmem + 128, res + kStep, ring + (v_next % kRing) * kStep, ksteps, id_s);
            mma_commit(&s.dp_full);
            mma_commit(&s.empty[v_next % kRing]);
            if (j + 2 == w.n_t) mma_commit(&s.res_empty);
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      it += 2 * w.n_t;
      done += w.n_t;
      ++cnt;
    }
    __syncwarp();
  } else {
    const int half = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem + lanes + half * 64, t_dp = t_s + 128, t_ds = tmem + lanes + 256 + half * 32, t_dq = tmem + lanes + 384;
    uint8_t* stage = s.out[warp];
    uint32_t cnt = 0;  // key tiles so far: the phase of every per-tile barrier
    uint32_t done = 0;
    int it = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const Item w = get(item);
      const int it0 = it;
      it += 2 * w.n_t;
      const int row = w.qt * kTile + r;
      const long long at = (static_cast<long long>(w.b) * a.s.hb + w.hb) * a.s.rows_pad + row;
      float lse = INFINITY, delta = 0.f;
      if (row < a.s.rows && w.n_t > 0) {
        lse = a.lse[at];
        const int pos = row / a.s.gp, head = w.hb * a.s.gp + row % a.s.gp;
        const uint4* po = reinterpret_cast<const uint4*>(
            static_cast<const T*>(a.out) + ((static_cast<long long>(w.b) * a.s.sq + pos) * a.s.hq + head) * a.s.d);
        const uint4* pg = reinterpret_cast<const uint4*>(
            static_cast<const T*>(a.dout) + w.b * a.do_b + pos * a.do_s + head * a.do_h);
        for (int v = 0; v < a.s.d / 8; ++v) {
          const uint4 x = __ldg(po + v), y = __ldg(pg + v);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 fx = unpack_pair<T>(xs[e]), fy = unpack_pair<T>(ys[e]);
            delta = fmaf(fx.x, fy.x, delta);
            delta = fmaf(fx.y, fy.y, delta);
          }
        }
      }
      if (half == 0) a.delta[at] = delta;
      for (int j = 0; j < w.n_t; ++j, ++cnt) {
        uint32_t bits[4];
        const bool partial = key_bits(a.mask, w.b, a.s.sk, w.n_keys, j, lane, bits);
        const uint32_t b0 = half == 0 ? bits[0] : bits[2], b1 = half == 0 ? bits[1] : bits[3];
        ok = warp_wait(&s.s_full, cnt & 1, abort_flag, a.sink, 128);
        if (!ok) break;
        tc_fence_after();
        float p[2][32];
        tc_ld32(t_s, p[0]);
        tc_ld32(t_s + 32, p[1]);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 32; ++e) p[i][e] = ex2_approx(fmaf(p[i][e], a.c, -lse));
        if (partial) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            p[0][e] = (b0 >> e) & 1u ? p[0][e] : 0.f;
            p[1][e] = (b1 >> e) & 1u ? p[1][e] : 0.f;
          }
          if (half == 0) {  // see the forward pass: a masked key's row of K must not reach the last product
            const int k_at = it0 + 2 * j;
            ok = warp_wait(&s.full[k_at % kRing], (k_at / kRing) & 1, abort_flag, a.sink, 129);
            if (!ok) break;
            if (!((bits[quarter] >> lane) & 1u)) clear_row<NB>(s.ring[k_at % kRing], r);
            fence_proxy_async_smem();
          }
        }
        ok = warp_wait(&s.dp_full, cnt & 1, abort_flag, a.sink, 130);
        if (!ok) break;
        tc_fence_after();
        float dp[2][32];
        tc_ld32(t_dp, dp[0]);
        tc_ld32(t_dp + 32, dp[1]);
        tc_wait_ld();
        if (partial) {  // dP of a masked key may be anything, NaN included
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            dp[0][e] = (b0 >> e) & 1u ? dp[0][e] : 0.f;
            dp[1][e] = (b1 >> e) & 1u ? dp[1][e] : 0.f;
          }
        }
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            pk[i * 16 + e / 2] = pack2<T>(p[i][e] * (dp[i][e] - delta), p[i][e + 1] * (dp[i][e + 1] - delta));
        if (cnt > 0) {
          ok = warp_wait(&s.ds_free, (cnt - 1) & 1, abort_flag, a.sink, 131);
          if (!ok) break;
          tc_fence_after();
        }
        tc_st32(t_ds, pk);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.ds_full);
      }
      if (!ok) break;
      if (w.n_t > 0) {
        ok = warp_wait(&s.acc_done, done & 1, abort_flag, a.sink, 132);
        if (!ok) break;
        ++done;
        tc_fence_after();
      }
      const int pos = w.qt * pos_per_tile + quarter * 32 / a.s.gp;
      for (int c = half * 32; c < a.s.d; c += 64) {
        float o[32];
        tc_ld32(t_dq + c, o);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = w.n_t == 0 ? 0.f : o[e] * a.scale;
        store_block<T>(&map_dq, stage, o, lane, c, w.hb * a.s.gp, pos, w.b, pos < a.s.sq);
      }
      tc_fence_before();
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_free<512>(tmem);
}

// ------------------------------------------------------------------ dK and dV
// TMEM columns: S 0, dP 128, dV 256, dK 384; P and dS as 16-bit pairs at columns 0..31 and 64..95 of S and dP
template <int NB, typename T>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ CUtensorMap map_dk, const __grid_constant__ CUtensorMap map_dv, const BwdArgs a) {
  constexpr int kRing = BwdSmem<NB>::kRing;
  constexpr int kTileBytes = NB * kBlkBytes;
  extern __shared__ uint8_t smem_raw[];
  BwdSmem<NB>& s = *reinterpret_cast<BwdSmem<NB>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort_flag;
  if (threadIdx.x == 0) bwd_init<NB>(s);
  if (warp == 9) tmem_alloc<512>(&s.tmem_base);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  griddep_launch_dependents();
  griddep_wait();

  const int group_blocks = a.s.hb / a.s.hkv;
  const int pos_per_tile = kTile / a.s.gp;
  constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  struct Item {
    int b, h, kt, split, n_keys, i0, n_i;  // query tiles [i0, i0 + n_i) of the group, head block by head block
  };
  auto get = [&](int item) {
    Item w;
    w.split = item % a.splits;
    int r = item / a.splits;
    w.kt = r % a.s.ktiles;
    r /= a.s.ktiles;
    w.h = r % a.s.hkv;
    w.b = r / a.s.hkv;
    w.n_keys = key_count(a.mask, w.b, a.s.sk, lane);
    w.i0 = w.split * a.steps_per_split;
    w.n_i = a.steps - w.i0 < a.steps_per_split ? a.steps - w.i0 : a.steps_per_split;
    if (w.kt * kTile >= w.n_keys || w.n_i < 0) w.n_i = 0;
    return w;
  };

  if (warp == 8) {
    int it = 0, cnt = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const Item w = get(item);
      if (w.n_i == 0) continue;
      if (lane == 0) {
        ok = mbar_wait(&s.res_empty, (cnt & 1) ^ 1, abort_flag, a.sink, 141);
        if (ok) {
          mbar_expect_tx(&s.res_full, 2 * kTileBytes);
          load_tile<NB>(s.res[0], &map_k, &s.res_full, w.h, w.kt * kTile, w.b);
          load_tile<NB>(s.res[1], &map_v, &s.res_full, w.h, w.kt * kTile, w.b);
        }
        for (int i = 0; i < w.n_i && ok; ++i) {
          const int sub = (w.i0 + i) / a.s.qtiles, qt = (w.i0 + i) - sub * a.s.qtiles;
          const int hb = w.h * group_blocks + sub;
          const int qa = it + 2 * i, da = qa + 1;
          ok = mbar_wait(&s.empty[qa % kRing], ((qa / kRing) & 1) ^ 1, abort_flag, a.sink, 142);
          if (!ok) break;
          mbar_expect_tx(&s.full[qa % kRing], kTileBytes + 2 * kTile * 4);
          load_tile<NB>(s.ring[qa % kRing], &map_q, &s.full[qa % kRing], hb * a.s.gp, qt * pos_per_tile, w.b);
          const long long at = (static_cast<long long>(w.b) * a.s.hb + hb) * a.s.rows_pad + qt * kTile;
          bulk_load_1d(s.stat[(qa % kRing) / 2][0], a.lse + at, kTile * 4, &s.full[qa % kRing]);
          bulk_load_1d(s.stat[(qa % kRing) / 2][1], a.delta + at, kTile * 4, &s.full[qa % kRing]);
          ok = mbar_wait(&s.empty[da % kRing], ((da / kRing) & 1) ^ 1, abort_flag, a.sink, 143);
          if (!ok) break;
          mbar_expect_tx(&s.full[da % kRing], kTileBytes);
          load_tile<NB>(s.ring[da % kRing], &map_do, &s.full[da % kRing], hb * a.s.gp, qt * pos_per_tile, w.b);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      it += 2 * w.n_i;
      ++cnt;
    }
    if (!ok) settle();
  } else if (warp == 9) {
    const int ksteps = a.s.dn / 16;
    const uint32_t id_s = attn_idesc(kFmt, kTile, false), id_o = attn_idesc(kFmt, a.s.dn, true);
    const uint64_t res = desc_k(smem_u32(s.res[0])), ring = desc_k(smem_u32(s.ring[0])), ring_mn = desc_mn<>(smem_u32(s.ring[0]));
    constexpr uint32_t kStep = kTileBytes >> 4;
    int it = 0, cnt = 0;
    uint32_t done = 0;  // query tiles of the items before
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const Item w = get(item);
      if (w.n_i == 0) continue;
      if (elect_one()) {
        ok = mbar_wait(&s.res_full, cnt & 1, abort_flag, a.sink, 144);
        for (int i = -1; i < w.n_i && ok; ++i) {
          const int qa = it + 2 * i, da = qa + 1, qn = qa + 2, dn = qa + 3;
          const bool more = i + 1 < w.n_i;
          if (i >= 0) {  // dV += P(i) dO(i)
            ok = mbar_wait(&s.p_full, (done + i) & 1, abort_flag, a.sink, 145);
            if (!ok) break;
            tc_fence_after();
            issue_tn(tmem + 256, tmem, 64, ring_mn + (da % kRing) * kStep, 8, id_o, i > 0 ? 1u : 0u);
            mma_commit(&s.empty[da % kRing]);
          }
          if (more) {  // S(i + 1) over P(i), which dV(i) reads first
            ok = mbar_wait(&s.full[qn % kRing], (qn / kRing) & 1, abort_flag, a.sink, 146);
            if (!ok) break;
            tc_fence_after();
            issue_nt(tmem, res, ring + (qn % kRing) * kStep, ksteps, id_s);
            mma_commit(&s.s_full);
          }
          if (i >= 0) {  // dK += dS(i) Q(i)
            ok = mbar_wait(&s.ds_full, (done + i) & 1, abort_flag, a.sink, 147);
            if (!ok) break;
            tc_fence_after();
            issue_tn(tmem + 384, tmem + 128, 64, ring_mn + (qa % kRing) * kStep, 8, id_o, i > 0 ? 1u : 0u);
            mma_commit(&s.empty[qa % kRing]);
            if (!more) mma_commit(&s.acc_done);
          }
          if (more) {
            ok = mbar_wait(&s.full[dn % kRing], (dn / kRing) & 1, abort_flag, a.sink, 148);
            if (!ok) break;
            tc_fence_after();
            issue_nt(tmem + 128, res + kStep, ring + (dn % kRing) * kStep, ksteps, id_s);
            mma_commit(&s.dp_full);
            if (i + 2 == w.n_i) mma_commit(&s.res_empty);
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      it += 2 * w.n_i;
      done += w.n_i;
      ++cnt;
    }
    __syncwarp();
  } else {
    const int half = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem + lanes + half * 64, t_dp = t_s + 128, t_dv = tmem + lanes + 256, t_dk = tmem + lanes + 384;
    uint8_t* stage = s.out[warp];
    uint32_t cnt = 0, done = 0;
    int it = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const Item w = get(item);
      const int it0 = it;
      it += 2 * w.n_i;
      bool mine = false;  // this thread's key takes part
      if (w.n_i > 0) {
        uint32_t bits[4];
        key_bits(a.mask, w.b, a.s.sk, w.n_keys, w.kt, lane, bits);
        mine = (bits[quarter] >> lane) & 1u;
      }
      for (int i = 0; i < w.n_i; ++i, ++cnt) {
        const int qa = it0 + 2 * i;
        ok = warp_wait(&s.full[qa % kRing], (qa / kRing) & 1, abort_flag, a.sink, 149);  // the statistics have landed
        if (!ok) break;
        const float4* st_l = reinterpret_cast<const float4*>(s.stat[(qa % kRing) / 2][0]) + half * 16;
        const float4* st_d = reinterpret_cast<const float4*>(s.stat[(qa % kRing) / 2][1]) + half * 16;
        ok = warp_wait(&s.s_full, cnt & 1, abort_flag, a.sink, 150);
        if (!ok) break;
        tc_fence_after();
        float p[2][32];
        tc_ld32(t_s, p[0]);
        tc_ld32(t_s + 32, p[1]);
        tc_wait_ld();
        uint32_t pk[32];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 l4 = st_l[h * 8 + e / 4];
            p[h][e] = ex2_approx(fmaf(p[h][e], a.c, -l4.x));
            p[h][e + 1] = ex2_approx(fmaf(p[h][e + 1], a.c, -l4.y));
            p[h][e + 2] = ex2_approx(fmaf(p[h][e + 2], a.c, -l4.z));
            p[h][e + 3] = ex2_approx(fmaf(p[h][e + 3], a.c, -l4.w));
            pk[h * 16 + e / 2] = mine ? pack2<T>(p[h][e], p[h][e + 1]) : 0u;
            pk[h * 16 + e / 2 + 1] = mine ? pack2<T>(p[h][e + 2], p[h][e + 3]) : 0u;
          }
        tc_st32(t_s, pk);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full);
        ok = warp_wait(&s.dp_full, cnt & 1, abort_flag, a.sink, 151);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float dp[32];
          tc_ld32(t_dp + h * 32, dp);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 d4 = st_d[h * 8 + e / 4];
            const uint32_t lo = pack2<T>(p[h][e] * (dp[e] - d4.x), p[h][e + 1] * (dp[e + 1] - d4.y));
            const uint32_t hi = pack2<T>(p[h][e + 2] * (dp[e + 2] - d4.z), p[h][e + 3] * (dp[e + 3] - d4.w));
            pk[h * 16 + e / 2] = mine ? lo : 0u;
            pk[h * 16 + e / 2 + 1] = mine ? hi : 0u;
          }
        }
        tc_st32(t_dp, pk);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.ds_full);
      }
      if (!ok) break;
      if (w.n_i > 0) {
        ok = warp_wait(&s.acc_done, done & 1, abort_flag, a.sink, 152);
        if (!ok) break;
        ++done;
        tc_fence_after();
      }
      // dV, then dK, 32 columns at a time, the two halves taking turns
      const int key = w.kt * kTile + r;
      for (int which = 0; which < 2; ++which) {
        const uint32_t src = which == 0 ? t_dv : t_dk;
        const float mul = which == 0 ? 1.f : a.scale;
        for (int c = half * 32; c < a.s.d; c += 64) {
          float o[32];
          tc_ld32(src + c, o);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = w.n_i == 0 ? 0.f : o[e] * mul;
          if (a.splits > 1) {
            const long long n = static_cast<long long>(a.s.batch) * a.s.sk * a.s.hkv;
            const long long at = (static_cast<long long>(w.b) * a.s.sk + key) * a.s.hkv + w.h;
            if (key < a.s.sk) {
              float4* dst = reinterpret_cast<float4*>(a.part + ((static_cast<long long>(w.split) * 2 + which) * n + at) * a.s.d + c);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (c + e * 4 < a.s.d) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          } else {
            const int k0 = w.kt * kTile + quarter * 32;
            store_block<T>(which == 0 ? &map_dv : &map_dk, stage, o, lane, c, w.h, k0, w.b, k0 < a.s.sk);
          }
        }
      }
      tc_fence_before();
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_free<512>(tmem);
}

// adds the partial dK and dV of the query ranges, in their order
template <typename T>
__global__ void __launch_bounds__(256) attn_dkv_join_kernel(const float* __restrict__ part, T* __restrict__ dk, T* __restrict__ dv,
                                                            long long n4, int splits) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  griddep_wait();
  if (i >= 2 * n4) return;
  const float4* p = reinterpret_cast<const float4*>(part) + i;
  float4 acc = p[0];
  for (int s = 1; s < splits; ++s) {
    const float4 x = p[static_cast<long long>(s) * 2 * n4];
    acc.x += x.x;
    acc.y += x.y;
    acc.z += x.z;
    acc.w += x.w;
  }
  T* dst = i < n4 ? dv + i * 4 : dk + (i - n4) * 4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x, acc.y), pack2<T>(acc.z, acc.w));
}

// ------------------------------------------------------------------ host side
static void bwd_plan(BwdArgs& a) {
  a.steps = a.s.qtiles * (a.s.hb / a.s.hkv);
  const long long items = static_cast<long long>(a.s.batch) * a.s.hkv * a.s.ktiles;
  const int sms = sm_count();
  a.splits = 1;
  if (items > 0 && items < sms) {
    const int want = static_cast<int>(sms / items);
    a.splits = want < a.steps ? want : a.steps;
  }
  a.steps_per_split = (a.steps + a.splits - 1) / a.splits;
  a.splits = (a.steps + a.steps_per_split - 1) / a.steps_per_split;
}

static size_t bwd_delta_bytes(const AttnShape& s) {
  return static_cast<size_t>(s.batch) * s.hb * s.rows_pad * sizeof(float);
}
static size_t bwd_ws(const BwdArgs& a) {
  size_t n = bwd_delta_bytes(a.s);
  if (a.splits > 1) n += static_cast<size_t>(a.splits) * 2 * a.s.batch * a.s.sk * a.s.hkv * a.s.d * sizeof(float);
  return n;
}
}  // namespace nd

extern "C" {

size_t nd_attn_bwd_ws_bytes(int64_t batch, int64_t sq, int64_t sk, int64_t hq, int64_t hkv, int64_t head_dim) {
  if (nd::attn_check(ND_BF16, batch, sq, sk, hq, hkv, head_dim, 1.f) != ND_OK || batch == 0 || sq == 0 || sk == 0) return 0;
  nd::BwdArgs a{};
  a.s = nd::attn_shape(batch, sq, sk, hq, hkv, head_dim);
  nd::bwd_plan(a);
  return nd::bwd_ws(a);
}

int nd_attn_bwd(int dtype, const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse,
                void* dq, void* dk, void* dv, const void* key_mask, const int* kv_lens, int64_t batch, int64_t sq, int64_t sk,
                int64_t hq, int64_t hkv, int64_t head_dim, const int64_t* strides, float scale, void* ws, size_t ws_bytes,
                void* stream) {
  using namespace nd;
  const int rc = attn_check(dtype, batch, sq, sk, hq, hkv, head_dim, scale);
  if (rc != ND_OK) return rc;
  if (batch == 0 || (sq == 0 && sk == 0)) return ND_OK;
  if (sq == 0 || sk == 0) {  // nothing to attend with, or to: zero gradients
    const size_t n = static_cast<size_t>(batch) * head_dim * 2;
    cudaStream_t zs = static_cast<cudaStream_t>(stream);
    if (sq == 0 ? (!dk || !dv) : !dq) return ND_ERR_BAD_ARG;
    cudaError_t e = cudaSuccess;
    if (sq == 0) {
      e = cudaMemsetAsync(dk, 0, n * sk * hkv, zs);
      if (e == cudaSuccess) e = cudaMemsetAsync(dv, 0, n * sk * hkv, zs);
    } else {
      e = cudaMemsetAsync(dq, 0, n * sq * hq, zs);
    }
    if (e == cudaSuccess) return ND_OK;
    set_last_cuda_error(e);
    (void)cudaGetLastError();
    return ND_ERR_LAUNCH;
  }
  if (!dout || !q || !k || !v || !out || !lse || !dq || !dk || !dv || !strides || (key_mask && kv_lens)) return ND_ERR_BAD_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  BwdArgs a{};
  a.s = attn_shape(batch, sq, sk, hq, hkv, head_dim);
  bwd_plan(a);
  if (static_cast<long long>(a.s.sq) * a.s.gp > (1 << 30)) return ND_ERR_UNSUPPORTED;
  const long long q_items = static_cast<long long>(a.s.batch) * a.s.hb * a.s.qtiles;
  const long long k_items = static_cast<long long>(a.s.batch) * a.s.hkv * a.s.ktiles * a.splits;
  if (q_items > INT32_MAX / 2 || k_items > INT32_MAX / 2) return ND_ERR_UNSUPPORTED;
  for (const void* p : {dout, q, k, v, out, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv),
                        static_cast<const void*>(lse)})
    if (!aligned16(p)) return ND_ERR_UNSUPPORTED;
  for (int i = 0; i < 12; ++i)
    if (strides[i] < 0 || strides[i] % 8 != 0) return ND_ERR_UNSUPPORTED;
  if (ws == nullptr || ws_bytes < bwd_ws(a) || !aligned16(ws)) return ND_ERR_WORKSPACE;
  a.mask = AttnMask{static_cast<const unsigned char*>(key_mask), kv_lens};
  a.sink = WaitSink{nullptr, device_error_ptr()};
  a.lse = lse;
  a.delta = static_cast<float*>(ws);
  a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + bwd_delta_bytes(a.s));
  a.out = out;
  a.dout = dout;
  a.do_b = strides[9]; a.do_s = strides[10]; a.do_h = strides[11];
  a.scale = scale;
  a.c = scale * 1.4426950408889634f;
  CUtensorMap mq, mdo, mk, mv, mdq, mdk, mdv;
  const int64_t ro = hq * head_dim, rk = hkv * head_dim;
  if (!attn_map(&mq, dtype, q, batch, sq, hq, head_dim, strides[0], strides[1], strides[2], 64, a.s.gp, kTile / a.s.gp) ||
      !attn_map(&mdo, dtype, dout, batch, sq, hq, head_dim, strides[9], strides[10], strides[11], 64, a.s.gp, kTile / a.s.gp) ||
      !attn_map(&mk, dtype, k, batch, sk, hkv, head_dim, strides[3], strides[4], strides[5], 64, 1, kTile) ||
      !attn_map(&mv, dtype, v, batch, sk, hkv, head_dim, strides[6], strides[7], strides[8], 64, 1, kTile) ||
      !attn_map(&mdq, dtype, dq, batch, sq, hq, head_dim, sq * ro, ro, head_dim, 32, a.s.gp, 32 / a.s.gp) ||
      !attn_map(&mdk, dtype, dk, batch, sk, hkv, head_dim, sk * rk, rk, head_dim, 32, 1, 32) ||
      !attn_map(&mdv, dtype, dv, batch, sk, hkv, head_dim, sk * rk, rk, head_dim, 32, 1, 32))
    return ND_ERR_LAUNCH;
  const bool bf = dtype == ND_BF16, one = head_dim <= 64;
  const size_t smem = (one ? sizeof(BwdSmem<1>) : sizeof(BwdSmem<2>)) + 1024;
  const int sms = sm_count();
  const void* f1 = one ? (bf ? (const void*)attn_dq_kernel<1, __nv_bfloat16> : (const void*)attn_dq_kernel<1, __half>)
                       : (bf ? (const void*)attn_dq_kernel<2, __nv_bfloat16> : (const void*)attn_dq_kernel<2, __half>);
  const void* f2 = one ? (bf ? (const void*)attn_dkv_kernel<1, __nv_bfloat16> : (const void*)attn_dkv_kernel<1, __half>)
                       : (bf ? (const void*)attn_dkv_kernel<2, __nv_bfloat16> : (const void*)attn_dkv_kernel<2, __half>);
  a.items = static_cast<int>(q_items);
  void* p1[] = {&mq, &mdo, &mk, &mv, &mdq, &a};
  int e = attn_launch(f1, a.items < sms ? a.items : sms, kBwdThreads, smem, p1, st);
  if (e != ND_OK) return e;
  a.items = static_cast<int>(k_items);
  void* p2[] = {&mq, &mdo, &mk, &mv, &mdk, &mdv, &a};
  e = attn_launch(f2, a.items < sms ? a.items : sms, kBwdThreads, smem, p2, st);
  if (e != ND_OK || a.splits == 1) return e;
  long long n4 = static_cast<long long>(batch) * sk * rk / 4;
  const float* part = a.part;
  void* p3[] = {&part, &dk, &dv, &n4, &a.splits};
  return attn_launch(bf ? (const void*)attn_dkv_join_kernel<__nv_bfloat16> : (const void*)attn_dkv_join_kernel<__half>,
                     static_cast<int>((2 * n4 + 255) / 256), 256, 0, p3, st);
}

}  // extern "C"
