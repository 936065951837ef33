// Attention backward (sm_100a). With P = 2^(S c - lse) recomputed from the saved log-sum-exp,
//   delta = rowsum(dO * O),  dP = dO V^T,  dS = P (dP - delta),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
// in two kernels. One holds a query tile and walks the keys (dQ, and delta on the way), the other holds a key tile and
// walks the queries of all heads that share it (dK, dV). Recomputing S and dP for both costs two products more than one
// kernel that adds dQ up in global memory, but every sum stays in tensor memory in one fixed order: no atomics, results
// do not change from run to run, and the second operand of every product is a tile that lies in shared memory already.
//
// Both: one persistent CTA per SM, 640 threads, warps 0-15 the elementwise part, warp 16 copies, warp 17 issues the MMAs (two
// more complete its warpgroup, which hands registers over: 16 x 32 x 104 + 4 x 32 x 64 = 640 x 96). A thread has a row and
// 32 of the tile's 128 columns. Each half of the columns (two warpgroups) has products and barriers of its own, and the
// issuing thread takes the halves half a step apart: while one waits for its products the other computes. P and dS are
// the A operands of the last products straight from tensor memory, in 16 bits (one rounding, unbiased, below that of the
// output); scores, dP, statistics and accumulators stay in 32 bits.
//
// dQ kernel, per key tile j and half:  S(j) = Q K^T, dP(j) = dO V^T, dQ += dS(j) K. S(j + 1) is issued as soon as S(j) is
// in registers, dP(j + 1) behind dQ(j). delta comes from the row's dO and O tiles - or, where a sample has one key tile,
// from P and dP, exactly and without O: with few keys the rounding of O is what would be left of dS.
// dK/dV kernel, per query tile i and half (everything transposed: lanes are keys):  S(i) = K Q^T, dP(i) = V dO^T,
// dV += P(i) dO, dK += dS(i) Q. P lies over S's columns and dS over dP's; S(i + 1) is issued behind dV(i) while dS(i) is
// computed, dP(i + 1) behind dK(i) while the next exponentials run. Rows of masked keys hold anything: a row of A only
// reaches its own row of the product, and those rows are written as zeros.
//
// Bound: the tensor cores (seven products cannot be done without, the forward's two included: 292 us at 2 x 16 heads x
// 4096^2 x 64 bf16; nine are computed). Measured 848 us, forward included, 567 TFLOP/s by the seven. Tensor pipe 26 % (dQ) and 34 % (dK/dV) busy, issue slots a third: what is
// left are the waits for tensor-memory loads and stores and for the barriers between the products. 16 x 16 heads x 1024
// queries x 300 keys x 72: 260 us forward and backward.
//
// fp16. Weights below 2^-14 and gradients far from 1 would fall out of its range: P goes into its product times a power
// of two (the length's, at most 2^12), dS times a power of two that brings the largest |dO| (of the row for dQ, of the
// rows that share a key head for dK) to 1/16; the accumulators are scaled back.
#include "attn.cuh"

namespace nd {

constexpr int kBwdThreads = 640;

struct BwdArgs {
  AttnShape s;
  AttnMask mask;
  WaitSink sink;
  const float* lse;   // [batch, hb, rows_pad]: minus the log-sum-exp
  float* delta;       // [batch, hb, rows_pad]: minus delta
  float* peak;        // fp16: [batch, hb, rows_pad], largest |dO| of a row
  float* part;        // dK/dV, splits > 1: [splits][2][B * Sk * Hkv][D]
  float c, scale;
  float p_shift;      // fp16, dK/dV: log2 of the factor on P
  int items;
  int splits, steps, steps_per_split;  // dK/dV: query tiles of all head blocks of a key head
};

template <int NB> struct __align__(1024) BwdSmem {
  static constexpr int kRing = NB == 1 ? 8 : 4;
  uint8_t res[2][NB * kBlkBytes];        // dQ: Q, dO; dK/dV: K, V
  uint8_t ring[kRing][NB * kBlkBytes];   // dQ: K, V, K, V, ...; dK/dV: Q, dO, ...
  // staging of the first half's warps, which write the results: block c of 32 rows holds columns 32 c .., the fourth goes
  // where the second was
  uint8_t out[4][(NB == 1 ? 2 : 3) * kStageBytes];
  int lens[kLens];
  union {
    alignas(16) float stat[kRing / 2][2][kTile];  // dK/dV: log-sum-exp and delta of the query tile
    float2 red[2][4][kTile];                      // dQ: [exchange parity][warpgroup][row]
  };
  uint64_t res_full, res_empty;
  uint64_t full[kRing], empty[kRing];
  uint64_t s_full[2], dp_full[2];   // MMA -> elementwise, per half
  uint64_t p_full[2], ds_full[2];   // elementwise -> MMA (dQ: p_full = "S is in registers")
  uint64_t ds_free[2];              // dQ: dS has been read
  uint64_t acc_done;                // the accumulators are complete
  uint64_t o_read;                  // dQ: the elementwise warps have read dO and O
  uint64_t swap[4];                 // dQ: the four warps of 32 rows have written to `red`
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
  for (int h = 0; h < 2; ++h) {
    mbar_init(&s.s_full[h], 1);
    mbar_init(&s.dp_full[h], 1);
    mbar_init(&s.p_full[h], 8);
    mbar_init(&s.ds_full[h], 8);
    mbar_init(&s.ds_free[h], 1);
  }
  for (int i = 0; i < 4; ++i) mbar_init(&s.swap[i], 4);
  mbar_init(&s.acc_done, 1);
  mbar_init(&s.o_read, 16);
  s.abort_flag = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

// fp16: the power of two that brings `peak` to 2^-4 (1 where there is nothing to scale)
__device__ __forceinline__ float grad_factor(float peak) {
  if (!(peak > 0.f) || isinf(peak)) return 1.f;
  const int e = static_cast<int>((__float_as_uint(peak) >> 23) & 255u) - 127;  // peak is a 16-bit value: a normal number
  return __uint_as_float(static_cast<uint32_t>(127 - 4 - e) << 23);
}

// largest |value| of four 16-bit pairs
template <typename T> __device__ __forceinline__ float peak8(const uint4& v, float top) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = unpack_pair<T>(w[e]);
    top = max3(top, fabsf(f.x), fabsf(f.y));
  }
  return top;
}

// 32 rows x 32 columns from `c` on, through the block of their own and to the copy engine
template <typename T>
__device__ __forceinline__ void put_block(const CUtensorMap* map, uint8_t* out, const float (&v)[32], int lane, int c, int head,
                                          int pos, int b, bool inside) {
  if (c == 96) {
    if (lane == 0) bulk_wait_read_all();
    __syncwarp();
  }
  uint8_t* stage = out + (c == 96 ? 1 : c / 32) * kStageBytes;
  stage_block<T>(stage, v, lane);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0 && inside) {
    tma_store_4d(map, stage, c, head, pos, b);
    bulk_commit();
  }
}

// ------------------------------------------------------------------ dQ
// TMEM columns: S 0, dP 128, dS 256 (32 columns of 16-bit pairs per half), dQ 384
template <int NB, typename T>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
               const __grid_constant__ CUtensorMap map_o, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_dq, const BwdArgs a) {
  constexpr int kRing = BwdSmem<NB>::kRing;
  constexpr int kTileBytes = NB * kBlkBytes;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  BwdSmem<NB>& s = *reinterpret_cast<BwdSmem<NB>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort_flag;
  if (threadIdx.x == 0) bwd_init<NB>(s);
  if (warp == 17) tmem_alloc<512>(&s.tmem_base);
  griddep_launch_dependents();
  griddep_wait();
  const bool cached = lens_cached(a.mask, a.s.batch, a.s.sk);
  if (cached) fill_lens(s.lens, a.mask, a.s.batch, a.s.sk, warp, kBwdThreads / 32, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;

  const int group_blocks = a.s.hb / a.s.hkv;
  const int pos_per_tile = kTile / a.s.gp;
  constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  struct Item {
    int b, hb, qt, n_keys, n_t;
    int o;      // 1: an O tile comes first in the ring
    int n1;     // key tiles of the second half (the last one may have no keys there)
  };
  auto get = [&](int item) {
    Item w;
    w.qt = item % a.s.qtiles;
    const int r = item / a.s.qtiles;
    w.hb = r % a.s.hb;
    w.b = r / a.s.hb;
    w.n_keys = cached ? s.lens[w.b] : key_count(a.mask, w.b, a.s.sk, lane);
    w.n_t = (w.n_keys + kTile - 1) / kTile;
    w.n1 = (w.n_keys + 63) / kTile;
    w.o = w.n_t > 1 ? 1 : 0;
    return w;
  };

  if (warp >= 16) {
   reg_give<64>();
   if (warp == 16) {
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
        for (int j = -w.o; j < 2 * w.n_t && ok; ++j) {  // (O,) K(0), V(0), K(1), ...
          const int at = it + w.o + j, slot = at % kRing;
          ok = mbar_wait(&s.empty[slot], ((at / kRing) & 1) ^ 1, abort_flag, a.sink, 122);
          if (!ok) break;
          mbar_expect_tx(&s.full[slot], kTileBytes);
          if (j < 0) load_tile<NB>(s.ring[slot], &map_o, &s.full[slot], w.hb * a.s.gp, w.qt * pos_per_tile, w.b);
          else load_tile<NB>(s.ring[slot], (j & 1) ? &map_v : &map_k, &s.full[slot], w.hb / group_blocks, (j >> 1) * kTile, w.b);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      it += w.o + 2 * w.n_t;
      ++cnt;
    }
    if (!ok) settle();
   } else if (warp == 17) {
    const int ksteps = a.s.dn / 16;
    const uint32_t id_o = attn_idesc(kFmt, a.s.dn, true);
    const uint64_t res = desc_k(smem_u32(s.res[0])), ring = desc_k(smem_u32(s.ring[0])), ring_mn = desc_mn<>(smem_u32(s.ring[0]));
    constexpr uint32_t kStep = kTileBytes >> 4;
    constexpr uint32_t kHalfRows = 64 * 128 >> 4;  // the second half of a tile's rows
    with_steps(ksteps, [&](auto ks) {
    int it = 0, cnt = 0, o_cnt = 0;
    uint32_t done[2] = {0, 0};  // key tiles of the items before, per half
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const Item w = get(item);
      if (w.n_t == 0) continue;
      if (elect_one()) {
        const int n_h[2] = {w.n_t, w.n1};
        const int it1 = it + w.o;
        auto keys = [&](int j, int h) {  // of this half, in 16s
          const int left = w.n_keys - j * kTile - h * 64;
          return left >= 64 ? 64 : (left + 15) & ~15;
        };
        auto wait = [&](uint64_t* bar, uint32_t n, int code) {
          if (ok) ok = mbar_wait(bar, n & 1, abort_flag, a.sink, code);
          return ok;
        };
        auto full = [&](int at, int code) { return wait(&s.full[at % kRing], static_cast<uint32_t>(at / kRing), code); };
        auto issue_s = [&](int j, int h) {
          const int k_at = it1 + 2 * j;
          if (!full(k_at, 125)) return;
          tc_fence_after();
          issue_nt<decltype(ks)::value>(tmem + h * 64, res, ring + (k_at % kRing) * kStep + h * kHalfRows, ksteps, attn_idesc(kFmt, keys(j, h), false));
          mma_commit(&s.s_full[h]);
        };
        auto issue_dp = [&](int j, int h) {
          const int v_at = it1 + 2 * j + 1;
          if (!full(v_at, 127)) return;
          tc_fence_after();
          issue_nt<decltype(ks)::value>(tmem + 128 + h * 64, res + kStep, ring + (v_at % kRing) * kStep + h * kHalfRows, ksteps,
                   attn_idesc(kFmt, keys(j, h), false));
          mma_commit(&s.dp_full[h]);
        };
        auto issue_dq = [&](int j, int h) {
          const int k_at = it1 + 2 * j;
          tc_fence_after();
          issue_tn<4, 4>(tmem + 384, tmem + 256 + h * 32, 0, ring_mn + (k_at % kRing) * kStep + h * kHalfRows, keys(j, h) / 16, id_o,
                      (j > 0 || h > 0) ? 1u : 0u);
          mma_commit(&s.ds_free[h]);
        };
        // the ends of a key tile: its V has been read by both halves' dP, its K by both halves' dQ
        auto end_v = [&](int j) {
          mma_commit(&s.empty[(it1 + 2 * j + 1) % kRing]);
          if (j + 1 == w.n_t) mma_commit(&s.res_empty);
        };
        auto end_k = [&](int j) {
          mma_commit(&s.empty[(it1 + 2 * j) % kRing]);
          if (j + 1 == w.n_t) mma_commit(&s.acc_done);
        };
        wait(&s.res_full, static_cast<uint32_t>(cnt), 123);
        for (int h = 0; h < 2; ++h)
          if (n_h[h] > 0 && ok) issue_s(0, h);
        for (int h = 0; h < 2; ++h)
          if (n_h[h] > 0 && ok) issue_dp(0, h);
        if (w.o || kHalf) {  // the rows' dO and O have been read: before either tile may be overwritten
          if (wait(&s.o_read, static_cast<uint32_t>(o_cnt), 133) && w.o) mbar_arrive(&s.empty[it % kRing]);
        }
        if (ok) end_v(0);
        for (int j = 0; j < w.n_t && ok; ++j) {
          const bool more0 = j + 1 < n_h[0], more1 = j + 1 < n_h[1];
          // half 1 has dS(j - 1); first, because K(j + 1) may need the place of K(j - 1)
          if (j > 0) {
            if (!wait(&s.ds_full[1], done[1] + j - 1, 126)) break;
            issue_dq(j - 1, 1);
            end_k(j - 1);
            if (j < n_h[1]) issue_dp(j, 1);
            if (!ok) break;
            end_v(j);
          }
          // half 0 has S(j) in registers
          if (!wait(&s.p_full[0], done[0] + j, 124)) break;
          if (more0) issue_s(j + 1, 0);
          // half 0 has dS(j)
          if (!wait(&s.ds_full[0], done[0] + j, 134)) break;
          issue_dq(j, 0);
          if (more0) issue_dp(j + 1, 0);
          // half 1 has S(j) in registers
          if (j < n_h[1]) {
            if (!wait(&s.p_full[1], done[1] + j, 135)) break;
            if (more1) issue_s(j + 1, 1);
          }
        }
        if (ok) {
          if (n_h[1] == w.n_t) {
            if (wait(&s.ds_full[1], done[1] + w.n_t - 1, 136)) issue_dq(w.n_t - 1, 1);
          }
          if (ok) end_k(w.n_t - 1);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      it += w.o + 2 * w.n_t;
      done[0] += w.n_t;
      done[1] += w.n1;
      o_cnt += (w.o || kHalf) ? 1 : 0;
      ++cnt;
    }
    });
    __syncwarp();
   }
  } else {
    reg_take<104>();
    const int half = warp >> 3, sub = (warp >> 2) & 1, group = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem + lanes + group * 32, t_dp = t_s + 128, t_ds = tmem + lanes + 256 + group * 16, t_dq = tmem + lanes + 384;
    uint32_t cnt = 0;  // key tiles of this half so far: the phase of every per-tile barrier
    uint32_t items = 0;
    int it = 0;
    bool ok = true;
    // sums over the four threads of a row, once per item
    auto exchange = [&](float2 v, float2& sum) -> bool {
      s.red[items & 1][group][r] = v;
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.swap[quarter]);
      if (!warp_wait(&s.swap[quarter], items & 1, abort_flag, a.sink, 139)) return false;
      const float2* red = s.red[items & 1][0] + r;
      sum.x = (red[0].x + red[kTile].x) + (red[2 * kTile].x + red[3 * kTile].x);
      sum.y = (red[0].y + red[kTile].y) + (red[2 * kTile].y + red[3 * kTile].y);
      return true;
    };
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const Item w = get(item);
      const int it1 = it + w.o;
      const int row = w.qt * kTile + r;
      const long long at = (static_cast<long long>(w.b) * a.s.hb + w.hb) * a.s.rows_pad + row;
      float nlse = -INFINITY, ndelta = 0.f, peak = 0.f;
      if (w.n_t > 0) {
        nlse = __ldg(a.lse + at);
        if (w.o || kHalf) {  // the row's dO (and O), 16 bytes of each at a time; chunk c of row r lies at c ^ (r & 7)
          ok = warp_wait(&s.res_full, items & 1, abort_flag, a.sink, 137);
          if (ok && w.o) ok = warp_wait(&s.full[it % kRing], (it / kRing) & 1, abort_flag, a.sink, 138);
          if (!ok) break;
          for (int c = kHalf ? 0 : group; c < a.s.d / 8; c += kHalf ? 1 : 4) {  // a quarter each; fp16 looks at the whole row
            const int off = (c >> 3) * kBlkBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
            const uint4 g = *reinterpret_cast<const uint4*>(s.res[1] + off);
            if constexpr (kHalf) peak = peak8<T>(g, peak);
            if (w.o && (!kHalf || (c & 3) == group)) {
              const uint4 o = *reinterpret_cast<const uint4*>(s.ring[it % kRing] + off);
              const uint32_t gs[4] = {g.x, g.y, g.z, g.w}, os[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 fg = unpack_pair<T>(gs[e]), fo = unpack_pair<T>(os[e]);
                ndelta = fmaf(-fg.x, fo.x, ndelta);
                ndelta = fmaf(-fg.y, fo.y, ndelta);
              }
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.o_read);
        }
        if (w.o || (half == 1 && w.n1 == 0)) {  // (the second: nothing to add to the one tile's sum below)
          float2 sum;
          ok = exchange(make_float2(ndelta, 0.f), sum);
          if (!ok) break;
          ndelta = sum.x;
        }
      }
      const float factor = kHalf ? grad_factor(peak) : 1.f;
      const int mine = half == 0 ? w.n_t : w.n1;
      const uint64_t c2 = f2_pack(a.c, a.c), nlse2 = f2_pack(nlse, nlse);
      for (int j = 0; j < mine; ++j, ++cnt) {
        const int col = j * kTile + group * 32, left = w.n_keys - col;  // this thread's columns
        uint32_t bits = left >= 32 ? 0xffffffffu : (left <= 0 ? 0u : (1u << left) - 1u);
        if (a.mask.key_mask != nullptr) bits = key_word(a.mask, w.b, a.s.sk, w.n_keys, col, lane);
        ok = warp_wait(&s.s_full[half], cnt & 1, abort_flag, a.sink, 128);
        if (!ok) break;
        tc_fence_after();
        float p[32];
        tc_ld32(t_s, p);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[half]);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 y = f2_unpack(f2_fma(f2_pack(p[e], p[e + 1]), c2, nlse2));
          p[e] = ex2_approx(y.x);
          p[e + 1] = ex2_approx(y.y);
        }
        ok = warp_wait(&s.dp_full[half], cnt & 1, abort_flag, a.sink, 130);
        if (!ok) break;
        tc_fence_after();
        float dp[32];
        tc_ld32(t_dp, dp);
        tc_wait_ld();
        if (bits != 0xffffffffu) {  // S and dP of a masked key may be anything, NaN included
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            p[e] = (bits >> e) & 1u ? p[e] : 0.f;
            dp[e] = (bits >> e) & 1u ? dp[e] : 0.f;
          }
          // ... and its row of K must not reach the last product: the 32 rows of this warpgroup's columns
          const int k_at = it1 + 2 * j;
          ok = warp_wait(&s.full[k_at % kRing], (k_at / kRing) & 1, abort_flag, a.sink, 129);
          if (!ok) break;
          if (quarter == 0 && !((bits >> lane) & 1u)) clear_row<NB>(s.ring[k_at % kRing], group * 32 + lane);
          fence_proxy_async_smem();
        }
        if (!w.o) {  // one key tile: delta = sum of P dP over the row's keys, over the sum of P (1 but for its last bits)
          uint64_t acc = 0, norm = 0;
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            acc = f2_fma(f2_pack(p[e], p[e + 1]), f2_pack(dp[e], dp[e + 1]), acc);
            norm = f2_add(norm, f2_pack(p[e], p[e + 1]));
          }
          const float2 v = f2_unpack(acc), n = f2_unpack(norm);
          float2 sum;
          ok = exchange(make_float2(v.x + v.y, n.x + n.y), sum);
          if (!ok) break;
          ndelta = sum.y > 0.f ? -sum.x / sum.y : -sum.x;
        }
        uint32_t pk[16];
        const uint64_t nd2 = f2_pack(ndelta * factor, ndelta * factor), factor2 = f2_pack(factor, factor);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const uint64_t x = f2_pack(dp[e], dp[e + 1]);
          const uint64_t d = kHalf ? f2_fma(x, factor2, nd2) : f2_add(x, nd2);
          const float2 ds = f2_unpack(f2_mul(f2_pack(p[e], p[e + 1]), d));
          pk[e / 2] = pack2<T>(ds.x, ds.y);
        }
        if (cnt > 0) {
          ok = warp_wait(&s.ds_free[half], (cnt - 1) & 1, abort_flag, a.sink, 131);
          if (!ok) break;
          tc_fence_after();
        }
        tc_st16(t_ds, pk);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.ds_full[half]);
      }
      if (!ok) break;
      it = it1 + 2 * w.n_t;
      if (group == 0) {
        a.delta[at] = ndelta;
        if constexpr (kHalf) a.peak[at] = peak;
      }
      if (w.n_t > 0) {
        ++items;
        ok = warp_wait(&s.acc_done, (items - 1) & 1, abort_flag, a.sink, 132);
        if (!ok) break;
        tc_fence_after();
      }
      if (half == 0) {  // its next dS is what the next item's first product waits for
        const float mul = a.scale / factor;
        const int pos = w.qt * pos_per_tile + quarter * 32 / a.s.gp;
        if (lane == 0) bulk_wait_read_all();  // the blocks of the item before have left
        __syncwarp();
        for (int c = sub * 32; c < a.s.d; c += 64) {
          float o[32];
          tc_ld32(t_dq + c, o);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = w.n_t == 0 ? 0.f : o[e] * mul;
          put_block<T>(&map_dq, s.out[quarter], o, lane, c, w.hb * a.s.gp, pos, w.b, pos < a.s.sq);
        }
        tc_fence_before();
      }
    }
    if (half == 0 && lane == 0) bulk_wait_all();  // this warp's blocks are written before the CTA may exit
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 17) tmem_free<512>(tmem);
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
  constexpr bool kHalf = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  BwdSmem<NB>& s = *reinterpret_cast<BwdSmem<NB>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort_flag;
  if (threadIdx.x == 0) bwd_init<NB>(s);
  if (warp == 17) tmem_alloc<512>(&s.tmem_base);
  griddep_launch_dependents();
  griddep_wait();
  const bool cached = lens_cached(a.mask, a.s.batch, a.s.sk);
  if (cached) fill_lens(s.lens, a.mask, a.s.batch, a.s.sk, warp, kBwdThreads / 32, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;

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
    w.n_keys = cached ? s.lens[w.b] : key_count(a.mask, w.b, a.s.sk, lane);
    w.i0 = w.split * a.steps_per_split;
    w.n_i = a.steps - w.i0 < a.steps_per_split ? a.steps - w.i0 : a.steps_per_split;
    if (w.kt * kTile >= w.n_keys || w.n_i < 0) w.n_i = 0;
    return w;
  };

  if (warp >= 16) {
   reg_give<64>();
   if (warp == 16) {
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
   } else if (warp == 17) {
    const int ksteps = a.s.dn / 16;
    const uint32_t id_s = attn_idesc(kFmt, 64, false), id_o = attn_idesc(kFmt, a.s.dn, true);
    const uint64_t res = desc_k(smem_u32(s.res[0])), ring = desc_k(smem_u32(s.ring[0])), ring_mn = desc_mn<>(smem_u32(s.ring[0]));
    constexpr uint32_t kStep = kTileBytes >> 4;
    constexpr uint32_t kHalfRows = 64 * 128 >> 4;  // the second half of a tile's rows
    with_steps(ksteps, [&](auto ks) {
    int it = 0, cnt = 0;
    uint32_t done = 0;  // query tiles of the items before
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const Item w = get(item);
      if (w.n_i == 0) continue;
      if (elect_one()) {
        auto wait = [&](uint64_t* bar, uint32_t n, int code) {
          if (ok) ok = mbar_wait(bar, n & 1, abort_flag, a.sink, code);
          return ok;
        };
        auto full = [&](int at, int code) { return wait(&s.full[at % kRing], static_cast<uint32_t>(at / kRing), code); };
        auto issue_s = [&](int i, int h) {
          const int q_at = it + 2 * i;
          if (!full(q_at, 146)) return;
          tc_fence_after();
          issue_nt<decltype(ks)::value>(tmem + h * 64, res, ring + (q_at % kRing) * kStep + h * kHalfRows, ksteps, id_s);
          mma_commit(&s.s_full[h]);
        };
        auto issue_dp = [&](int i, int h) {
          const int d_at = it + 2 * i + 1;
          if (!full(d_at, 148)) return;
          tc_fence_after();
          issue_nt<decltype(ks)::value>(tmem + 128 + h * 64, res + kStep, ring + (d_at % kRing) * kStep + h * kHalfRows, ksteps, id_s);
          mma_commit(&s.dp_full[h]);
          if (h == 1 && i + 1 == w.n_i) mma_commit(&s.res_empty);
        };
        // acc += A(i) of half h times the rows of that half of the tile in ring position `at`
        auto issue_acc = [&](uint32_t acc, uint32_t src, int at, int i, int h) {
          tc_fence_after();
          issue_tn<4, 2>(acc, src + h * 64, 32, ring_mn + (at % kRing) * kStep + h * kHalfRows, 4, id_o, (i > 0 || h > 0) ? 1u : 0u);
        };
        wait(&s.res_full, static_cast<uint32_t>(cnt), 144);
        for (int h = 0; h < 2; ++h)
          if (ok) issue_s(0, h);
        for (int h = 0; h < 2; ++h)
          if (ok) issue_dp(0, h);
        for (int i = 0; i < w.n_i && ok; ++i) {
          const int q_at = it + 2 * i, d_at = q_at + 1;
          const bool more = i + 1 < w.n_i;
          if (i > 0) {  // first, because Q(i + 1) may need the place of Q(i - 1)
            if (!wait(&s.ds_full[1], done + i - 1, 147)) break;
            issue_acc(tmem + 384, tmem + 128, q_at - 2, i - 1, 1);
            mma_commit(&s.empty[(q_at - 2) % kRing]);  // Q(i - 1)
            issue_dp(i, 1);
          }
          if (!wait(&s.p_full[0], done + i, 145)) break;
          issue_acc(tmem + 256, tmem, d_at, i, 0);  // dV += P(i) dO(i), then S(i + 1) over P(i)
          if (more) issue_s(i + 1, 0);
          if (!wait(&s.ds_full[0], done + i, 153)) break;
          issue_acc(tmem + 384, tmem + 128, q_at, i, 0);  // dK += dS(i) Q(i), then dP(i + 1) over dS(i)
          if (more) issue_dp(i + 1, 0);
          if (!wait(&s.p_full[1], done + i, 154)) break;
          issue_acc(tmem + 256, tmem, d_at, i, 1);
          mma_commit(&s.empty[d_at % kRing]);  // dO(i)
          if (more) issue_s(i + 1, 1);
        }
        if (wait(&s.ds_full[1], done + w.n_i - 1, 155)) {
          issue_acc(tmem + 384, tmem + 128, it + 2 * (w.n_i - 1), w.n_i - 1, 1);
          mma_commit(&s.empty[(it + 2 * (w.n_i - 1)) % kRing]);
          mma_commit(&s.acc_done);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      it += 2 * w.n_i;
      done += w.n_i;
      ++cnt;
    }
    });
    __syncwarp();
   }
  } else {
    reg_take<104>();
    const int half = warp >> 3, sub = (warp >> 2) & 1, group = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem + lanes + group * 32, t_dp = t_s + 128, t_dv = tmem + lanes + 256, t_dk = tmem + lanes + 384;
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
        mine = ((quarter < 2 ? (quarter == 0 ? bits[0] : bits[1]) : (quarter == 2 ? bits[2] : bits[3])) >> lane) & 1u;
      }
      float factor = 1.f;  // fp16: on dS
      if constexpr (kHalf) {
        if (w.n_i > 0) {
          float top = 0.f;
          for (int i = 0; i < a.steps; ++i) {
            const int sub_block = i / a.s.qtiles, qt = i - sub_block * a.s.qtiles;
            const float4 v = __ldg(reinterpret_cast<const float4*>(
                a.peak + (static_cast<long long>(w.b) * a.s.hb + w.h * group_blocks + sub_block) * a.s.rows_pad + qt * kTile) + lane);
            top = max3(max3(top, v.x, v.y), v.z, v.w);
          }
#pragma unroll
          for (int d = 16; d >= 1; d >>= 1) top = max3(top, __shfl_xor_sync(0xffffffffu, top, d), top);
          factor = grad_factor(top);
        }
      }
      const float p_up = kHalf ? exp2f(a.p_shift) : 1.f;
      const uint64_t c2 = f2_pack(a.c, a.c), shift2 = f2_pack(a.p_shift, a.p_shift);
      const uint64_t fac2 = f2_pack(factor / p_up, factor / p_up);
      const bool any = __any_sync(0xffffffffu, mine);  // a warp without keys leaves its rows as they are: zeros are written
      for (int i = 0; i < w.n_i; ++i, ++cnt) {
        const int qa = it0 + 2 * i;
        ok = warp_wait(&s.full[qa % kRing], (qa / kRing) & 1, abort_flag, a.sink, 149);  // the statistics have landed
        if (!ok) break;
        const ulonglong2* st_l = reinterpret_cast<const ulonglong2*>(s.stat[(qa % kRing) / 2][0]) + group * 8;
        const ulonglong2* st_d = reinterpret_cast<const ulonglong2*>(s.stat[(qa % kRing) / 2][1]) + group * 8;
        ok = warp_wait(&s.s_full[half], cnt & 1, abort_flag, a.sink, 150);
        if (!ok) break;
        tc_fence_after();
        float p[32];
        uint32_t pk[16];
        if (any) {
          tc_ld32(t_s, p);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const ulonglong2 l4 = st_l[e / 4];
            const uint64_t la = kHalf ? f2_add(l4.x, shift2) : l4.x, lb = kHalf ? f2_add(l4.y, shift2) : l4.y;
            const float2 ya = f2_unpack(f2_fma(f2_pack(p[e], p[e + 1]), c2, la));
            const float2 yb = f2_unpack(f2_fma(f2_pack(p[e + 2], p[e + 3]), c2, lb));
            p[e] = ex2_approx(ya.x);
            p[e + 1] = ex2_approx(ya.y);
            p[e + 2] = ex2_approx(yb.x);
            p[e + 3] = ex2_approx(yb.y);
            pk[e / 2] = pack2<T>(p[e], p[e + 1]);
            pk[e / 2 + 1] = pack2<T>(p[e + 2], p[e + 3]);
          }
          tc_st16(t_s, pk);
          tc_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[half]);
        ok = warp_wait(&s.dp_full[half], cnt & 1, abort_flag, a.sink, 151);
        if (!ok) break;
        tc_fence_after();
        if (any) {
          float dp[32];
          tc_ld32(t_dp, dp);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const ulonglong2 d4 = st_d[e / 4];
            uint64_t da = f2_add(f2_pack(dp[e], dp[e + 1]), d4.x), db = f2_add(f2_pack(dp[e + 2], dp[e + 3]), d4.y);
            if constexpr (kHalf) {
              da = f2_mul(da, fac2);
              db = f2_mul(db, fac2);
            }
            const float2 sa = f2_unpack(f2_mul(f2_pack(p[e], p[e + 1]), da));
            const float2 sb = f2_unpack(f2_mul(f2_pack(p[e + 2], p[e + 3]), db));
            pk[e / 2] = pack2<T>(sa.x, sa.y);
            pk[e / 2 + 1] = pack2<T>(sb.x, sb.y);
          }
          tc_st16(t_dp, pk);
          tc_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.ds_full[half]);
      }
      if (!ok) break;
      if (half == 1) continue;
      if (w.n_i > 0) {
        ok = warp_wait(&s.acc_done, done & 1, abort_flag, a.sink, 152);
        if (!ok) break;
        ++done;
        tc_fence_after();
      }
      // dV, then dK, 32 columns at a time; this half's next P and dS are what the next item's first products wait for
      const int key = w.kt * kTile + r;
      for (int which = 0; which < 2; ++which) {
        if (lane == 0) bulk_wait_read_all();  // the blocks before have left
        __syncwarp();
        const uint32_t src = which == 0 ? t_dv : t_dk;
        const float mul = which == 0 ? 1.f / p_up : a.scale / factor;
        for (int c = sub * 32; c < a.s.d; c += 64) {
          float o[32];
          tc_ld32(src + c, o);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = mine ? o[e] * mul : 0.f;
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
            put_block<T>(which == 0 ? &map_dv : &map_dk, s.out[quarter], o, lane, c, w.h, k0, w.b, k0 < a.s.sk);
          }
        }
      }
      tc_fence_before();
    }
    if (half == 0 && lane == 0) bulk_wait_all();  // this warp's blocks are written before the CTA may exit
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 17) tmem_free<512>(tmem);
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

static size_t bwd_stat_bytes(const AttnShape& s) {  // delta, and the row peaks of fp16
  return 2 * static_cast<size_t>(s.batch) * s.hb * s.rows_pad * sizeof(float);
}
static size_t bwd_ws(const BwdArgs& a) {
  size_t n = bwd_stat_bytes(a.s);
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
  if (!attn_strides_ok(strides, batch, sq, hq) || !attn_strides_ok(strides + 3, batch, sk, hkv) ||
      !attn_strides_ok(strides + 6, batch, sk, hkv) || !attn_strides_ok(strides + 9, batch, sq, hq))
    return ND_ERR_UNSUPPORTED;
  if (ws == nullptr || ws_bytes < bwd_ws(a) || !aligned16(ws)) return ND_ERR_WORKSPACE;
  a.mask = AttnMask{static_cast<const unsigned char*>(key_mask), kv_lens};
  a.sink = WaitSink{nullptr, device_error_ptr()};
  a.lse = lse;
  a.delta = static_cast<float*>(ws);
  a.peak = a.delta + static_cast<size_t>(a.s.batch) * a.s.hb * a.s.rows_pad;
  a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + bwd_stat_bytes(a.s));
  for (int n = a.s.sk; dtype == ND_F16 && n > 1 && a.p_shift < 12.f; n >>= 1) a.p_shift += 1.f;
  a.scale = scale;
  a.c = scale * 1.4426950408889634f;
  CUtensorMap mq, mdo, mo, mk, mv, mdq, mdk, mdv;
  const int64_t ro = hq * head_dim, rk = hkv * head_dim;
  if (!attn_map(&mq, dtype, q, batch, sq, hq, head_dim, strides[0], strides[1], strides[2], 64, a.s.gp, kTile / a.s.gp) ||
      !attn_map(&mdo, dtype, dout, batch, sq, hq, head_dim, strides[9], strides[10], strides[11], 64, a.s.gp, kTile / a.s.gp) ||
      !attn_map(&mo, dtype, out, batch, sq, hq, head_dim, sq * ro, ro, head_dim, 64, a.s.gp, kTile / a.s.gp) ||
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
  void* p1[] = {&mq, &mdo, &mo, &mk, &mv, &mdq, &a};
  int e = attn_launch(f1, dim3(a.items < sms ? a.items : sms), kBwdThreads, smem, p1, st);
  if (e != ND_OK) return e;
  a.items = static_cast<int>(k_items);
  void* p2[] = {&mq, &mdo, &mk, &mv, &mdk, &mdv, &a};
  e = attn_launch(f2, dim3(a.items < sms ? a.items : sms), kBwdThreads, smem, p2, st);
  if (e != ND_OK || a.splits == 1) return e;
  long long n4 = static_cast<long long>(batch) * sk * rk / 4;
  const float* part = a.part;
  void* p3[] = {&part, &dk, &dv, &n4, &a.splits};
  return attn_launch(bf ? (const void*)attn_dkv_join_kernel<__nv_bfloat16> : (const void*)attn_dkv_join_kernel<__half>,
                     dim3(static_cast<unsigned>((2 * n4 + 255) / 256)), 256, 0, p3, st);
}

}  // extern "C"
