// Attention forward (sm_100a): out = softmax(scale q k^T) v over the keys that take part, one pass over the keys with the
// running maximum and sum of the softmax.
//
// One persistent CTA per SM, 384 threads: warps 0-3 and 4-7 hold one query tile of 128 rows each (a thread owns a row),
// warp 8 copies (TMA), warp 9 issues the MMAs (two more complete its warpgroup, which hands registers to the softmax:
// 8 x 32 x 216 + 4 x 32 x 72 = 384 x 168, what the CTA is launched with). Per tile of KT keys and query tile
//   S = Q K^T      both operands from shared memory, fp32 into KT TMEM columns
//   softmax        the row's KT scores in registers; P = 2^(S c - m c) in 16 bits into KT / 2 columns
//   O += P V       A from tensor memory, V read where it lies (MN-major), fp32 into dn columns
// Both query tiles share the key tiles. S and P have columns of their own, so S(j + 1) is issued as soon as S(j) is in
// registers and is there when its softmax begins: with P over S's columns the chain softmax - O - S left both warpgroups
// waiting half of the time (4000 cycles per 128 keys and two tiles at D = 72, where the exponentials alone take 2048).
// Tensor memory holds 512 columns, 2 (KT + KT / 2 + dn) of which are used: KT is the largest multiple of 16 that fits,
// 128 keys for heads up to 64 dimensions, 112 up to 80, 96 up to 112, 80 for 128.
// The maximum. Only its order of magnitude matters: any m gives the same quotient as long as nothing overflows, and
// 16-bit floats hold a weight of 2^20 with the same relative error as one of 1. So a tile's weights are computed under the
// maximum as it stands, chunk by chunk while the scores arrive, and their sum tells afterwards whether it was far too
// small (then it is raised, O and the sum are rescaled and the weights computed again). Only an item's first tile and
// tiles with masked keys look for their maximum first.
// Two of eight pairs of exponentials go to the multiply-add units: the special-function unit gives 16 a clock.
// P is rounded to the element type for the second product (at most 2^-8 or 2^-11 of a weight, unbiased: averaged
// over the keys no more than the rounding of the output); scores, sums and O stay in 32 bits.
// Work items are (sample, head block, pair of query tiles, range of keys); the range is the whole length unless there
// are fewer items than SMs: then partial (O, log-sum-exp) go through the workspace to a second small kernel.
// Bound: the exponentials, 240 us of the special-function unit at 4 x 16 heads x 4096^2 x 72 bf16 where the products take
// 188; measured 445 us, 695 TFLOP/s. Tensor pipe and special-function unit are each busy 30 - 40 % of the time: the rest
// is the chain scores - softmax - weights of a tile, of which an SM holds two. 32 x 16 heads x 256 x 77 x 72 (one key
// tile): 29 us, of which loads, one softmax and the stores are a chain without overlap inside an item.
#include "attn.cuh"

namespace nd {

constexpr int kFwdThreads = 384;
constexpr int kPoly = 2;       // of eight pairs of exponentials, how many go to the multiply-add units
// Sum of a tile's weights up to which the maximum is left as it is: far from the end of the 32-bit sums, and for fp16
// every single weight stays below 65504.
template <typename T> constexpr float kRaise = std::is_same<T, __half>::value ? 16384.f : 1099511627776.f;

inline int fwd_key_tile(int dn) { return dn <= 64 ? 128 : (dn <= 80 ? 112 : (dn <= 112 ? 96 : 80)); }

template <int NB, int KT> struct __align__(1024) FwdSmem {
  static constexpr int kKv = NB == 1 ? 8 : 4;  // key / value tiles in flight
  uint8_t q[2][NB * kBlkBytes];
  uint8_t kv[kKv][NB * KT * 128];
  uint8_t out[8][(NB == 1 ? 2 : KT == 112 ? 3 : 4) * kStageBytes];  // every warp's rows
  int lens[kLens];
  uint64_t q_full, q_empty;
  uint64_t kv_full[kKv], kv_empty[kKv];
  uint64_t s_full[2], s_free[2], p_full[2], o_done[2];
  uint32_t tmem_base;
  int abort_flag;
};

struct FwdArgs {
  AttnShape s;
  AttnMask mask;
  WaitSink sink;
  float* lse;      // [batch, hb, rows_pad], minus log2 of the sum of 2^(score c); nullable
  float* part_o;   // splits > 1: [splits][batch * hb][rows_pad][d], normalised
  float* part_l;   // splits > 1: [splits][batch * hb][rows_pad], -inf: no keys
  float c;         // scale * log2(e)
  int pairs, splits, ktiles, tiles_per_split;
  int items;
};

struct FwdItem {
  int b, hb, pair, split, t0, n_t, n_keys;  // key tiles [t0, t0 + n_t)
  bool two;                                 // the pair's second tile has rows
};

template <int KT> __device__ __forceinline__ FwdItem fwd_item(const FwdArgs& a, const int* lens, int item, int lane) {
  FwdItem w;
  w.split = item % a.splits;
  int r = item / a.splits;
  w.pair = r % a.pairs;
  r /= a.pairs;
  w.hb = r % a.s.hb;
  w.b = r / a.s.hb;
  w.two = 2 * w.pair + 1 < a.s.qtiles;
  w.n_keys = lens != nullptr ? lens[w.b] : key_count(a.mask, w.b, a.s.sk, lane);
  const int all = (w.n_keys + KT - 1) / KT;
  w.t0 = w.split * a.tiles_per_split;
  const int left = all - w.t0;
  w.n_t = left < 0 ? 0 : (left < a.tiles_per_split ? left : a.tiles_per_split);
  return w;
}

template <int NB, int KT, typename T>
__global__ void __launch_bounds__(kFwdThreads, 1)
attn_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o, const FwdArgs a) {
  using Smem = FwdSmem<NB, KT>;
  constexpr int kKv = Smem::kKv;
  constexpr int kQBytes = NB * kBlkBytes, kKvBytes = NB * KT * 128;
  constexpr int kCh = KT / 16;  // chunks of 16 keys
  extern __shared__ uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort_flag;

  if (threadIdx.x == 0) {
    mbar_init(&s.q_full, 1);
    mbar_init(&s.q_empty, 1);
    for (int i = 0; i < kKv; ++i) {
      mbar_init(&s.kv_full[i], 1);
      mbar_init(&s.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.s_free[i], 4);
      mbar_init(&s.p_full[i], 4);
      mbar_init(&s.o_done[i], 1);
    }
    s.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) tmem_alloc<512>(&s.tmem_base);
  griddep_launch_dependents();
  griddep_wait();
  const int* lens = lens_cached(a.mask, a.s.batch, a.s.sk) ? s.lens : nullptr;
  if (lens != nullptr) fill_lens(s.lens, a.mask, a.s.batch, a.s.sk, warp, kFwdThreads / 32, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;

  const int group_blocks = a.s.hb / a.s.hkv;  // head blocks per key head
  const int pos_per_tile = kTile / a.s.gp;
  constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  const uint32_t tm_p = tmem + 2 * KT, tm_o = tmem + 3 * KT;  // S of tile t at t * KT, P at t * KT / 2, O at t * dn

  if (warp >= 8) {
   reg_give<72>();
   if (warp == 8) {
    // ------------------------------------------------------------------ copies (one thread)
    int it = 0, q_cnt = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const FwdItem w = fwd_item<KT>(a, lens, item, lane);
      if (w.n_t == 0) continue;
      if (lane == 0) {
        const int kvh = w.hb / group_blocks;
        ok = mbar_wait(&s.q_empty, (q_cnt & 1) ^ 1, abort_flag, a.sink, 101);
        if (ok) {
          mbar_expect_tx(&s.q_full, (w.two ? 2 : 1) * kQBytes);
          for (int t = 0; t < (w.two ? 2 : 1); ++t)
            load_tile<NB>(s.q[t], &map_q, &s.q_full, w.hb * a.s.gp, (2 * w.pair + t) * pos_per_tile, w.b);
        }
        for (int j = 0; j < 2 * w.n_t && ok; ++j) {  // K(0), V(0), K(1), ...
          const int slot = (it + j) % kKv;
          ok = mbar_wait(&s.kv_empty[slot], (((it + j) / kKv) & 1) ^ 1, abort_flag, a.sink, 102);
          if (!ok) break;
          mbar_expect_tx(&s.kv_full[slot], kKvBytes);
          load_tile<NB, KT>(s.kv[slot], (j & 1) ? &map_v : &map_k, &s.kv_full[slot], kvh, (w.t0 + (j >> 1)) * KT, w.b);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      it += 2 * w.n_t;
      ++q_cnt;
    }
    if (!ok) settle();
   } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA issue (one elected thread)
    const int ksteps = a.s.dn / 16;
    const uint32_t id_o = attn_idesc(kFmt, a.s.dn, true);
    const uint64_t q_desc = desc_k(smem_u32(s.q[0])), k_desc = desc_k(smem_u32(s.kv[0])), v_desc = desc_mn<KT>(smem_u32(s.kv[0]));
    with_steps(ksteps, [&](auto ks) {
    int it = 0, q_cnt = 0;
    uint32_t base[2] = {0, 0};  // key tiles of the items before, per query tile
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const FwdItem w = fwd_item<KT>(a, lens, item, lane);
      if (w.n_t == 0) continue;
      const int nt = w.two ? 2 : 1;
      if (elect_one()) {
        ok = mbar_wait(&s.q_full, q_cnt & 1, abort_flag, a.sink, 103);
        // Step j, one query tile after the other: S(j + 1), then O(j). Their softmaxes run half a step apart, and what one
        // of them waits for must not stand behind the other's. (Polling for whichever comes first costs this thread more
        // than the fixed order: a pass over the barriers takes it longer than an MMA group runs.)
        for (int j = -1; j < w.n_t && ok; ++j) {
          const int v_at = it + 2 * j + 1, k_at = v_at + 1;
          const int s_left = w.n_keys - (w.t0 + j + 1) * KT, o_left = s_left + KT;
          const uint32_t id_s = attn_idesc(kFmt, s_left >= KT ? KT : (s_left + 15) & ~15, false);
          const int steps = o_left >= KT ? kCh : (o_left + 15) >> 4;
          const bool more = j + 1 < w.n_t;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t >= nt || !ok) break;
            if (more) {
              if (t == 0) ok = mbar_wait(&s.kv_full[k_at % kKv], (k_at / kKv) & 1, abort_flag, a.sink, 106);
              const uint32_t n = base[t] + j + 1;  // scores of this tile so far
              if (ok && n > 0) ok = mbar_wait(&s.s_free[t], (n - 1) & 1, abort_flag, a.sink, 104);
              if (!ok) break;
              tc_fence_after();
              issue_nt<decltype(ks)::value, KT>(tmem + t * KT, q_desc + t * (kQBytes >> 4), k_desc + (k_at % kKv) * (kKvBytes >> 4), ksteps, id_s);
              mma_commit(&s.s_full[t]);
              if (t == nt - 1) {
                mma_commit(&s.kv_empty[k_at % kKv]);
                if (j + 2 == w.n_t) mma_commit(&s.q_empty);  // the last scores of the item
              }
            }
            if (j >= 0) {
              if (t == 0) ok = mbar_wait(&s.kv_full[v_at % kKv], (v_at / kKv) & 1, abort_flag, a.sink, 113);
              if (ok) ok = mbar_wait(&s.p_full[t], (base[t] + j) & 1, abort_flag, a.sink, 105);
              if (!ok) break;
              tc_fence_after();
              issue_tn<kCh, kCh>(tm_o + t * a.s.dn, tm_p + t * (KT / 2), 0, v_desc + (v_at % kKv) * (kKvBytes >> 4), steps, id_o,
                            j > 0 ? 1u : 0u);
              mma_commit(&s.o_done[t]);
              if (t == nt - 1) mma_commit(&s.kv_empty[v_at % kKv]);
            }
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      it += 2 * w.n_t;
      base[0] += w.n_t;
      if (w.two) base[1] += w.n_t;
      ++q_cnt;
    }
    });
    __syncwarp();
   }
  } else {
    reg_take<216>();
    // ------------------------------------------------------------------ softmax and epilogue: a thread per row
    const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t ts = tmem + lanes + t * KT, tp = tm_p + lanes + t * (KT / 2), to = tm_o + lanes + t * a.s.dn;
    uint32_t cnt = 0;  // key tiles so far
    int it = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < a.items && ok; item += gridDim.x) {
      const FwdItem w = fwd_item<KT>(a, lens, item, lane);
      const int it0 = it;
      it += 2 * w.n_t;
      if (t == 1 && !w.two) continue;
      float m = -INFINITY, l = 0.f;  // maximum of the raw scores as used, sum of P
      const uint64_t c2 = f2_pack(a.c, a.c);
      float x[kCh][16];
      uint64_t sum[2];
      auto weights = [&](int i, uint64_t base2) {  // P of chunk i
        uint32_t pk[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint64_t y = f2_fma(f2_pack(x[i][2 * e], x[i][2 * e + 1]), c2, base2);
          float2 p;
          if (e < kPoly) {
            p = exp2_poly(y);
          } else {
            const float2 z = f2_unpack(y);
            p = make_float2(ex2_approx(z.x), ex2_approx(z.y));
          }
          sum[e & 1] = f2_add(sum[e & 1], f2_pack(p.x, p.y));
          pk[e] = pack2<T>(p.x, p.y);
        }
        tc_st8(tp + i * 8, pk);
      };
      auto total = [&]() {
        const float2 v = f2_unpack(f2_add(sum[0], sum[1]));
        return v.x + v.y;
      };
      auto minus_max = [&]() {
        const float base = m == -INFINITY ? 0.f : m * a.c;
        return f2_pack(-base, -base);
      };
      // raises the maximum to that of x; O follows, if there is any yet
      auto raise_max = [&](bool have_o) {
        float mx[4] = {m, m, m, m};
#pragma unroll
        for (int i = 0; i < kCh; ++i)
#pragma unroll
          for (int e = 0; e < 16; e += 2) mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], x[i][e], x[i][e + 1]);
        const float m_new = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
        const float alpha = m == -INFINITY ? 0.f : ex2_approx((m - m_new) * a.c);
        m = m_new;
        l *= alpha;
        if (have_o) {
          for (int c = 0; c < a.s.dn; c += 16) {
            float o[16];
            tc_ld16(to + c, o);
            tc_wait_ld();
            uint32_t u[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * alpha);
            tc_st16(to + c, u);
          }
        }
      };
      for (int j = 0; j < w.n_t; ++j, ++cnt) {
        const bool whole = a.mask.key_mask == nullptr && (w.t0 + j + 1) * KT <= w.n_keys;  // all of its keys take part
        ok = warp_wait(&s.s_full[t], cnt & 1, abort_flag, a.sink, 107);
        if (!ok) break;
        tc_fence_after();
        sum[0] = sum[1] = 0;
        if (__builtin_expect(whole && j > 0, 1)) {
          // Weights under the maximum as it stands, while the scores still arrive; looked at afterwards.
          tc_ld16(ts, x[0]);
          const uint64_t base2 = minus_max();
          ok = warp_wait(&s.o_done[t], (cnt - 1) & 1, abort_flag, a.sink, 109);  // O(j - 1) is complete, P(j - 1) read
          if (!ok) break;
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < kCh; ++i) {
            if (i + 1 < kCh) tc_ld16(ts + (i + 1) * 16, x[i + 1]);
            weights(i, base2);
            if (i + 1 < kCh) tc_wait_ld();
            if (i + 2 == kCh) {  // the scores are in registers
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&s.s_free[t]);
            }
          }
          if (__builtin_expect(__any_sync(0xffffffffu, !(total() <= kRaise<T>)), 0)) {
            tc_wait_st();  // the weights just written are written again
            raise_max(true);
            sum[0] = sum[1] = 0;
            const uint64_t again = minus_max();
#pragma unroll
            for (int i = 0; i < kCh; ++i) weights(i, again);
          }
        } else {
          const int left = w.n_keys - (w.t0 + j) * KT;
          const int n_ch = left >= KT ? kCh : (left + 15) >> 4;  // the others were not even computed
#pragma unroll
          for (int i = 0; i < kCh; ++i) tc_ld16(ts + i * 16, x[i]);
          tc_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.s_free[t]);
          bool clear = false;  // this thread's key of the tile takes no part
          if (a.mask.key_mask != nullptr) {
            uint32_t bits[4];
            key_bits<KT>(a.mask, w.b, a.s.sk, w.n_keys, w.t0 + j, lane, bits);
#pragma unroll
            for (int i = 0; i < kCh; ++i)
#pragma unroll
              for (int e = 0; e < 16; ++e) x[i][e] = (bits[i >> 1] >> ((i & 1) * 16 + e)) & 1u ? x[i][e] : -INFINITY;
            clear = r < KT && !((bits[quarter] >> lane) & 1u);
          } else if (left < KT) {  // the end of the keys: one chunk is cut, those behind it are not looked at
#pragma unroll
            for (int i = 0; i < kCh; ++i) {
              if (left - i * 16 < 16) {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[i][e] = e < left - i * 16 ? x[i][e] : -INFINITY;
              }
            }
            clear = r < n_ch * 16 && r >= left;
          }
          // O(j) of tile 1 is issued after that of tile 0: one warpgroup's clearing serves both
          if (t == 0 && __any_sync(0xffffffffu, clear)) {
            const int v_at = it0 + 2 * j + 1;
            ok = warp_wait(&s.kv_full[v_at % kKv], (v_at / kKv) & 1, abort_flag, a.sink, 108);
            if (!ok) break;
            if (clear) clear_row<NB, KT>(s.kv[v_at % kKv], r);
            fence_proxy_async_smem();
          }
          if (j > 0) {
            ok = warp_wait(&s.o_done[t], (cnt - 1) & 1, abort_flag, a.sink, 111);
            if (!ok) break;
            tc_fence_after();
          }
          raise_max(j > 0);
          const uint64_t base2 = minus_max();
#pragma unroll
          for (int i = 0; i < kCh; ++i)
            if (i < n_ch) weights(i, base2);
        }
        l += total();
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[t]);
      }
      if (!ok) break;
      if (w.n_t > 0) {
        ok = warp_wait(&s.o_done[t], (cnt - 1) & 1, abort_flag, a.sink, 110);
        if (!ok) break;
        tc_fence_after();
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int row = (2 * w.pair + t) * kTile + r;
      const long long head_row = static_cast<long long>(w.b) * a.s.hb + w.hb;
      if (a.splits > 1) {
        const long long at = (static_cast<long long>(w.split) * a.s.batch * a.s.hb + head_row) * a.s.rows_pad + row;
        a.part_l[at] = l == 0.f ? -INFINITY : m * a.c + log2f(l);
        if (w.n_t > 0) {
          for (int c = 0; c < a.s.dn; c += 16) {
            float o[16];
            tc_ld16(to + c, o);
            tc_wait_ld();
            float4* dst = reinterpret_cast<float4*>(a.part_o + at * a.s.d + c);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (c + e * 4 < a.s.d && row < a.s.rows)
                dst[e] = make_float4(o[4 * e] * inv, o[4 * e + 1] * inv, o[4 * e + 2] * inv, o[4 * e + 3] * inv);
          }
        }
      } else {
        if (a.lse != nullptr)  // -inf where there is nothing: 2^(s - inf) = 0 in the backward pass
          a.lse[head_row * a.s.rows_pad + row] = (l == 0.f || row >= a.s.rows) ? -INFINITY : -(m * a.c + log2f(l));
        const int pos = (2 * w.pair + t) * pos_per_tile + quarter * 32 / a.s.gp;
        if (lane == 0) bulk_wait_read_all();  // the blocks of the item before have left
        __syncwarp();
#pragma unroll
        for (int c = 0; c < static_cast<int>(sizeof(s.out[0])) / kStageBytes * 32; c += 32) {
          if (c >= a.s.d) break;
          float o[2][16];
          tc_ld16(to + c, o[0]);
          if (c + 16 < a.s.dn) tc_ld16(to + c + 16, o[1]);  // (columns behind dn are clipped when the block is stored)
          tc_wait_ld();
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = l == 0.f ? 0.f : o[e >> 4][e & 15] * inv;
          stage_block<T>(s.out[warp] + c / 32 * kStageBytes, v, lane);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && pos < a.s.sq) {
          for (int c = 0; c < a.s.d; c += 32) tma_store_4d(&map_o, s.out[warp] + c / 32 * kStageBytes, c, w.hb * a.s.gp, pos, w.b);
          bulk_commit();
        }
      }
      tc_fence_before();  // these reads of O come before the next item's products
    }
    if (lane == 0) bulk_wait_all();  // this warp's blocks are written before the CTA may exit
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_free<512>(tmem);
}

// Joins the key ranges of a row: weights 2^(lse_i - max), a warp per row.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const FwdArgs a, T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const long long rows_all = static_cast<long long>(a.s.batch) * a.s.hb * a.s.rows_pad;
  const long long at = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  griddep_wait();
  if (at >= rows_all) return;
  const long long head_row = at / a.s.rows_pad;
  const int row = static_cast<int>(at - head_row * a.s.rows_pad);
  float top = -INFINITY;
  for (int i = lane; i < a.splits; i += 32) top = fmaxf(top, a.part_l[i * rows_all + at]);
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float total = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < a.splits; ++i) {
    const float li = a.part_l[i * rows_all + at];
    if (li == -INFINITY) continue;  // no keys: its O was never written
    const float wgt = ex2_approx(li - top);
    total += wgt;
    if (lane * 4 < a.s.d && row < a.s.rows) {
      const float4 o = *reinterpret_cast<const float4*>(a.part_o + (i * rows_all + at) * a.s.d + lane * 4);
      acc.x = fmaf(wgt, o.x, acc.x);
      acc.y = fmaf(wgt, o.y, acc.y);
      acc.z = fmaf(wgt, o.z, acc.z);
      acc.w = fmaf(wgt, o.w, acc.w);
    }
  }
  if (lane == 0 && a.lse != nullptr) a.lse[at] = (total == 0.f || row >= a.s.rows) ? -INFINITY : -(top + log2f(total));
  if (row >= a.s.rows || lane * 4 >= a.s.d) return;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int b = static_cast<int>(head_row / a.s.hb), hb = static_cast<int>(head_row - static_cast<long long>(b) * a.s.hb);
  const int pos = row / a.s.gp, g = row - pos * a.s.gp;
  T* dst = out + ((static_cast<long long>(b) * a.s.sq + pos) * a.s.hq + hb * a.s.gp + g) * a.s.d + lane * 4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
}

// ------------------------------------------------------------------ host side
static void fwd_plan(FwdArgs& a) {
  a.pairs = (a.s.qtiles + 1) / 2;
  const int kt = fwd_key_tile(a.s.dn);
  a.ktiles = (a.s.sk + kt - 1) / kt;
  const long long items = static_cast<long long>(a.s.batch) * a.s.hb * a.pairs;
  const int sms = sm_count();
  a.splits = 1;
  if (items < sms && a.ktiles > 1) {
    const int want = static_cast<int>(sms / items);
    a.splits = want < a.ktiles ? want : a.ktiles;
  }
  a.tiles_per_split = (a.ktiles + a.splits - 1) / a.splits;
  if (a.tiles_per_split < 1) a.tiles_per_split = 1;
  a.splits = (a.ktiles + a.tiles_per_split - 1) / a.tiles_per_split;
  if (a.splits < 1) a.splits = 1;
}

static size_t fwd_ws(const FwdArgs& a) {
  if (a.splits <= 1) return 0;
  return static_cast<size_t>(a.splits) * a.s.batch * a.s.hb * a.s.rows_pad * (a.s.d + 1) * sizeof(float);
}

template <typename T> static const void* pick_fwd(int kt) {
  switch (kt) {
    case 128: return (const void*)attn_fwd_kernel<1, 128, T>;
    case 112: return (const void*)attn_fwd_kernel<2, 112, T>;
    case 96: return (const void*)attn_fwd_kernel<2, 96, T>;
    default: return (const void*)attn_fwd_kernel<2, 80, T>;
  }
}

int attn_launch(const void* fn, dim3 grid, int threads, size_t smem, void** params, cudaStream_t st) {
  RelaxedCapture relaxed;  // the attribute and a first launch load the kernel's module
  if (smem > 0) {
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) {
      set_last_cuda_error(e);
      (void)cudaGetLastError();
      return ND_ERR_LAUNCH;
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelExC(&cfg, fn, params);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    (void)cudaGetLastError();
    return ND_ERR_LAUNCH;
  }
  return ND_OK;
}

}  // namespace nd

extern "C" {

int64_t nd_attn_lse_floats(int64_t batch, int64_t sq, int64_t hq, int64_t hkv) {
  if (batch <= 0 || sq <= 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || batch > 65535 || hq > 65535 || sq > (1 << 25)) return 0;
  const nd::AttnShape s = nd::attn_shape(batch, sq, 1, hq, hkv, 8);
  return static_cast<int64_t>(s.batch) * s.hb * s.rows_pad;
}

size_t nd_attn_fwd_ws_bytes(int64_t batch, int64_t sq, int64_t sk, int64_t hq, int64_t hkv, int64_t head_dim) {
  if (nd::attn_check(ND_BF16, batch, sq, sk, hq, hkv, head_dim, 1.f) != ND_OK || batch == 0 || sq == 0) return 0;
  nd::FwdArgs a{};
  a.s = nd::attn_shape(batch, sq, sk, hq, hkv, head_dim);
  if (nd::attn_few_takes(a.s)) return nd::attn_few_ws(a.s);
  nd::fwd_plan(a);
  return nd::fwd_ws(a);
}

int nd_attn_fwd(int dtype, const void* q, const void* k, const void* v, void* out, float* lse, const void* key_mask,
                const int* kv_lens, int64_t batch, int64_t sq, int64_t sk, int64_t hq, int64_t hkv, int64_t head_dim,
                const int64_t* strides, float scale, void* ws, size_t ws_bytes, void* stream) {
  using namespace nd;
  const int rc = attn_check(dtype, batch, sq, sk, hq, hkv, head_dim, scale);
  if (rc != ND_OK) return rc;
  if (batch == 0 || sq == 0) return ND_OK;
  if (!q || !out || !strides || (sk > 0 && (!k || !v)) || (key_mask && kv_lens)) return ND_ERR_BAD_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  FwdArgs a{};
  a.s = attn_shape(batch, sq, sk, hq, hkv, head_dim);
  if (static_cast<long long>(a.s.sq) * a.s.gp > (1 << 30)) return ND_ERR_UNSUPPORTED;
  if (!aligned16(q) || !aligned16(out) || (sk > 0 && (!aligned16(k) || !aligned16(v)))) return ND_ERR_UNSUPPORTED;
  if (!attn_strides_ok(strides, batch, sq, hq) || !attn_strides_ok(strides + 3, batch, sk, hkv) ||
      !attn_strides_ok(strides + 6, batch, sk, hkv))
    return ND_ERR_UNSUPPORTED;
  const AttnMask mask{static_cast<const unsigned char*>(key_mask), kv_lens};
  const float c = scale * 1.4426950408889634f;
  if (attn_few_takes(a.s)) {
    const size_t need = attn_few_ws(a.s);
    if (need > 0 && (ws == nullptr || ws_bytes < need || !aligned16(ws))) return ND_ERR_WORKSPACE;
    return attn_few(dtype, q, k, v, out, lse, mask, a.s, strides, c, ws, st);
  }
  fwd_plan(a);
  const long long items = static_cast<long long>(a.s.batch) * a.s.hb * a.pairs * a.splits;
  if (items > INT32_MAX / 2) return ND_ERR_UNSUPPORTED;
  if (fwd_ws(a) > 0 && (ws == nullptr || ws_bytes < fwd_ws(a) || !aligned16(ws))) return ND_ERR_WORKSPACE;
  a.items = static_cast<int>(items);
  a.mask = mask;
  a.sink = WaitSink{nullptr, device_error_ptr()};
  a.lse = lse;
  a.c = c;
  a.part_o = static_cast<float*>(ws);
  a.part_l = a.splits > 1 ? a.part_o + static_cast<size_t>(a.splits) * a.s.batch * a.s.hb * a.s.rows_pad * a.s.d : nullptr;
  CUtensorMap mq, mk, mv, mo;
  const int64_t ro = hq * head_dim;
  const void* kb = sk > 0 ? k : q;  // never read without keys; a map needs an address
  const void* vb = sk > 0 ? v : q;
  const int64_t sk1 = sk > 0 ? sk : 1;
  const int kt = fwd_key_tile(a.s.dn);
  if (!attn_map(&mq, dtype, q, batch, sq, hq, head_dim, strides[0], strides[1], strides[2], 64, a.s.gp, kTile / a.s.gp) ||
      !attn_map(&mk, dtype, kb, batch, sk1, hkv, head_dim, strides[3], strides[4], strides[5], 64, 1, kt) ||
      !attn_map(&mv, dtype, vb, batch, sk1, hkv, head_dim, strides[6], strides[7], strides[8], 64, 1, kt) ||
      !attn_map(&mo, dtype, out, batch, sq, hq, head_dim, sq * ro, ro, head_dim, 32, a.s.gp, 32 / a.s.gp))
    return ND_ERR_LAUNCH;
  const bool bf = dtype == ND_BF16;
  const void* fn = bf ? pick_fwd<__nv_bfloat16>(kt) : pick_fwd<__half>(kt);
  const size_t smem = (kt == 128  ? sizeof(FwdSmem<1, 128>)
                       : kt == 112 ? sizeof(FwdSmem<2, 112>)
                       : kt == 96  ? sizeof(FwdSmem<2, 96>)
                                   : sizeof(FwdSmem<2, 80>)) + 1024;
  const int sms = sm_count();
  void* params[] = {&mq, &mk, &mv, &mo, &a};
  int e = attn_launch(fn, dim3(a.items < sms ? a.items : sms), kFwdThreads, smem, params, st);
  if (e != ND_OK || a.splits == 1) return e;
  const long long rows_all = static_cast<long long>(a.s.batch) * a.s.hb * a.s.rows_pad;
  void* jp[] = {&a, &out};
  return attn_launch(bf ? (const void*)attn_join_kernel<__nv_bfloat16> : (const void*)attn_join_kernel<__half>,
                     dim3(static_cast<unsigned>((rows_all + 7) / 8)), 256, 0, jp, st);
}

}  // extern "C"
