// Attention of a few query rows per key head (a decoding step): the keys and values are read once, and that is all the
// work there is - with one row a 128-row MMA tile is empty but for a line, and its softmax one busy warp.
//
// LPK lanes (the head's dimensions in 16-byte pieces, rounded up to a power of two) hold one key: its piece of K, then of
// V, and the query rows' pieces in fp32. A score is 8 products per lane and a sum over the LPK lanes; every group of LPK
// lanes ("slot") keeps its own running maximum, sum and output over the keys it sees, kFewUnroll of them at a time so that
// 2 x kFewUnroll 16-byte loads are in flight per lane and the rescaling is paid once for all of them. Slots and warps are
// joined at the end. Weights are never rounded; everything is 32-bit until the output.
//
// A CTA takes (sample, key head, range of keys): the sample's own keys cut evenly into as many ranges as it takes to give
// every SM several CTAs. More than one range: normalised partial outputs and their log-sum-exp go through the workspace
// to a second kernel. Bound: HBM (K and V once): 32 x 20 heads x
// up to 1500 keys x 64, one token: 30 us, 0.63 of the copy rate; one query, one key: 6.4 - 6.8 us, the launch.
#include "attn.cuh"

namespace nd {

constexpr int kFewThreads = 128;
// CTAs per SM, by rows: what the registers of R query rows, their outputs and the loads in flight leave without spills
template <int R> constexpr int kFewCtas = R == 1 ? 6 : R == 2 ? 5 : 3;
constexpr int kFewUnroll = 4;
constexpr int kFewRows = 4;  // query rows per key head this kernel takes

struct FewArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;     // nullable, in the order of the tile kernels
  float* part_o;  // [splits][batch][hkv][rows][d]
  float* part_l;  // [splits][batch][hkv][rows]
  AttnShape s;
  AttnMask mask;
  long long st[9];
  float c;
  int group, rows, splits;
};

// row r of key head h of sample b: its place in the padded order of the backward pass
__device__ __forceinline__ long long lse_at(const FewArgs& a, int b, int h, int r) {
  const int pos = r / a.group, head = h * a.group + r % a.group;
  return (static_cast<long long>(b) * a.s.hb + head / a.s.gp) * a.s.rows_pad + pos * a.s.gp + head % a.s.gp;
}

// the rows that pad a head block to whole tiles count as empty
__device__ __forceinline__ void pad_lse(const FewArgs& a, int b, int h) {
  if (a.lse == nullptr) return;
  const int blocks = a.group / a.s.gp, pad = a.s.rows_pad - a.s.rows;
  for (int i = threadIdx.x; i < blocks * pad; i += blockDim.x)
    a.lse[(static_cast<long long>(b) * a.s.hb + h * blocks + i / pad) * a.s.rows_pad + a.s.rows + i % pad] = -INFINITY;
}

template <typename T> __device__ __forceinline__ void unpack8(const uint4& w, uint64_t (&f)[4]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 p = unpack_pair<T>(u[e]);
    f[e] = f2_pack(p.x, p.y);
  }
}

template <typename T, int LPK, int R>
__global__ void __launch_bounds__(kFewThreads, kFewCtas<R>) attn_few_kernel(const FewArgs a) {
  constexpr int kSlots = 32 / LPK;                          // keys per warp and step
  constexpr int kStep = kFewThreads / 32 * kSlots;          // keys per CTA and unrolled step
  __shared__ alignas(8) float sh_o[kFewThreads / 32][R][LPK * 8];
  __shared__ float sh_m[kFewThreads / 32][R], sh_l[kFewThreads / 32][R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = lane % LPK, slot = lane / LPK;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  griddep_launch_dependents();
  griddep_wait();
  const bool mine = piece * 8 < a.s.d;  // lanes behind the head's dimensions hold zeros
  uint4 qw[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    qw[r] = make_uint4(0, 0, 0, 0);
    if (r < a.rows && mine) {
      const int pos = r / a.group, head = h * a.group + r % a.group;
      qw[r] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.st[0] + pos * a.st[1] + head * a.st[2] + piece * 8));
    }
  }
  const int n_keys = key_count(a.mask, b, a.s.sk, lane);
  uint64_t q[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    unpack8<T>(qw[r], q[r]);
#pragma unroll
    for (int e = 0; e < 4; ++e) q[r][e] = f2_mul(q[r][e], f2_pack(a.c, a.c));
  }
  const int per = (n_keys + a.splits - 1) / a.splits;
  const int first = split * per, end = first + per < n_keys ? first + per : n_keys;
  const T* kp = static_cast<const T*>(a.k) + b * a.st[3] + h * a.st[5] + piece * 8;
  const T* vp = static_cast<const T*>(a.v) + b * a.st[6] + h * a.st[8] + piece * 8;
  const unsigned char* mask = a.mask.key_mask != nullptr ? a.mask.key_mask + static_cast<long long>(b) * a.s.sk : nullptr;
  // With one or two rows the R x kFewUnroll scores of a step lie spread over the LPK lanes: value i (row i / kFewUnroll, key
  // i % kFewUnroll) with the lanes of group i / kOwn, so a sum over the lanes is a few exchanges and a lane works out its own
  // weights only (2 x 8 heads x 50021 keys of 128, one row: 72 us, 78 with every weight on every lane; two rows: 76.5 / 77.2).
  // With four rows independent sums hide one another's latency and the longer chain costs more than it saves (four rows there:
  // 166 us against 139): every lane has all of them. Running maximum and sum are those of a lane's own values.
  constexpr int kVals = R * kFewUnroll, kGroups = R > 2 ? 1 : kVals < LPK ? kVals : LPK;
  constexpr int kOwn = kVals / kGroups, kRep = LPK / kGroups;                    // values per lane, lanes with the same ones
  constexpr int kOwnRows = kOwn > kFewUnroll ? kOwn / kFewUnroll : 1, kOwnKeys = kOwn / kOwnRows;
  constexpr int kRowLanes = kRep * (kFewUnroll / kOwnKeys);                      // lanes that share a row
  const int key0 = piece / kRep * kOwn % kFewUnroll;
  auto of_group = [](float x, int g) { return kGroups == 1 ? x : __shfl_sync(0xffffffffu, x, g * kRep, LPK); };
  float m[kOwnRows], l[kOwnRows];
#pragma unroll
  for (int i = 0; i < kOwnRows; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  uint64_t o[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[r][e] = 0;
  for (int k0 = first; k0 < end; k0 += kStep * kFewUnroll) {
    uint4 kw[kFewUnroll], vw[kFewUnroll];
    bool on[kFewUnroll];
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u) {
      const int key = k0 + u * kStep + warp * kSlots + slot;
      on[u] = key < end;
      kw[u] = vw[u] = make_uint4(0, 0, 0, 0);
      if (on[u] && mine) {
        kw[u] = __ldcs(reinterpret_cast<const uint4*>(kp + static_cast<long long>(key) * a.st[4]));
        vw[u] = __ldcs(reinterpret_cast<const uint4*>(vp + static_cast<long long>(key) * a.st[7]));
      }
      if (mask != nullptr && on[u]) on[u] = __ldg(mask + key) != 0;
    }
    float w[kVals];
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u) {
      uint64_t kf[4];
      unpack8<T>(kw[u], kf);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        uint64_t x = f2_mul(q[r][0], kf[0]);
#pragma unroll
        for (int e = 1; e < 4; ++e) x = f2_fma(q[r][e], kf[e], x);
        const float2 y = f2_unpack(x);
        w[r * kFewUnroll + u] = y.x + y.y;
      }
    }
    // sums over the lanes: as long as it has more than its own values a lane gives half of them away and keeps the other half
#pragma unroll
    for (int d = LPK / 2, n = kVals; d >= 1; d >>= 1) {
      if (n > kOwn) {
        n >>= 1;
        const bool upper = (piece & d) != 0;
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float give = upper ? w[i] : w[n + i];
          w[i] = (upper ? w[n + i] : w[i]) + __shfl_xor_sync(0xffffffffu, give, d);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) w[i] += __shfl_xor_sync(0xffffffffu, w[i], d);
      }
    }
    unsigned keep = 0;
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u) keep |= on[u] ? 1u << u : 0u;
    float alpha[kOwnRows];
    bool moved = false;
#pragma unroll
    for (int i = 0; i < kOwnRows; ++i) {
      float top = m[i];
#pragma unroll
      for (int u = 0; u < kOwnKeys; ++u) {
        float& x = w[i * kOwnKeys + u];
        x = keep >> (key0 + u) & 1 ? x : -INFINITY;
        top = max3(top, x, x);
      }
#pragma unroll
      for (int d = kRep; d < kRowLanes; d <<= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, top, d);
        top = max3(top, other, other);
      }
      const float base = top == -INFINITY ? 0.f : top;
      alpha[i] = ex2_approx(m[i] - base);
      moved |= alpha[i] != 1.f;
      m[i] = top;
      l[i] *= alpha[i];
#pragma unroll
      for (int u = 0; u < kOwnKeys; ++u) {
        float& x = w[i * kOwnKeys + u];
        x = ex2_approx(x - base);
        l[i] += x;
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float x = of_group(alpha[r * kFewUnroll % kOwn / kOwnKeys], r * kFewUnroll / kOwn);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][e] = f2_mul(o[r][e], f2_pack(x, x));
      }
    }
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u) {
      uint64_t vf[4];
      unpack8<T>(on[u] ? vw[u] : make_uint4(0, 0, 0, 0), vf);  // a key that takes no part may hold NaN
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int i = r * kFewUnroll + u;
        const float x = of_group(w[i % kOwn], i / kOwn);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][e] = f2_fma(f2_pack(x, x), vf[e], o[r][e]);
      }
    }
  }
  // every lane with the maximum and the sum of every row
#pragma unroll
  for (int i = 0; i < kOwnRows; ++i)
#pragma unroll
    for (int d = kRep; d < kRowLanes; d <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
  float rm[R], rl[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    rm[r] = of_group(m[r * kFewUnroll % kOwn / kOwnKeys], r * kFewUnroll / kOwn);
    rl[r] = of_group(l[r * kFewUnroll % kOwn / kOwnKeys], r * kFewUnroll / kOwn);
  }
  // the slots of a warp, then the warps
#pragma unroll
  for (int d = LPK; d < 32; d <<= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float mo = __shfl_xor_sync(0xffffffffu, rm[r], d), lo = __shfl_xor_sync(0xffffffffu, rl[r], d);
      const float top = max3(rm[r], mo, mo), base = top == -INFINITY ? 0.f : top;
      const float wa = ex2_approx(rm[r] - base), wb = ex2_approx(mo - base);
      rm[r] = top;
      rl[r] = rl[r] * wa + lo * wb;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[r][e] = f2_fma(__shfl_xor_sync(0xffffffffu, o[r][e], d), f2_pack(wb, wb), f2_mul(o[r][e], f2_pack(wa, wa)));
    }
  if (slot == 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<float2*>(&sh_o[warp][r][piece * 8 + 2 * e]) = f2_unpack(o[r][e]);
      if (piece == 0) {
        sh_m[warp][r] = rm[r];
        sh_l[warp][r] = rl[r];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.rows * a.s.d / 2; i += kFewThreads) {  // pairs of output elements
    const int r = i / (a.s.d / 2), e = (i - r * (a.s.d / 2)) * 2;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kFewThreads / 32; ++w) top = max3(top, sh_m[w][r], sh_m[w][r]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < kFewThreads / 32; ++w) {
      const float wgt = ex2_approx(sh_m[w][r] - base);
      sum = fmaf(sh_l[w][r], wgt, sum);
      x = fmaf(sh_o[w][r][e], wgt, x);
      y = fmaf(sh_o[w][r][e + 1], wgt, y);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (a.splits > 1) {
      const long long at = ((static_cast<long long>(split) * a.s.batch + b) * a.s.hkv + h) * a.rows + r;
      *reinterpret_cast<float2*>(a.part_o + at * a.s.d + e) = make_float2(x * inv, y * inv);
      if (e == 0) a.part_l[at] = sum == 0.f ? -INFINITY : base + log2f(sum);
    } else {
      const int pos = r / a.group, head = h * a.group + r % a.group;
      *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + ((static_cast<long long>(b) * a.s.sq + pos) * a.s.hq + head) * a.s.d + e) =
          pack2<T>(x * inv, y * inv);
      if (e == 0 && a.lse != nullptr) a.lse[lse_at(a, b, h, r)] = sum == 0.f ? -INFINITY : -(base + log2f(sum));
    }
  }
  if (a.splits == 1) pad_lse(a, b, h);
}

// joins the ranges of one (sample, key head): a thread per pair of output elements
template <typename T> __global__ void __launch_bounds__(kFewThreads) attn_few_join_kernel(const FewArgs a) {
  const int h = blockIdx.x, b = blockIdx.y;
  griddep_launch_dependents();
  griddep_wait();
  const long long n = static_cast<long long>(a.s.batch) * a.s.hkv * a.rows;
  for (int i = threadIdx.x; i < a.rows * a.s.d / 2; i += kFewThreads) {
    const int r = i / (a.s.d / 2), e = (i - r * (a.s.d / 2)) * 2;
    const long long at = (static_cast<long long>(b) * a.s.hkv + h) * a.rows + r;
    float top = -INFINITY;
    for (int s = 0; s < a.splits; ++s) top = max3(top, a.part_l[s * n + at], a.part_l[s * n + at]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x = 0.f, y = 0.f;
    for (int s = 0; s < a.splits; ++s) {  // a range without keys weighs 2^-inf and holds zeros
      const float wgt = ex2_approx(a.part_l[s * n + at] - base);
      const float2 o = *reinterpret_cast<const float2*>(a.part_o + (s * n + at) * a.s.d + e);
      sum += wgt;
      x = fmaf(o.x, wgt, x);
      y = fmaf(o.y, wgt, y);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int pos = r / a.group, head = h * a.group + r % a.group;
    *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + ((static_cast<long long>(b) * a.s.sq + pos) * a.s.hq + head) * a.s.d + e) =
        pack2<T>(x * inv, y * inv);
    if (e == 0 && a.lse != nullptr) a.lse[lse_at(a, b, h, r)] = sum == 0.f ? -INFINITY : -(base + log2f(sum));
  }
  pad_lse(a, b, h);
}

// ------------------------------------------------------------------ host side
// Up to two rows always (one row: 72 us against 91 us of the tile kernel at 2 x 8 heads x 50021 keys of 128, 30 against 59
// at 32 x 20 x 750 x 64; two rows: 76 / 90 and 27 / 59). With three or four the arithmetic counts: short keys only (32 x 16
// x 77 x 72, four rows: 12.7 us against 19.1, 64 x 4 x 300 x 64: 11.9 / 18.7; but 64 x 16 x 300 x 128, three queries: 67 / 60,
// 2 x 8 x 50021 x 128, four rows: 139 / 94) - unless the heads that share a key head do not pack into one tile (three of
// them): there the tile kernel reads the keys once per head (2 x 8 x 50021 x 128: 139 / 248, 32 x 8 x 3000 x 64: 53 / 136).
bool attn_few_takes(const AttnShape& s) {
  const int group = s.hq / s.hkv;
  if (s.sq > kFewRows || group > kFewRows || s.sq * group > kFewRows) return false;
  return s.sq * group <= 2 || s.gp < group || static_cast<long long>(s.sk) * s.d <= 32768;
}

static int few_splits(const AttnShape& s, bool varies) {
  // CTAs run in rounds of what the GPU holds at once. Less than half a round: as many ranges as fill one (2 x 8 key heads x
  // 50021 keys: 1.3 times as long with 1.1 rounds as with one), none below 64 keys. More: the fewest ranges of 512 keys and more that
  // fill four fifths of their rounds, else the best filled; shorter ranges do not pay for the second kernel (64 x 4 x 300
  // keys: 16 us in three ranges, 12 in one). Where lengths differ the longest sample's CTA would be the last one running:
  // a round and a quarter of ranges, none below 256 keys (32 x 20 x up to 1500 keys: a third longer in one range than in two).
  const int rows = s.sq * (s.hq / s.hkv), ctas = rows == 1 ? kFewCtas<1> : rows == 2 ? kFewCtas<2> : kFewCtas<4>;
  const long long pairs = static_cast<long long>(s.batch) * s.hkv, room = static_cast<long long>(ctas) * sm_count();
  const long long most = s.sk / 64 > 1 ? s.sk / 64 : 1;
  if (pairs * 2 <= room) return static_cast<int>(room / pairs < most ? room / pairs : most);
  if (varies) {
    const long long n = (room * 5 / 4 + pairs - 1) / pairs, top = s.sk / 256 > 1 ? s.sk / 256 : 1;
    return static_cast<int>(n < top ? n : top);
  }
  int best = 1;
  double best_fill = 0;
  for (int n = 1; n <= 8 && (n == 1 || s.sk / n >= 512); ++n) {
    const double fill = static_cast<double>(pairs * n) / static_cast<double>((pairs * n + room - 1) / room * room);
    if (fill > best_fill - 1e-9) {
      best = n;
      best_fill = fill;
    }
    if (fill >= 0.8) break;
  }
  return best;
}

size_t attn_few_ws(const AttnShape& s) {
  const int one = few_splits(s, false), other = few_splits(s, true), splits = one > other ? one : other;
  if (splits == 1) return 0;
  return static_cast<size_t>(splits) * s.batch * s.hkv * s.sq * (s.hq / s.hkv) * (s.d + 1) * sizeof(float);
}

template <typename T, int R> static const void* pick_few(int d) {
  if (d <= 8) return (const void*)attn_few_kernel<T, 1, R>;
  if (d <= 16) return (const void*)attn_few_kernel<T, 2, R>;
  if (d <= 32) return (const void*)attn_few_kernel<T, 4, R>;
  if (d <= 64) return (const void*)attn_few_kernel<T, 8, R>;
  return (const void*)attn_few_kernel<T, 16, R>;
}
template <typename T> static const void* pick_few_rows(int rows, int d) {
  return rows == 1 ? pick_few<T, 1>(d) : rows == 2 ? pick_few<T, 2>(d) : pick_few<T, 4>(d);
}

int attn_few(int dtype, const void* q, const void* k, const void* v, void* out, float* lse, const AttnMask& mask,
             const AttnShape& s, const int64_t* strides, float c, void* ws, cudaStream_t st) {
  FewArgs a{};
  a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse; a.s = s; a.mask = mask; a.c = c;
  for (int i = 0; i < 9; ++i) a.st[i] = strides[i];
  a.group = s.hq / s.hkv;
  a.rows = s.sq * a.group;
  a.splits = few_splits(s, mask.key_mask != nullptr || mask.kv_lens != nullptr);
  a.part_o = static_cast<float*>(ws);
  a.part_l = a.part_o + static_cast<size_t>(a.splits) * s.batch * s.hkv * a.rows * s.d;
  void* params[] = {&a};
  const bool bf = dtype == ND_BF16;
  const int e = attn_launch(bf ? pick_few_rows<__nv_bfloat16>(a.rows, s.d) : pick_few_rows<__half>(a.rows, s.d),
                            dim3(a.splits, s.hkv, s.batch), kFewThreads, 0, params, st);
  if (e != ND_OK || a.splits == 1) return e;
  return attn_launch(bf ? (const void*)attn_few_join_kernel<__nv_bfloat16> : (const void*)attn_few_join_kernel<__half>,
                     dim3(s.hkv, s.batch), kFewThreads, 0, params, st);
}

}  // namespace nd
