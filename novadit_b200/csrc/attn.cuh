// What the attention kernels share: problem description, tensor maps of [B, S, heads, D] views, tcgen05 operand
// descriptors and MMA forms, and how a sample's keys are masked.
//
// Rows. The queries of one key head's group are packed: a "row" is (s, g), g = 0..gp-1 the head inside a block of gp
// query heads that share a key head (gp = the largest power of two, at most 32, that divides the group), row index
// s * gp + g. A tile is 128 rows: one TMA box of gp heads x 128 / gp positions, so a decoding step with shared heads
// fills a tile with all heads that read the same keys. Row statistics (log-sum-exp, delta) live in that order, each
// head block padded to whole tiles.
#pragma once

#include "tc.cuh"

namespace nd {

constexpr int kTile = 128;                // rows of a query tile; keys of a key tile in the backward pass
constexpr int kBlkBytes = kTile * 128;    // 64 16-bit columns of a tile, 128-byte swizzle: 16 KB

struct AttnShape {
  int batch, sq, sk, hq, hkv, d;
  int gp, hb, rows, rows_pad, qtiles, ktiles;  // rows = sq * gp; hb = hq / gp head blocks
  int dn;                                      // d rounded up to 16: columns of an accumulator
};

struct AttnMask {
  const unsigned char* key_mask;  // [batch, sk], nullable
  const int* kv_lens;             // [batch], nullable
};

inline AttnShape attn_shape(int64_t b, int64_t sq, int64_t sk, int64_t hq, int64_t hkv, int64_t d) {
  AttnShape s{};
  s.batch = static_cast<int>(b); s.sq = static_cast<int>(sq); s.sk = static_cast<int>(sk);
  s.hq = static_cast<int>(hq); s.hkv = static_cast<int>(hkv); s.d = static_cast<int>(d);
  const int group = s.hq / s.hkv;
  s.gp = 1;
  while (s.gp < 32 && group % (2 * s.gp) == 0) s.gp *= 2;
  s.hb = s.hq / s.gp;
  s.rows = s.sq * s.gp;
  s.qtiles = (s.rows + kTile - 1) / kTile;
  s.rows_pad = s.qtiles * kTile;
  s.ktiles = (s.sk + kTile - 1) / kTile;
  s.dn = (s.d + 15) / 16 * 16;
  return s;
}

int attn_launch(const void* fn, dim3 grid, int threads, size_t smem, void** params, cudaStream_t st);
// few query rows per key head (attn_few.cu)
bool attn_few_takes(const AttnShape& s);
size_t attn_few_ws(const AttnShape& s);
int attn_few(int dtype, const void* q, const void* k, const void* v, void* out, float* lse, const AttnMask& mask,
             const AttnShape& s, const int64_t* strides, float c, void* ws, cudaStream_t st);

inline int attn_check(int dtype, int64_t b, int64_t sq, int64_t sk, int64_t hq, int64_t hkv, int64_t d, float scale) {
  if (b < 0 || sq < 0 || sk < 0 || hq <= 0 || hkv <= 0 || d <= 0 || hq % hkv != 0) return ND_ERR_BAD_ARG;
  if (!(scale > 0.f) || scale > 3.0e38f) return ND_ERR_BAD_ARG;
  if (dtype != ND_F16 && dtype != ND_BF16) return ND_ERR_UNSUPPORTED;
  if (d % 8 != 0 || d > 128) return ND_ERR_UNSUPPORTED;
  if (b > 65535 || hq > 65535 || sq > (1 << 25) || sk > (1 << 30)) return ND_ERR_UNSUPPORTED;
  return ND_OK;
}

// Element strides of a [B, S, H, ..] view: multiples of 16 bytes, and not zero where there is more than one element (a
// tensor map walks no broadcast dimension)
inline bool attn_strides_ok(const int64_t* st, int64_t b, int64_t s, int64_t h) {
  const int64_t n[3] = {b, s, h};
  for (int i = 0; i < 3; ++i)
    if (st[i] < 0 || st[i] % 8 != 0 || (n[i] > 1 && st[i] == 0)) return false;
  return true;
}

// [B, S, H, D] view with element strides -> boxes of `cols` columns x `heads` heads x `pos` positions
static bool attn_map(CUtensorMap* map, int dtype, const void* base, int64_t b, int64_t s, int64_t h, int64_t d, int64_t sb,
                     int64_t ss, int64_t sh, int cols, int heads, int pos) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(h), static_cast<cuuint64_t>(s),
                              static_cast<cuuint64_t>(b)};
  // the stride of a dimension of one element is never used: any legal value
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(h > 1 ? sh * 2 : 16), static_cast<cuuint64_t>(s > 1 ? ss * 2 : 16),
                                 static_cast<cuuint64_t>(b > 1 ? sb * 2 : 16)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(cols), static_cast<cuuint32_t>(heads), static_cast<cuuint32_t>(pos), 1u};
  const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  return fn(map, dtype == ND_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ------------------------------------------------------------------ device side
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// a tile of NB 64-column blocks of ROWS rows
template <int NB, int ROWS = kTile>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int pos, int b) {
#pragma unroll
  for (int i = 0; i < NB; ++i) tma_load_4d(dst + i * ROWS * 128, map, bar, i * 64, head, pos, b);
}

// One lane of a converged warp. The MMA warp issues under a branch on this: the compiler then knows that a single thread
// runs it, and together with descriptors that are one addition away an MMA costs it some 10 cycles. Under a branch on the
// thread index the same loop takes 55 cycles per MMA, with descriptors put together per MMA 110 to 150 - whatever N is,
// where the tensor pipe needs 64 for N = 128 and 40 for N = 80 (148 CTAs of one issuing thread, K = 16, M = 128; with
// both operands in shared memory 32 + N / 4).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Operand descriptors of a tile [128 rows][64-column blocks], addresses in 16-byte units in the low word. K-major (the
// columns are the reduction): 32 bytes further per K = 16 step, the next block after four steps. MN-major (the rows are
// the reduction): 2048 bytes further per step, blocks ROWS * 128 bytes apart (the leading offset).
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) { return umma_desc(addr); }
template <int ROWS = kTile> __device__ __forceinline__ constexpr uint32_t step_k(int step) {
  return (step >> 2) * (ROWS * 128 >> 4) + (step & 3) * 2;
}
template <int ROWS = kTile> __device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
  return (static_cast<uint64_t>((addr & 0x3FFFFu) >> 4)) | (static_cast<uint64_t>(ROWS * 128 >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
__device__ __forceinline__ constexpr uint32_t step_mn(int step) { return step * 128; }
// M = 128, fp32 accumulator, both operands of one 16-bit type; b_mn: the B operand is MN-major
__device__ __forceinline__ uint32_t attn_idesc(uint32_t fmt, int n, bool b_mn) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn ? (1u << 16) : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
// A from tensor memory: lane = row, two 16-bit values of the reduction per column
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// A run of MMAs from shared memory without a branch between them. With one (a test of the step count before each) an MMA
// takes 75 cycles at N = 64 and 107 at N = 128 instead of 48 and 64: the issue of the next then waits for the one before. So
// the step count is a constant of the whole issue loop for the usual head sizes (forward + backward at 2 x 16 x 4096^2 x 64:
// 884 us against 822; as a switch in front of every run it costs more than it gives, 1003 us).
template <int STEPS, int ROWS> __device__ __forceinline__ void run_nt(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  mma_ss(d, a, b, idesc, 0u);
#pragma unroll
  for (int k = 1; k < STEPS; ++k) mma_ss(d, a + step_k(k), b + step_k<ROWS>(k), idesc, 1u);
}
// D = A B^T over STEPS K = 16 steps of two K-major tiles, B of ROWS rows; STEPS 0: `steps` of them
template <int STEPS, int ROWS = kTile>
__device__ __forceinline__ void issue_nt(uint32_t d, uint64_t a, uint64_t b, int steps, uint32_t idesc) {
  if constexpr (STEPS > 0) {
    run_nt<STEPS, ROWS>(d, a, b, idesc);
  } else {
    mma_ss(d, a, b, idesc, 0u);
    for (int k = 1; k < steps; ++k) mma_ss(d, a + step_k(k), b + step_k<ROWS>(k), idesc, 1u);
  }
}
// calls f with the step count as a constant where it is one of the usual ones (heads of 64, 72 / 80 and 128)
template <typename F> __device__ __forceinline__ void with_steps(int steps, F&& f) {
  if (steps == 4) f(std::integral_constant<int, 4>{});
  else if (steps == 5) f(std::integral_constant<int, 5>{});
  else if (steps == 8) f(std::integral_constant<int, 8>{});
  else f(std::integral_constant<int, 0>{});
}
// D (+)= A B over `steps` groups of 16 rows of B: A from tensor memory, 8 columns per step, every GROUP steps `stride` columns
// behind the ones before
template <int MAX, int GROUP>
__device__ __forceinline__ void issue_tn(uint32_t d, uint32_t a, uint32_t stride, uint64_t b, int steps, uint32_t idesc,
                                         uint32_t accumulate) {
  mma_ts(d, a, b, idesc, accumulate);
#pragma unroll
  for (int k = 1; k < MAX; ++k)
    if (k < steps) mma_ts(d, a + (k / GROUP) * stride + (k % GROUP) * 8, b + step_mn(k), idesc, 1u);
}

// Keys of sample b that take part lie below the returned index (exactly those, without a key mask). Called by whole
// warps; every warp of a CTA gets the same answer.
__device__ __forceinline__ int key_count(const AttnMask& m, int b, int sk, int lane) {
  if (m.kv_lens != nullptr) {
    const int n = __ldg(m.kv_lens + b);
    return n < 0 ? 0 : (n > sk ? sk : n);
  }
  if (m.key_mask == nullptr) return sk;
  const unsigned char* row = m.key_mask + static_cast<long long>(b) * sk;
  int end = sk;
  while (end > 0) {  // from the back, 1024 keys at a time: trailing padding is skipped, holes are not
    const int base = end > 1024 ? end - 1024 : 0;
    int last = -1;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int at = base + i * 32 + lane;
      if (at < end && __ldg(row + at) != 0) last = at;
    }
    last = __reduce_max_sync(0xffffffffu, last);
    if (last >= 0) return last + 1;
    end = base;
  }
  return 0;
}

__device__ __forceinline__ void fill_lens(int* lens, const AttnMask& m, int batch, int sk, int warp, int warps, int lane) {
  for (int b = warp; b < batch; b += warps) {
    const int n = key_count(m, b, sk, lane);
    if (lane == 0) lens[b] = n;
  }
}

// The key mask of keys at .. at + 31 that lie below n_keys; called by whole warps.
__device__ __forceinline__ uint32_t key_word(const AttnMask& m, int b, int sk, int n_keys, int at, int lane) {
  const bool on = at + lane < n_keys && __ldg(m.key_mask + static_cast<long long>(b) * sk + at + lane) != 0;
  return __ballot_sync(0xffffffffu, on);
}

// Which of the KT keys of tile `kt` take part, 32 per word; called by whole warps. True: some do not.
template <int KT = kTile>
__device__ __forceinline__ bool key_bits(const AttnMask& m, int b, int sk, int n_keys, int kt, int lane, uint32_t (&bits)[4]) {
  bool partial = false;
  const int end = n_keys < (kt + 1) * KT ? n_keys : (kt + 1) * KT;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = kt * KT + i * 32;
    const int left = end - at;
    const uint32_t all = KT - i * 32 >= 32 ? 0xffffffffu : (KT <= i * 32 ? 0u : (1u << (KT & 31)) - 1u);
    bits[i] = left >= 32 ? 0xffffffffu : (left <= 0 ? 0u : (1u << left) - 1u);
    if (m.key_mask != nullptr) bits[i] = key_word(m, b, sk, end, at, lane);
    partial |= bits[i] != all;
  }
  return partial;
}

// 2^y for two values on the multiply-add units instead of the special-function unit: 2^y = 2^n 2^f with n the nearest
// integer (the rounding of y + 1.5 * 2^23 leaves it in the low bits) and a degree-4 minimax polynomial for 2^f on
// [-1/2, 1/2] (relative error 2.7e-6 in 32 bits, fitted by a Remez exchange). y below -126 gives 2^-126, y above
// 127 and NaN give 2^127: a sum with it shows.
__device__ __forceinline__ float2 exp2_poly(uint64_t y2) {
  const float2 y = f2_unpack(y2);
  y2 = f2_pack(fmaxf(fminf(y.x, 127.f), -126.f), fmaxf(fminf(y.y, 127.f), -126.f));
  const uint64_t t2 = f2_add(y2, f2_pack(12582912.f, 12582912.f));
  const uint64_t f2 = f2_fma(f2_add(t2, f2_pack(-12582912.f, -12582912.f)), f2_pack(-1.f, -1.f), y2);
  uint64_t p = f2_fma(f2_pack(0.009570102207362652f, 0.009570102207362652f), f2, f2_pack(0.05591785907745361f, 0.05591785907745361f));
  p = f2_fma(p, f2, f2_pack(0.240247443318367f, 0.240247443318367f));
  p = f2_fma(p, f2, f2_pack(0.6931217908859253f, 0.6931217908859253f));
  p = f2_fma(p, f2, f2_pack(0.9999992847442627f, 0.9999992847442627f));
  const float2 t = f2_unpack(t2), r = f2_unpack(p);
  return make_float2(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(t.y) << 23)));
}

// a wait of a whole warp; most find the phase complete
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, WaitSink sink, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, sink, code));
}

// zero row r of a tile: keys that do not take part may hold infinities or NaN, and 0 * NaN in a product is NaN
template <int NB, int ROWS = kTile> __device__ __forceinline__ void clear_row(uint8_t* tile, int r) {
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(tile + i * ROWS * 128 + r * 128 + c * 16) = make_uint4(0, 0, 0, 0);
}

// One warp's 32 rows x 32 columns of 16-bit values (lane = row) in a 2 KB staging block, 64-byte swizzle, for the copy
// engine. A thread that writes its own row to global memory costs one line per lane and instruction (3900 cycles for the
// two tiles of an item at D = 72); a block that is waited for before the next is staged costs about as much. So a
// warp stages all its blocks, hands them over and looks at them again only when it needs the memory for the next item.
constexpr int kStageBytes = 2048;
template <typename T> __device__ __forceinline__ void stage_block(uint8_t* stage, const float (&v)[32], int lane) {
  const int sw = (lane >> 1) & 3;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4*>(stage + lane * 64 + ((c ^ sw) << 4)) =
        make_uint4(pack2<T>(v[c * 8 + 0], v[c * 8 + 1]), pack2<T>(v[c * 8 + 2], v[c * 8 + 3]),
                   pack2<T>(v[c * 8 + 4], v[c * 8 + 5]), pack2<T>(v[c * 8 + 6], v[c * 8 + 7]));
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}

// Key counts of all samples, worked out once by all warps of a CTA where they fit: every role of every item asks for one,
// and a dependent load from global memory each time is most of a short item's start.
constexpr int kLens = 256;
__device__ __forceinline__ bool lens_cached(const AttnMask& m, int batch, int sk) {
  return batch <= kLens && (m.key_mask == nullptr || static_cast<long long>(batch) * sk <= 65536);
}

// let copies already issued land in shared memory before the CTA may exit (after an expired wait)
__device__ __forceinline__ void settle() {
  const unsigned long long t0 = global_ns();
  while (global_ns() - t0 < 200000ull) __nanosleep(1000);
}

// Registers per thread of the calling warpgroup, given back or taken from what others gave back: over the CTA the sum must
// not exceed what it was launched with.
template <int N> __device__ __forceinline__ void reg_give() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void reg_take() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

template <int COLS> __device__ __forceinline__ void tmem_alloc(uint32_t* base) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base)), "r"(COLS) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLS> __device__ __forceinline__ void tmem_free(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(COLS) : "memory");
}

}  // namespace nd
