// Rotary positions (sm_100a): every pair (a, b) of a head's first 2 R dimensions becomes
//   (f (a cos t - b sin t), f (a sin t + b cos t)),   t = position[axis of the pair] * freq[pair]
// on a [B, S, heads, D] tensor, or on q and k while a fused projection [B, S, 3 heads D] is split into q, k, v (and on
// the way back). The gradient is the same rotation by -t, so forward and backward share the kernel.
//
// The angle. t in radians as a 32-bit float is off by t * 2^-24, 0.06 radians at position 10^6. Here a frequency
// becomes a 64-bit fixed-point fraction of a turn, and position * fraction is ONE 64-bit integer product whose overflow
// drops the whole turns: the remainder is exact, whatever the position. Its top 32 bits go to sincospi.
//
// Bound: HBM, one read and one write of every element (plus one position per token and axis). A CTA takes two or
// four tokens and fills a table of (cos, sin) for them in shared memory once; all heads of q and k read it, so a sine costs
// the kernel 1 / heads of what it would cost per element. 3 x 10007 x 12 x 64 fp32: 32 us, 5.8 TB/s, 0.88 of the copy rate;
// pack of [32, 256, 3 x 16 x 72] bf16: 24.6 us, 4.6 TB/s; one token of eight sequences: 5.6 us, the launch. A thread owns one vector slot of the token (a pair of vectors R
// apart in the half layout, one vector of adjacent pairs in the interleaved one, a plain copy elsewhere), of q and of k
// alike, and one 16-byte slot of v. The loads of its first slots, of all the CTA's tokens, are issued before the table is
// worked out and are in flight meanwhile: with the table first a CTA waits for memory four times in a row.
#include "common.cuh"

namespace nd {

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = 1024;  // table of at most 4 tokens * pairs * 8 bytes = 32 KB
// Tokens per CTA: two where a thread has q, k and v of each (8 x 4096 x 3 x 16 x 72 bf16: 83 us, with four 90, whose registers
// leave three CTAs on an SM), four of one tensor (30021 x 12 x 64 fp32: 31 us, with two 35)
template <int ROT> constexpr int rot_tokens = ROT == 2 ? 2 : 4;

struct RotSeg {  // one tensor of [tokens, heads, D]; strides in elements
  const void* src;
  void* dst;
  long long src_b, src_s, src_h;
  long long dst_b, dst_s, dst_h;
};

struct RotArgs {
  RotSeg seg[3];          // the rotated ones (one or two), then the copied one
  const void* positions;  // [B or 1, S, axes] of pos_bytes-byte integers, contiguous within a sample
  const double* freqs;    // [axes, pairs / axes] radians per position
  long long tokens, seq_len, pos_b;  // pos_b: elements between samples (0: shared)
  int heads, head_dim, pairs, axes, pos_bytes;
  int rot_units, units;   // vector slots per head of a rotated segment: rotated ones, all
  int copy_units;         // 16-byte (or narrower) slots per head of the copied segment
  unsigned units_mul, copy_mul;  // slot / units as a high product (0: units == 1)
  float factor;
  int inverse;
};

template <typename T, int V, bool ALIGNED> __device__ __forceinline__ void rot_load(Vec<T, V>& v, const T* p) {
  if constexpr (ALIGNED) {
    v.load_stream(p);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v.v[i] = p[i];
  }
}
template <typename T, int V, bool ALIGNED> __device__ __forceinline__ void rot_store(const Vec<T, V>& v, T* p) {
  if constexpr (ALIGNED) {
    v.store(p);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = v.v[i];
  }
}

// the two products of a rotation, contracted the same way in every variant: the vector width never changes a result
__device__ __forceinline__ float rot_re(float re, float im, float2 cs) { return fmaf(re, cs.x, -__fmul_rn(im, cs.y)); }
__device__ __forceinline__ float rot_im(float re, float im, float2 cs) { return fmaf(re, cs.y, __fmul_rn(im, cs.x)); }

// n / d for n < 2^16 and d < 2^16 with mul = ceil(2^32 / d): exact, since n * (mul * d - 2^32) < 2^32
__device__ __forceinline__ int rot_div(int n, unsigned mul) {
  return mul == 0 ? n : static_cast<int>(__umulhi(static_cast<unsigned>(n), mul));
}

// ROT rotated segments (x, or q and k), COPY: a copied one behind them (v), in vectors of CV elements
template <typename T, int V, int CV, bool ALIGNED, bool INTERLEAVED, int ROT, bool COPY>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotArgs a) {
  constexpr int kRotTokens = rot_tokens<ROT>;
  extern __shared__ float2 table[];  // [kRotTokens][pairs]
  constexpr int kParts = INTERLEAVED ? 1 : 2;  // vectors per rotated slot
  const long long t0 = static_cast<long long>(blockIdx.x) * kRotTokens;
  const int nt = a.tokens - t0 < kRotTokens ? static_cast<int>(a.tokens - t0) : kRotTokens;
  // sample and position of the CTA's tokens: one division (a 64-bit one is a hundred instructions), then steps
  const long long b0 = a.tokens <= 0x7FFFFFFFLL ? static_cast<long long>(static_cast<unsigned>(t0) / static_cast<unsigned>(a.seq_len))
                                                : t0 / a.seq_len;
  const long long s0 = t0 - b0 * a.seq_len;
  auto place = [&](int j, long long& b, long long& s) {
    b = b0;
    s = s0 + j;
    while (s >= a.seq_len) {
      s -= a.seq_len;
      ++b;
    }
  };
  long long tok_b[kRotTokens], tok_s[kRotTokens];
#pragma unroll
  for (int j = 0; j < kRotTokens; ++j) place(j, tok_b[j], tok_s[j]);
  Vec<T, V> x[ROT][kRotTokens][kParts];
  auto load = [&](int i) {
    const int head = rot_div(i, a.units_mul), u = i - head * a.units;
    const bool rotated = u < a.rot_units;
    const int e0 = rotated ? u * V : 2 * a.pairs + (u - a.rot_units) * V;
#pragma unroll
    for (int g = 0; g < ROT; ++g) {
      const T* src = static_cast<const T*>(a.seg[g].src) + head * a.seg[g].src_h + e0;
#pragma unroll
      for (int j = 0; j < kRotTokens; ++j)
        if (j < nt) {
          const T* at = src + tok_b[j] * a.seg[g].src_b + tok_s[j] * a.seg[g].src_s;
          rot_load<T, V, ALIGNED>(x[g][j][0], at);
          if (kParts == 2 && rotated) rot_load<T, V, ALIGNED>(x[g][j][kParts - 1], at + a.pairs);
        }
    }
  };
  auto finish = [&](int i) {
    const int head = rot_div(i, a.units_mul), u = i - head * a.units;
    const bool rotated = u < a.rot_units;
    const int e0 = rotated ? u * V : 2 * a.pairs + (u - a.rot_units) * V;
#pragma unroll
    for (int g = 0; g < ROT; ++g) {
      T* dst = static_cast<T*>(a.seg[g].dst) + head * a.seg[g].dst_h + e0;
#pragma unroll
      for (int j = 0; j < kRotTokens; ++j) {
        if (j >= nt) break;
        T* at = dst + tok_b[j] * a.seg[g].dst_b + tok_s[j] * a.seg[g].dst_s;
        if (rotated) {
          const float2* tab = table + j * a.pairs;
          float f[kParts][V];
          x[g][j][0].unpack(f[0]);
          if constexpr (INTERLEAVED) {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
              const float2 cs = tab[(u * V + e) / 2];
              const float re = f[0][e], im = f[0][e + 1];
              f[0][e] = rot_re(re, im, cs);
              f[0][e + 1] = rot_im(re, im, cs);
            }
          } else {
            x[g][j][kParts - 1].unpack(f[kParts - 1]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float2 cs = tab[u * V + e];
              const float re = f[0][e], im = f[kParts - 1][e];
              f[0][e] = rot_re(re, im, cs);
              f[kParts - 1][e] = rot_im(re, im, cs);
            }
            x[g][j][kParts - 1].pack(f[kParts - 1]);
            rot_store<T, V, ALIGNED>(x[g][j][kParts - 1], at + a.pairs);
          }
          x[g][j][0].pack(f[0]);
        }
        rot_store<T, V, ALIGNED>(x[g][j][0], at);
      }
    }
  };
  Vec<T, CV> y[COPY ? kRotTokens : 1];
  auto copy = [&](int i, bool store) {
    const int head = rot_div(i, a.copy_mul), e0 = (i - head * a.copy_units) * CV;
    const RotSeg& sg = a.seg[ROT];
#pragma unroll
    for (int j = 0; j < kRotTokens; ++j) {
      if (j >= nt) break;
      if (!store) rot_load<T, CV, ALIGNED>(y[COPY ? j : 0], static_cast<const T*>(sg.src) + tok_b[j] * sg.src_b + tok_s[j] * sg.src_s + head * sg.src_h + e0);
      else rot_store<T, CV, ALIGNED>(y[COPY ? j : 0], static_cast<T*>(sg.dst) + tok_b[j] * sg.dst_b + tok_s[j] * sg.dst_s + head * sg.dst_h + e0);
    }
  };

  const int n_rot = a.heads * a.units, n_copy = COPY ? a.heads * a.copy_units : 0;
  int i = threadIdx.x, c = threadIdx.x;
  if (i < n_rot) load(i);
  if constexpr (COPY) {
    if (c < n_copy) copy(c, false);
  }

  const int per_axis = a.pairs / a.axes;
  for (int k = threadIdx.x; k < nt * a.pairs; k += blockDim.x) {
    const int j = k / a.pairs, p = k - j * a.pairs;
    long long b, s;
    place(j, b, s);
    const long long at = b * a.pos_b + s * a.axes + p / per_axis;
    const long long pos = a.pos_bytes == 8 ? __ldg(static_cast<const long long*>(a.positions) + at)
                                           : static_cast<long long>(__ldg(static_cast<const int*>(a.positions) + at));
    const double f = __ldg(a.freqs + p) * 0.15915494309189533576888376337251;  // turns per position
    const unsigned long long frac = __double2ull_rz((f - floor(f)) * 18446744073709551616.0);
    const unsigned long long turn = static_cast<unsigned long long>(pos) * frac;  // whole turns overflow away
    float sn, cs;
    sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * 4.656612873077392578125e-10f, &sn, &cs);  // 2^-31
    if (!isfinite(f)) sn = cs = __int_as_float(0x7fffffff);
    table[k] = make_float2(cs * a.factor, (a.inverse ? -sn : sn) * a.factor);
  }
  __syncthreads();

  while (i < n_rot) {
    finish(i);
    i += blockDim.x;
    if (i < n_rot) load(i);
  }
  if constexpr (COPY) {
    while (c < n_copy) {
      copy(c, true);
      c += blockDim.x;
      if (c < n_copy) copy(c, false);
    }
  }
}

static unsigned rot_mul(int d) { return d <= 1 ? 0u : static_cast<unsigned>((0x100000000ull + d - 1) / d); }

template <typename T, int V, int CV, bool ALIGNED>
static int rot_launch_v(RotArgs& a, bool interleaved, bool pack, cudaStream_t st) {
  const int rest = a.head_dim - 2 * a.pairs;
  a.rot_units = interleaved ? 2 * a.pairs / V : a.pairs / V;
  a.units = a.rot_units + rest / V;
  a.copy_units = a.head_dim / CV;
  a.units_mul = rot_mul(a.units);
  a.copy_mul = rot_mul(a.copy_units);
  const long long all = static_cast<long long>(a.heads) * (a.units > a.copy_units ? a.units : a.copy_units);
  if (all >= 65536) return ND_ERR_UNSUPPORTED;  // rot_div's range
  const int per_cta = pack ? rot_tokens<2> : rot_tokens<1>;
  const long long grid = (a.tokens + per_cta - 1) / per_cta;
  if (grid > 0x7FFFFFFFLL) return ND_ERR_UNSUPPORTED;
  const int slots = a.heads * a.units;
  const int passes = (slots + kRotThreads - 1) / kRotThreads;
  const int nt = ((slots + passes - 1) / passes + 31) / 32 * 32;
  const void* fn;
  if constexpr (V == 1) {  // an interleaved pair needs two elements
    fn = pack ? (const void*)rotary_kernel<T, V, CV, ALIGNED, false, 2, true> : (const void*)rotary_kernel<T, V, CV, ALIGNED, false, 1, false>;
  } else {
    fn = interleaved ? (pack ? (const void*)rotary_kernel<T, V, CV, ALIGNED, true, 2, true> : (const void*)rotary_kernel<T, V, CV, ALIGNED, true, 1, false>)
                     : (pack ? (const void*)rotary_kernel<T, V, CV, ALIGNED, false, 2, true> : (const void*)rotary_kernel<T, V, CV, ALIGNED, false, 1, false>);
  }
  void* params[] = {&a};
  const size_t smem = sizeof(float2) * per_cta * static_cast<size_t>(a.pairs);
  cudaError_t e = cudaLaunchKernel(fn, dim3(static_cast<unsigned>(grid)), dim3(nt), params, smem, st);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    (void)cudaGetLastError();
    return ND_ERR_LAUNCH;
  }
  return ND_OK;
}

template <typename T> static int rot_launch(RotArgs& a, bool interleaved, bool pack, cudaStream_t st) {
  // the widest vector that divides every offset a slot can have and every base address: 16 bytes where R (half layout)
  // or 2 R (interleaved) allow it; half of 72 dimensions is 36, which makes it 8 bytes for 16-bit types (v keeps 16)
  unsigned long long mix = static_cast<unsigned long long>(a.head_dim), addr = 0;
  for (int g = 0; g < (pack ? 3 : 1); ++g) {
    const RotSeg& s = a.seg[g];
    mix |= static_cast<unsigned long long>(s.src_h) | static_cast<unsigned long long>(s.src_s) |
           static_cast<unsigned long long>(s.src_b) | static_cast<unsigned long long>(s.dst_h) |
           static_cast<unsigned long long>(s.dst_s) | static_cast<unsigned long long>(s.dst_b);
    addr |= reinterpret_cast<uintptr_t>(s.src) | reinterpret_cast<uintptr_t>(s.dst);
  }
  const unsigned long long rot = mix | (2ull * a.pairs) | (interleaved ? 0ull : static_cast<unsigned long long>(a.pairs));
  auto fits = [&](unsigned long long what, unsigned v) { return what % v == 0 && addr % (v * sizeof(T)) == 0; };
  constexpr int kWide = 16 / sizeof(T);
  if (fits(rot, kWide)) return rot_launch_v<T, kWide, kWide, true>(a, interleaved, pack, st);
  if constexpr (sizeof(T) == 2) {
    if (fits(rot, 4)) return fits(mix, 8) ? rot_launch_v<T, 4, 8, true>(a, interleaved, pack, st) : rot_launch_v<T, 4, 4, true>(a, interleaved, pack, st);
  }
  if (fits(rot, 2)) return rot_launch_v<T, 2, 2, true>(a, interleaved, pack, st);
  // odd head dimensions, odd strides or odd addresses: single elements (adjacent pairs as two of them, where the rest
  // of the head is even too)
  if (!interleaved) return rot_launch_v<T, 1, 1, true>(a, false, pack, st);
  if (a.head_dim % 2 == 0) return rot_launch_v<T, 2, 2, false>(a, true, pack, st);
  return ND_ERR_UNSUPPORTED;
}

static int rot_entry(int dtype, RotArgs& a, int64_t batch, int64_t seq_len, int64_t heads, int64_t head_dim,
                     const void* positions, int pos_bytes, int64_t pos_stride_b, const double* freqs, int64_t pairs,
                     int64_t axes, int interleaved, float factor, int inverse, bool pack, void* stream) {
  a.positions = positions; a.freqs = freqs;
  a.tokens = batch * seq_len; a.seq_len = seq_len; a.pos_b = pos_stride_b;
  a.heads = static_cast<int>(heads); a.head_dim = static_cast<int>(head_dim);
  a.pairs = static_cast<int>(pairs); a.axes = static_cast<int>(axes); a.pos_bytes = pos_bytes;
  a.factor = factor; a.inverse = inverse;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case ND_F16: return rot_launch<__half>(a, interleaved != 0, pack, st);
    case ND_BF16: return rot_launch<__nv_bfloat16>(a, interleaved != 0, pack, st);
    case ND_F32: return rot_launch<float>(a, interleaved != 0, pack, st);
    default: return ND_ERR_UNSUPPORTED;
  }
}

static int rot_check(int dtype, int64_t batch, int64_t seq_len, int64_t heads, int64_t head_dim, int pos_bytes,
                     int64_t pos_stride_b, int64_t pairs, int64_t axes) {
  if (batch < 0 || seq_len < 0 || heads <= 0 || head_dim <= 0 || pairs <= 0 || axes <= 0 || pos_stride_b < 0)
    return ND_ERR_BAD_ARG;
  if (pairs > head_dim / 2 || pairs % axes != 0 || (pos_bytes != 4 && pos_bytes != 8)) return ND_ERR_BAD_ARG;
  if (dtype != ND_F16 && dtype != ND_BF16 && dtype != ND_F32) return ND_ERR_UNSUPPORTED;
  if (pairs > kRotMaxPairs || heads > 65535 || head_dim > 65535) return ND_ERR_UNSUPPORTED;
  if (batch > 0 && seq_len > INT64_MAX / 2 / batch) return ND_ERR_UNSUPPORTED;
  return ND_OK;
}

}  // namespace nd

extern "C" {

int nd_rotary(int dtype, const void* x, void* y, int64_t batch, int64_t seq_len, int64_t heads, int64_t head_dim,
              int64_t stride_b, int64_t stride_s, int64_t stride_h, const void* positions, int pos_bytes,
              int64_t pos_stride_b, const double* freqs, int64_t pairs, int64_t axes, int interleaved, float factor,
              int inverse, void* stream) {
  using namespace nd;
  const int rc = rot_check(dtype, batch, seq_len, heads, head_dim, pos_bytes, pos_stride_b, pairs, axes);
  if (rc != ND_OK) return rc;
  if (stride_b < 0 || stride_s < 0 || stride_h < 0) return ND_ERR_BAD_ARG;
  if (batch == 0 || seq_len == 0) return ND_OK;
  if (!x || !y || !positions || !freqs) return ND_ERR_BAD_ARG;
  RotArgs a{};
  a.seg[0] = RotSeg{x, y, stride_b, stride_s, stride_h, seq_len * heads * head_dim, heads * head_dim, head_dim};
  return rot_entry(dtype, a, batch, seq_len, heads, head_dim, positions, pos_bytes, pos_stride_b, freqs, pairs, axes,
                   interleaved, factor, inverse, false, stream);
}

static int qkv_rotary(bool pack, int dtype, const void* qkv, const void* const* part, int64_t batch, int64_t seq_len,
                      int64_t heads, int64_t head_dim, const void* positions, int pos_bytes, int64_t pos_stride_b,
                      const double* freqs, int64_t pairs, int64_t axes, int interleaved, float factor, void* stream) {
  using namespace nd;
  const int rc = rot_check(dtype, batch, seq_len, heads, head_dim, pos_bytes, pos_stride_b, pairs, axes);
  if (rc != ND_OK) return rc;
  if (batch == 0 || seq_len == 0) return ND_OK;
  if (!qkv || !part[0] || !part[1] || !part[2] || !positions || !freqs) return ND_ERR_BAD_ARG;
  const int64_t hidden = heads * head_dim;
  const size_t es = dtype == ND_F32 ? 4 : 2;
  RotArgs a{};
  for (int g = 0; g < 3; ++g) {
    void* wide = const_cast<char*>(static_cast<const char*>(qkv)) + g * hidden * es;
    void* narrow = const_cast<void*>(part[g]);
    a.seg[g] = pack ? RotSeg{wide, narrow, seq_len * 3 * hidden, 3 * hidden, head_dim, seq_len * hidden, hidden, head_dim}
                    : RotSeg{narrow, wide, seq_len * hidden, hidden, head_dim, seq_len * 3 * hidden, 3 * hidden, head_dim};
  }
  return rot_entry(dtype, a, batch, seq_len, heads, head_dim, positions, pos_bytes, pos_stride_b, freqs, pairs, axes,
                   interleaved, factor, pack ? 0 : 1, true, stream);
}

int nd_qkv_pack_rotary_fwd(int dtype, const void* qkv, void* q, void* k, void* v, int64_t batch, int64_t seq_len,
                           int64_t heads, int64_t head_dim, const void* positions, int pos_bytes, int64_t pos_stride_b,
                           const double* freqs, int64_t pairs, int64_t axes, int interleaved, float factor, void* stream) {
  const void* part[3] = {q, k, v};
  return qkv_rotary(true, dtype, qkv, part, batch, seq_len, heads, head_dim, positions, pos_bytes, pos_stride_b, freqs,
                    pairs, axes, interleaved, factor, stream);
}

int nd_qkv_pack_rotary_bwd(int dtype, const void* dq, const void* dk, const void* dv, void* dqkv, int64_t batch,
                           int64_t seq_len, int64_t heads, int64_t head_dim, const void* positions, int pos_bytes,
                           int64_t pos_stride_b, const double* freqs, int64_t pairs, int64_t axes, int interleaved,
                           float factor, void* stream) {
  const void* part[3] = {dq, dk, dv};
  return qkv_rotary(false, dtype, dqkv, part, batch, seq_len, heads, head_dim, positions, pos_bytes, pos_stride_b, freqs,
                    pairs, axes, interleaved, factor, stream);
}

}  // extern "C"
