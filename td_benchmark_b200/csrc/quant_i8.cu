// 8-bit integer codes with one scale for each row (the token scales of the integer products).
//
//   scale = max(amax / 127, 1e-12)      IEEE fp32 division
//   q     = rne(x / scale) within +-127  IEEE fp32 division for each element
//
// A group of 32 to 1024 threads owns a row and keeps it in registers as loaded (up to four
// 16-byte vectors in each thread) between the maximum and the codes, so x is read once.
// Bound by HBM: size + 1 bytes for each element.  Rows that bulk copies can read go through a
// ring of three stages in shared memory, which keeps three rows of every block in flight; rows
// of other alignments are loaded by their threads, and rows wider than the group's registers
// are read a second time, from L2.
#include <cuda_fp16.h>
#include <math.h>

#include <atomic>

#include "b2m_common.cuh"
#include "b2m_host.h"

namespace b2m {
namespace {

constexpr int kVecs = 4;     // 16-byte vectors of a row in one thread's registers
constexpr int kBlock = 256;  // threads of a block that holds several rows

// Larger of the two; NaN when one of them is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// What a 32-bit word of the row holds: two 16-bit values or one of 32 bits.  `larger` keeps the
// larger magnitudes (its signs mean nothing), `top` is the larger magnitude of a word.
template <typename T>
struct Word;
template <>
struct Word<float> {
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t w) {
    return __float_as_uint(max_nan(__uint_as_float(a), fabsf(__uint_as_float(w))));
  }
  static __device__ __forceinline__ float top(uint32_t a) { return __uint_as_float(a); }
  static __device__ __forceinline__ void unpack(uint32_t w, float* f) { f[0] = __uint_as_float(w); }
};
template <>
struct Word<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t w) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(w));
    return r;
  }
  static __device__ __forceinline__ float top(uint32_t a) {
    return max_nan(fabsf(__uint_as_float(a << 16)), fabsf(__uint_as_float(a & 0xFFFF0000u)));
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float* f) {
    f[0] = __uint_as_float(w << 16);
    f[1] = __uint_as_float(w & 0xFFFF0000u);
  }
};
template <>
struct Word<__half> {
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t w) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(w));
    return r;
  }
  static __device__ __forceinline__ float top(uint32_t a) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&a));
    return max_nan(fabsf(v.x), fabsf(v.y));
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float* f) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
    f[0] = v.x;
    f[1] = v.y;
  }
};

// Vector `i` of a row (16 bytes), zero beyond the row.
template <typename T, bool kAligned>
__device__ __forceinline__ uint4 load_vec(const T* __restrict__ row, int64_t cols, int64_t i) {
  constexpr int N = 16 / sizeof(T);
  const int64_t c = i * N;
  if (kAligned && c + N <= cols) return __ldg(reinterpret_cast<const uint4*>(row + c));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (c + j >= cols) continue;
    if (sizeof(T) == 4)
      w[j & 3] = reinterpret_cast<const uint32_t*>(row)[c + j];
    else
      w[j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[c + j]) << (16 * (j & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ uint32_t larger_vec(uint32_t a, const uint4& v) {
  return Word<T>::larger(Word<T>::larger(Word<T>::larger(Word<T>::larger(a, v.x), v.y), v.z), v.w);
}

// Codes of one vector.  x * (1 / scale) is within 1.6e-5 of x / scale (two roundings of a
// value of at most 127) and the IEEE quotient within 4e-6, so both round to the same integer
// unless the product lies within 2e-5 of a tie; values that come within kNearTie of one are
// decided by the remainder.  (Of 16-bit values one in a thousand does, since x / scale is 127
// times a ratio of short integers; dividing those took 1.5 us more at 8192 x 7168.)  Adding
// 1.5 * 2^23 rounds to the nearest even integer and leaves it in the low byte.  A division for each element
// would cost more than the memory traffic (8192 x 7168 bf16: 81 us with them; 27 us is what HBM
// needs).
constexpr float kNearTie = 4e-5f;
constexpr float kRound = 12582912.0f;

// Two values at once: r = x * inv + kRound, and d = x * inv + (kRound - r), what rounding left.
__device__ __forceinline__ void round_two(float x0, float x1, float inv, float& r0, float& r1, float& d0, float& d1) {
  asm("{\n\t.reg .b64 x, i, k, n, r, d;\n\t"
      "mov.b64 x, {%4, %5};\n\t"
      "mov.b64 i, {%6, %6};\n\t"
      "mov.b64 k, {%7, %7};\n\t"
      "mov.b64 n, {%8, %8};\n\t"
      "fma.rn.f32x2 r, x, i, k;\n\t"
      "fma.rn.f32x2 d, r, n, k;\n\t"
      "fma.rn.f32x2 d, x, i, d;\n\t"
      "mov.b64 {%0, %1}, r;\n\t"
      "mov.b64 {%2, %3}, d;\n\t}"
      : "=f"(r0), "=f"(r1), "=f"(d0), "=f"(d1)
      : "f"(x0), "f"(x1), "f"(inv), "f"(kRound), "f"(-1.0f));
}

// The code (plus kRound) of an x whose product with 1 / scale lies `d` from the integer m, close
// to the tie t = m +- 1/2.  e = x - t scale is exact: t has eight bits, so both terms are multiples
// of 2^-25 of scale's power of two P, and they differ by less than 2^12 of those (kNearTie and the
// product's error make 6e-5 of scale, which is below 2 P).  The IEEE quotient is t itself when
// x / scale is within half a step of it.  (Only at t = 1/2, a power of two, is the step below it
// shorter; both answers are 0 there.)
__device__ __forceinline__ float code_near_tie(float x, float scale, float m, float d) {
  const float t = m + copysignf(0.5f, d);
  const float e = __fmaf_rn(-t, scale, x);
  const float half_step = __uint_as_float(__float_as_uint(t) & 0x7f800000u) * 5.9604644775390625e-8f;  // 2^-24
  if (fabsf(e) <= scale * half_step) return t + kRound;  // the even one
  return (e > 0.0f ? t + 0.5f : t - 0.5f) + kRound;
}

template <int N>
__device__ __forceinline__ void codes_of(const float (&f)[N], float scale, float inv, bool divide,
                                         uint32_t (&w)[N / 4]) {
  float r[N], off = 0.0f;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    float d0, d1;
    round_two(f[j], f[j + 1], inv, r[j], r[j + 1], d0, d1);
    off = fmaxf(off, fmaxf(fabsf(d0), fabsf(d1)));
  }
  if (divide) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      r[j] = __int_as_float(max(-127, min(127, __float2int_rn(f[j] / scale))));  // a NaN quotient converts to 0
  } else if (off > 0.5f - kNearTie) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = __fmaf_rn(f[j], inv, kRound - r[j]);
      if (fabsf(d) > 0.5f - kNearTie) r[j] = code_near_tie(f[j], scale, r[j] - kRound, d);
    }
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    w[i] = __byte_perm(__byte_perm(__float_as_uint(r[4 * i]), __float_as_uint(r[4 * i + 1]), 0x0040),
                       __byte_perm(__float_as_uint(r[4 * i + 2]), __float_as_uint(r[4 * i + 3]), 0x0040), 0x5410);
}

template <typename T, bool kAligned>
__device__ __forceinline__ void store_codes(int8_t* __restrict__ q, int64_t cols, int64_t i, float scale, float inv,
                                            bool divide, const uint4& v) {
  constexpr int N = 16 / sizeof(T);
  constexpr int kIn = 4 / sizeof(T);  // values in a word
  const int64_t c = i * N;
  float f[N];
  Word<T>::unpack(v.x, f);
  Word<T>::unpack(v.y, f + kIn);
  Word<T>::unpack(v.z, f + 2 * kIn);
  Word<T>::unpack(v.w, f + 3 * kIn);
  uint32_t w[N / 4];
  codes_of<N>(f, scale, inv, divide, w);
  if (kAligned && c + N <= cols) {
    if (N == 8)
      *reinterpret_cast<uint2*>(q + c) = make_uint2(w[0], w[N / 4 - 1]);
    else
      *reinterpret_cast<uint32_t*>(q + c) = w[0];
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (c + j < cols) q[c + j] = static_cast<int8_t>(w[j / 4] >> (8 * (j & 3)));
  }
}

// Largest value of the group's partial maxima, in every thread of it.  `part`: one value for
// each warp of the block, of two sets used in turn.  False in all threads when `ok` is in one.
__device__ __forceinline__ bool group_max(float& amax, float* part, int group, bool ok) {
  // bits of values that are not negative order as the values do, with NaN above infinity
  const int lane = threadIdx.x & 31;
  uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
  if (lane == 0) part[threadIdx.x >> 5] = __uint_as_float(most);
  ok = __syncthreads_and(ok);
  if (group > 32)
    most = __reduce_max_sync(
        0xffffffffu, __float_as_uint(part[((threadIdx.x & ~(group - 1)) >> 5) + (lane & (group / 32 - 1))]));
  amax = __uint_as_float(most);
  return ok;
}

constexpr int kRing = 3;

// blockDim = rows of a stage x group; group = 32 .. 1024 threads of a row.  Rows are `row_bytes`
// (a multiple of 16) in stages of `stage_bytes`, 16-byte aligned in x.
template <typename T>
__global__ void __launch_bounds__(1024)
    quant_i8_ring_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t ldx, int8_t* __restrict__ q,
                         int64_t ldq, float* __restrict__ scale, int group, int stage_bytes, int32_t* status,
                         uint64_t timeout_ns) {
  constexpr int N = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ uint64_t full[kRing];
  __shared__ float part[2][32];
  __shared__ int abort;
  const int in_row = threadIdx.x & (group - 1);
  const int at = threadIdx.x / group, per = blockDim.x / group;  // row of the stage
  const int row_bytes = static_cast<int>(cols * sizeof(T)), vecs = row_bytes / 16;
  const int64_t step = static_cast<int64_t>(gridDim.x) * per;
  auto fetch = [&](int64_t first, int s) {  // rows first .. first + per - 1
    const int n = static_cast<int>(rows - first < per ? rows - first : per);
    mbar_arrive_expect_tx(&full[s], static_cast<uint32_t>(n * row_bytes));
    for (int i = 0; i < n; ++i)
      bulk_load(ring + s * stage_bytes + i * row_bytes, x + (first + i) * ldx, static_cast<uint32_t>(row_bytes), &full[s]);
  };
  int64_t first = static_cast<int64_t>(blockIdx.x) * per;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kRing; ++s) mbar_init(&full[s], 1);
    abort = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    for (int s = 0; s < kRing; ++s)
      if (first + s * step < rows) fetch(first + s * step, s);
  }
  __syncthreads();
  int s = 0, phase = 0;
  for (int round = 0; first < rows; first += step, round ^= 1) {
    bool ok = mbar_wait(&full[s], phase, timeout_ns, status, B2M_STATUS_TIMEOUT_PRODUCER, &abort);
    const int64_t r = first + at;
    const uint4* row = reinterpret_cast<const uint4*>(ring + s * stage_bytes + at * row_bytes);
    uint4 v[kVecs];
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < kVecs; ++u)
      if (r < rows && in_row + u * group < vecs) v[u] = row[in_row + u * group];
#pragma unroll
    for (int u = 0; u < kVecs; ++u)
      if (r < rows && in_row + u * group < vecs) most = larger_vec<T>(most, v[u]);
    float amax = Word<T>::top(most);
    ok = group_max(amax, part[round], group, ok);  // and everyone has read the stage
    if (!ok) break;
    if (threadIdx.x == 0 && first + kRing * step < rows) {
      fence_proxy_async_smem();
      fetch(first + kRing * step, s);
    }
    if (r < rows) {
      const float sc = max_nan(amax / 127.0f, 1e-12f);
      if (in_row == 0) scale[r] = sc;
      const float inv = 1.0f / sc;
      const bool divide = !(sc < INFINITY);  // the row holds a NaN or an infinity
#pragma unroll
      for (int u = 0; u < kVecs; ++u)
        if (in_row + u * group < vecs)
          store_codes<T, true>(q + r * ldq, cols, in_row + u * group, sc, inv, divide, v[u]);
    }
    if (++s == kRing) s = 0, phase ^= 1;
  }
  // after a timeout: the copies in flight may still land; wait for them, within the limit
  if (first < rows && threadIdx.x == 0) {
    for (int i = 0; i < kRing && first < rows; ++i, first += step) {
      mbar_wait(&full[s], phase, timeout_ns, status, B2M_STATUS_TIMEOUT_DRAIN, nullptr);
      if (++s == kRing) s = 0, phase ^= 1;
    }
  }
}

// The same for any alignment and width; each thread loads what it works on.
template <typename T, bool kAligned, bool kInRegisters>
__global__ void __launch_bounds__(1024)
    quant_i8_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t ldx, int8_t* __restrict__ q,
                    int64_t ldq, float* __restrict__ scale, int group) {
  constexpr int N = 16 / sizeof(T);
  __shared__ float part[32];
  const int in_row = threadIdx.x & (group - 1);
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (blockDim.x / group) + threadIdx.x / group;
  const int64_t vecs = r < rows ? (cols + N - 1) / N : 0;
  const T* row = x + r * ldx;
  uint4 v[kInRegisters ? kVecs : 1];
  uint32_t most = 0;
  if (kInRegisters) {
#pragma unroll
    for (int u = 0; u < kVecs; ++u)
      if (in_row + u * group < vecs) v[u] = load_vec<T, kAligned>(row, cols, in_row + u * group);
#pragma unroll
    for (int u = 0; u < kVecs; ++u)
      if (in_row + u * group < vecs) most = larger_vec<T>(most, v[u]);
  } else {
    for (int64_t i = in_row; i < vecs; i += group) most = larger_vec<T>(most, load_vec<T, kAligned>(row, cols, i));
  }
  float amax = Word<T>::top(most);
  group_max(amax, part, group, true);
  if (r >= rows) return;
  const float sc = max_nan(amax / 127.0f, 1e-12f);
  if (in_row == 0) scale[r] = sc;
  const float inv = 1.0f / sc;
  const bool divide = !(sc < INFINITY);  // the row holds a NaN or an infinity
  int8_t* qr = q + r * ldq;
  if (kInRegisters) {
#pragma unroll
    for (int u = 0; u < kVecs; ++u)
      if (in_row + u * group < vecs)
        store_codes<T, kAligned>(qr, cols, in_row + u * group, sc, inv, divide, v[u]);
  } else {
    for (int64_t i = in_row; i < vecs; i += group)
      store_codes<T, kAligned>(qr, cols, i, sc, inv, divide, load_vec<T, kAligned>(row, cols, i));
  }
}

template <typename T>
int launch_quant(const void* x, int64_t rows, int64_t cols, int64_t ldx, void* q, int64_t ldq, float* scale,
                 int32_t* status, int num_sms, cudaStream_t s) {
  constexpr int N = 16 / sizeof(T);
  const int64_t vecs = (cols + N - 1) / N;
  // Threads of a row: as few as hold it, and more while there are too few rows to fill the
  // GPU (one row of 7168: 1024 threads of one vector each, not 256 of four).
  int group = 32;
  while (group < 1024 && group < vecs && (int64_t(group) * kVecs < vecs || rows * group < int64_t(num_sms) * 1024))
    group *= 2;
  const bool fits = int64_t(group) * kVecs >= vecs;
  const bool aligned = aligned16(x) && ldx * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(q) % N == 0 && ldq % N == 0;
  const int block = group > kBlock ? group : kBlock;
  const int64_t per_block = block / group;
  const int64_t blocks = (rows + per_block - 1) / per_block;
  if (blocks > INT32_MAX) return fail(B2M_ERR_ARG, "quant_i8: too many rows (%lld)", (long long)rows);
  // Blocks that are resident together: 1024 threads an SM (64 registers each), and their rings.
  const int64_t stage = per_block * cols * sizeof(T);
  int64_t per_sm = 1024 / block;
  if (per_sm * (kRing * stage + 2048) > 225 * 1024) per_sm = 225 * 1024 / (kRing * stage + 2048);
  // The ring pays from the second row of a block on; with one row each, its set-up only adds to
  // the row's time.
  if (aligned && fits && cols % N == 0 && per_sm > 0 && blocks > per_sm * num_sms) {
    static std::atomic<bool> attr_done[64];
    int dev = 0;
    B2M_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
    if (dev >= 64 || !attr_done[dev].load(std::memory_order_acquire)) {
      B2M_TRY(check_cuda(cudaFuncSetAttribute(quant_i8_ring_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                              224 * 1024),
                         "quant_i8: cudaFuncSetAttribute"));
      if (dev < 64) attr_done[dev].store(true, std::memory_order_release);
    }
    quant_i8_ring_kernel<T><<<static_cast<int>(per_sm * num_sms), block, kRing * stage, s>>>(
        static_cast<const T*>(x), rows, cols, ldx, static_cast<int8_t*>(q), ldq, scale, group, static_cast<int>(stage),
        status, 2 * timeout_ns());
    return check_cuda(cudaGetLastError(), "quant_i8 launch");
  }
  auto kernel = aligned ? (fits ? quant_i8_kernel<T, true, true> : quant_i8_kernel<T, true, false>)
                        : (fits ? quant_i8_kernel<T, false, true> : quant_i8_kernel<T, false, false>);
  kernel<<<static_cast<int>(blocks), block, 0, s>>>(static_cast<const T*>(x), rows, cols, ldx, static_cast<int8_t*>(q),
                                                    ldq, scale, group);
  return check_cuda(cudaGetLastError(), "quant_i8 launch");
}

}  // namespace
}  // namespace b2m

extern "C" int b2m_quant_i8(const void* x, int32_t in_type, int64_t rows, int64_t cols, int64_t ldx, void* q,
                            int64_t ldq, float* scale, int32_t* dev_status, void* stream) {
  using namespace b2m;
  if (rows < 0 || cols < 1 || cols > (int64_t(1) << 30) || ldx < cols || ldq < cols ||
      ldx > (int64_t(1) << 38) || ldq > (int64_t(1) << 38))
    return fail(B2M_ERR_ARG, "quant_i8: bad shape [%lld, %lld], row strides %lld and %lld", (long long)rows,
                (long long)cols, (long long)ldx, (long long)ldq);
  if (in_type != B2M_BF16 && in_type != B2M_FP16 && in_type != B2M_FP32)
    return fail(B2M_ERR_ARG, "quant_i8: unknown input type %d", in_type);
  if (rows > 0 && (!x || !q || !scale)) return fail(B2M_ERR_ARG, "quant_i8: null pointer");
  if (reinterpret_cast<uintptr_t>(x) % (in_type == B2M_FP32 ? 4 : 2))
    return fail(B2M_ERR_ARG, "quant_i8: misaligned input");
  if (!aligned4(scale) || !aligned4(dev_status))
    return fail(B2M_ERR_ARG, "quant_i8: scale and status must be 4-byte aligned");
  int num_sms = 0;
  B2M_TRY(require_sm100(&num_sms));
  if (rows == 0) return B2M_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (in_type == B2M_BF16)
    return launch_quant<__nv_bfloat16>(x, rows, cols, ldx, q, ldq, scale, dev_status, num_sms, s);
  if (in_type == B2M_FP16) return launch_quant<__half>(x, rows, cols, ldx, q, ldq, scale, dev_status, num_sms, s);
  return launch_quant<float>(x, rows, cols, ldx, q, ldq, scale, dev_status, num_sms, s);
}
