// Global 2-norm of a list of gradient tensors, and clipping by it:
//   norm = sqrt(sum over all tensors and elements of g^2),   g <- g * min(1, max_norm / (norm + 1e-6)).
//
// Bound by memory: one read for the norm, one read and one write where the factor is below 1 (nothing is written
// otherwise). Two launches whatever the number of tensors (up to 1,500 per launch): the tensors' addresses
// and sizes travel as kernel arguments, so nothing is copied to the device and a captured graph keeps its own
// table. The data are cut into equal chunks across all tensors and the chunks dealt round-robin to a fixed
// grid, so a block's share does not depend on how the sizes are spread, and the sum is made in the same order every
// time: no atomics. The second launch walks the chunks backwards: what the first one read last is still in the
// L2 cache (126 MB), so gradients that fit are read from memory once. Runs of neighbouring chunks per block instead of the
// dealing were 7 % slower.
// Measured: 537 M fp32 values in 64 tensors 336 us for the norm (6.4 TB/s) and 1,094 us with the scaling (two reads and a
// write, 5.9 TB/s); 50 M bf16 values in 301 tensors, which fit the L2 cache, 28 and 60 us; six tensors of 0.8 MB 4 us.
// Sums: squares of one 16-byte vector in 32 bits, everything above in 64 bits; a vector whose squares
// leave the safe range of 32 bits is squared again in 64 (see vector_square).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <vector>

#include "common.cuh"

namespace evox {
namespace {

constexpr int kThreads = 256;
constexpr int kBlocksPerSm = 8;  // 2,048 resident threads

template <int N>
struct Table {
  unsigned long long address[N];
  unsigned long long extent[N];  // bytes * 4 + type
  int begin[N + 1];              // first chunk of every tensor; begin[count] is the number of chunks
  int count;
  int chunk_bytes;
};

struct Chunk {
  unsigned long long low, high;    // bytes of the tensor that belong to this chunk
  unsigned long long first, last;  // 16-byte vectors that cover them
  int type;
};

// Chunks are cut at 16-byte addresses: only the first and the last vector of a tensor can be partial.
template <int N>
__device__ __forceinline__ Chunk chunk_of(const Table<N>& t, int c) {
  int lo = 0, hi = t.count;  // begin[lo] <= c < begin[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.begin[mid] <= c) lo = mid; else hi = mid;
  }
  Chunk k;
  const unsigned long long start = t.address[lo], end = start + (t.extent[lo] >> 2), base = start & ~15ull;
  k.type = (int)(t.extent[lo] & 3);
  k.first = base + (unsigned long long)(c - t.begin[lo]) * t.chunk_bytes;
  k.last = min(k.first + t.chunk_bytes, (end + 15) & ~15ull);
  k.low = start;
  k.high = end;
  return k;
}

// x[0..n) of a 16-byte vector as 32-bit values.
__device__ __forceinline__ int unpack(const uint4& v, int type, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if (type == EVOX_DTYPE_FP32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(w[j]);
    return 4;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (type == EVOX_DTYPE_BF16) {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
  }
  return 8;
}

// Sum of squares of a vector. In 32 bits it is right to 8 roundings unless it overflows, or is so small that squares
// were lost to underflow (below 1e-25 those lost, each under 1e-38, could count): then 64 bits.
__device__ __forceinline__ double vector_square(const uint4& v, int type) {
  float x[8];
  float s = 0.f;
  if (unpack(v, type, x) == 4) {
    s = fmaf(x[0], x[0], fmaf(x[1], x[1], fmaf(x[2], x[2], x[3] * x[3])));
    if (s > 1.0e-25f && s < 1.0e37f) return (double)s;
    return (double)x[0] * x[0] + (double)x[1] * x[1] + (double)x[2] * x[2] + (double)x[3] * x[3];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) s = fmaf(x[j], x[j], s);
  if (s > 1.0e-25f && s < 1.0e37f) return (double)s;
  double d = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) d += (double)x[j] * x[j];
  return d;
}

__device__ __forceinline__ float load_one(unsigned long long at, int type) {
  if (type == EVOX_DTYPE_FP32) return *reinterpret_cast<const float*>(at);
  const unsigned short u = *reinterpret_cast<const unsigned short*>(at);
  return type == EVOX_DTYPE_BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}

__device__ __forceinline__ void store_one(unsigned long long at, int type, float x) {
  if (type == EVOX_DTYPE_FP32) *reinterpret_cast<float*>(at) = x;
  else if (type == EVOX_DTYPE_BF16) *reinterpret_cast<__nv_bfloat16*>(at) = __float2bfloat16_rn(x);
  else *reinterpret_cast<__half*>(at) = __float2half_rn(x);
}

__device__ __forceinline__ uint4 scaled(const uint4& v, int type, float f) {
  float x[8];
  unpack(v, type, x);
  uint4 r;
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (type == EVOX_DTYPE_FP32) {
      w[j] = __float_as_uint(x[j] * f);
    } else if (type == EVOX_DTYPE_BF16) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * j] * f, x[2 * j + 1] * f);
      w[j] = *reinterpret_cast<const uint32_t*>(&p);
    } else {
      const __half2 p = __floats2half2_rn(x[2 * j] * f, x[2 * j + 1] * f);
      w[j] = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
  return r;
}

__device__ __forceinline__ double warp_sum_double(double x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// Sum over the block, in every thread.
__device__ __forceinline__ double block_sum_double(double x) {
  __shared__ double part[kThreads / 32];
  x = warp_sum_double(x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
  __syncthreads();
  x = part[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) x += part[w];
  return x;
}

template <int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    grad_square_kernel(const __grid_constant__ Table<N> t, double* __restrict__ partial) {
  overlapped_start();
  double sum = 0.0;
  const int chunks = t.begin[t.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const Chunk k = chunk_of(t, c);
    const int size = k.type == EVOX_DTYPE_FP32 ? 4 : 2;
    if (k.first >= k.low && k.last <= k.high) {
#pragma unroll 4
      for (unsigned long long a = k.first + threadIdx.x * 16ull; a < k.last; a += kThreads * 16ull)
        sum += vector_square(__ldg(reinterpret_cast<const uint4*>(a)), k.type);
    } else {
      for (unsigned long long a = k.first + threadIdx.x * 16ull; a < k.last; a += kThreads * 16ull) {
        if (a >= k.low && a + 16 <= k.high) {
          sum += vector_square(__ldg(reinterpret_cast<const uint4*>(a)), k.type);
        } else {
          for (unsigned long long e = max(a, k.low); e < min(a + 16, k.high); e += size) {
            const double x = load_one(e, k.type);
            sum += x * x;
          }
        }
      }
    }
  }
  sum = block_sum_double(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The norm from the first launches' partial sums (every block adds them up in the same order), then the scaling.
template <int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    grad_scale_kernel(const __grid_constant__ Table<N> t, const double* __restrict__ partial, int n_partial, float max_norm,
                      int write_norm, float* __restrict__ norm_out) {
  overlapped_start();
  double sum = 0.0;
  for (int i = threadIdx.x; i < n_partial; i += kThreads) sum += partial[i];
  const float norm = (float)sqrt(block_sum_double(sum));
  if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = norm;
  const float f = max_norm / (norm + 1e-6f);
  if (f >= 1.0f) return;  // a NaN norm goes on: it makes every gradient NaN
  const int chunks = t.begin[t.count];
  for (int i = blockIdx.x; i < chunks; i += gridDim.x) {
    const Chunk k = chunk_of(t, chunks - 1 - i);
    const int size = k.type == EVOX_DTYPE_FP32 ? 4 : 2;
    if (k.first >= k.low && k.last <= k.high) {
#pragma unroll 4
      for (unsigned long long a = k.first + threadIdx.x * 16ull; a < k.last; a += kThreads * 16ull) {
        uint4* p = reinterpret_cast<uint4*>(a);
        __stcs(p, scaled(*p, k.type, f));
      }
    } else {
      for (unsigned long long a = k.first + threadIdx.x * 16ull; a < k.last; a += kThreads * 16ull) {
        if (a >= k.low && a + 16 <= k.high) {
          uint4* p = reinterpret_cast<uint4*>(a);
          *p = scaled(*p, k.type, f);
        } else {
          for (unsigned long long e = max(a, k.low); e < min(a + 16, k.high); e += size) store_one(e, k.type, load_one(e, k.type) * f);
        }
      }
    }
  }
}

// Tensors per launch, 20 bytes each: 2, 8 or 30 KB of arguments (32,764 bytes are the limit). A launch pays for copying what it carries: both
// launches for 301 tensors take the host 18 us with 30 KB each, 11 with 8.
constexpr int kSmall = 96, kMiddle = 400, kLarge = 1500;

struct Batch {
  int first, count, grid;
};

int type_size(int type) { return type == EVOX_DTYPE_FP32 ? 4 : 2; }

template <int N>
void fill(Table<N>& t, const Batch& b, const uint64_t* address, const int64_t* numel, const int32_t* dtype, int chunk_bytes) {
  t.count = b.count;
  t.chunk_bytes = chunk_bytes;
  int chunks = 0;
  for (int i = 0; i < b.count; ++i) {
    const uint64_t bytes = (uint64_t)numel[b.first + i] * type_size(dtype[b.first + i]), at = address[b.first + i];
    t.address[i] = at;
    t.extent[i] = bytes << 2 | (uint32_t)dtype[b.first + i];
    t.begin[i] = chunks;
    if (bytes) chunks += (int)((((at + bytes + 15) & ~15ull) - (at & ~15ull) + chunk_bytes - 1) / chunk_bytes);
  }
  t.begin[b.count] = chunks;
}

template <int N>
int launch_square(const Batch& b, const uint64_t* address, const int64_t* numel, const int32_t* dtype, int chunk_bytes, double* partial,
                  cudaStream_t stream) {
  Table<N> t;
  fill(t, b, address, numel, dtype, chunk_bytes);
  EVOX_CUDA(launch_overlapped(grad_square_kernel<N>, dim3((unsigned)b.grid), kThreads, 0, 1, stream, t, partial));
  return EVOX_OK;
}

template <int N>
int launch_scale(const Batch& b, const uint64_t* address, const int64_t* numel, const int32_t* dtype, int chunk_bytes, const double* partial,
                 int n_partial, float max_norm, int write_norm, float* norm, cudaStream_t stream) {
  Table<N> t;
  fill(t, b, address, numel, dtype, chunk_bytes);
  EVOX_CUDA(launch_overlapped(grad_scale_kernel<N>, dim3((unsigned)b.grid), kThreads, 0, 1, stream, t, partial, n_partial, max_norm, write_norm, norm));
  return EVOX_OK;
}

// Whether two of the tensors share memory. False if the host's memory does not suffice to tell (no exception may
// leave a C entry point).
bool overlap(const uint64_t* address, const int64_t* numel, const int32_t* dtype, int n, bool* shared) {
  bool ascending = true;  // pieces of one flat buffer usually come in order
  uint64_t end = 0;
  for (int i = 0; i < n && ascending; ++i) {
    if (numel[i] == 0) continue;
    ascending = address[i] >= end;
    end = address[i] + (uint64_t)numel[i] * type_size(dtype[i]);
  }
  *shared = false;
  if (ascending) return true;
  try {
    std::vector<std::pair<uint64_t, uint64_t>> span;
    span.reserve((size_t)n);
    for (int i = 0; i < n; ++i)
      if (numel[i]) span.emplace_back(address[i], address[i] + (uint64_t)numel[i] * type_size(dtype[i]));
    std::sort(span.begin(), span.end());
    for (size_t i = 1; i < span.size(); ++i) *shared |= span[i].first < span[i - 1].second;
  } catch (...) {
    return false;
  }
  return true;
}

int grid_limit() { return sm_count() * kBlocksPerSm; }

}  // namespace
}  // namespace evox

using namespace evox;

extern "C" size_t evox_grad_norm_workspace_bytes(int32_t n_tensors) {
  if (n_tensors < 0) return 0;
  return sizeof(double) * (size_t)(n_tensors / kLarge + 1) * (size_t)grid_limit();
}

extern "C" int evox_clip_grad_norm(const uint64_t* address, const int64_t* numel, const int32_t* dtype, int32_t n_tensors, float max_norm,
                                   int32_t clip, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  EVOX_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || (address && numel && dtype)), EVOX_ERR_INVALID, "clip_grad_norm: NULL table");
  EVOX_REQUIRE(norm && workspace, EVOX_ERR_INVALID, "clip_grad_norm: NULL pointer");
  EVOX_REQUIRE(((uintptr_t)workspace & 7u) == 0, EVOX_ERR_INVALID, "clip_grad_norm: workspace must be 8-byte aligned");
  EVOX_REQUIRE(workspace_bytes >= evox_grad_norm_workspace_bytes(n_tensors), EVOX_ERR_WORKSPACE, "clip_grad_norm: workspace too small");
  EVOX_REQUIRE(!clip || max_norm >= 0.f, EVOX_ERR_INVALID, "clip_grad_norm: max_norm must not be negative or NaN");
  uint64_t total = 0;
  for (int i = 0; i < n_tensors; ++i) {
    EVOX_REQUIRE(dtype[i] == EVOX_DTYPE_BF16 || dtype[i] == EVOX_DTYPE_FP16 || dtype[i] == EVOX_DTYPE_FP32, EVOX_ERR_INVALID,
                 "clip_grad_norm: tensor %d must be bf16, fp16 or fp32", i);
    EVOX_REQUIRE(numel[i] >= 0 && numel[i] < (1ll << 40), EVOX_ERR_INVALID, "clip_grad_norm: tensor %d has %lld elements", i, (long long)numel[i]);
    EVOX_REQUIRE(numel[i] == 0 || (address[i] != 0 && address[i] % type_size(dtype[i]) == 0), EVOX_ERR_INVALID,
                 "clip_grad_norm: tensor %d has a bad address", i);
    total += (uint64_t)numel[i] * type_size(dtype[i]);
  }
  if (clip) {  // two chunks of one address would be scaled twice, and race
    bool shared = false;
    EVOX_REQUIRE(overlap(address, numel, dtype, n_tensors, &shared), EVOX_ERR_INVALID, "clip_grad_norm: out of host memory");
    EVOX_REQUIRE(!shared, EVOX_ERR_INVALID, "clip_grad_norm: two tensors share memory");
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // chunks: at least two for each resident block where the gradients allow it, between 4 and 32 KB
  const int limit = grid_limit();
  int chunk_bytes = 4096;
  while (chunk_bytes < 32768 && total / (2 * chunk_bytes) >= 2ull * limit) chunk_bytes *= 2;
  // a tensor's chunk numbers are 32-bit: larger chunks where the gradients pass that
  while (total / chunk_bytes > (1ull << 30)) chunk_bytes *= 2;
  double* partial = reinterpret_cast<double*>(workspace);
  int n_partial = 0;
  auto batch_at = [&](int first) {
    Batch b;
    b.first = first;
    b.count = n_tensors - first < kLarge ? n_tensors - first : kLarge;
    long long chunks = 0;
    for (int i = first; i < first + b.count; ++i) chunks += (long long)((uint64_t)numel[i] * type_size(dtype[i]) / chunk_bytes) + 2;
    b.grid = (int)(chunks < limit ? (chunks > 0 ? chunks : 1) : limit);
    return b;
  };
  int first = 0;
  do {  // once at least: the norm of nothing is 0
    const Batch b = batch_at(first);
    if (int rc = b.count <= kSmall    ? launch_square<kSmall>(b, address, numel, dtype, chunk_bytes, partial + n_partial, s)
                 : b.count <= kMiddle ? launch_square<kMiddle>(b, address, numel, dtype, chunk_bytes, partial + n_partial, s)
                                      : launch_square<kLarge>(b, address, numel, dtype, chunk_bytes, partial + n_partial, s))
      return rc;
    n_partial += b.grid;
    first += b.count;
  } while (first < n_tensors);
  if (!clip) {
    const Batch none = {0, 0, 1};
    return launch_scale<kSmall>(none, address, numel, dtype, chunk_bytes, partial, n_partial, INFINITY, 1, norm, s);
  }
  first = 0;
  do {
    const Batch b = batch_at(first);
    const int write_norm = first == 0;
    if (int rc = b.count <= kSmall    ? launch_scale<kSmall>(b, address, numel, dtype, chunk_bytes, partial, n_partial, max_norm, write_norm, norm, s)
                 : b.count <= kMiddle ? launch_scale<kMiddle>(b, address, numel, dtype, chunk_bytes, partial, n_partial, max_norm, write_norm, norm, s)
                                      : launch_scale<kLarge>(b, address, numel, dtype, chunk_bytes, partial, n_partial, max_norm, write_norm, norm, s))
      return rc;
    first += b.count;
  } while (first < n_tensors);
  return EVOX_OK;
}
