// Log probability of a given token per row of logits, entropy of the row, and
// its top alternatives:
//   m = max x, Z = sum e^(x - m), S = sum (x - m) e^(x - m)  (0 where x = -inf)
//   logprob = x[token] - m - log Z
//   entropy = log Z - S / Z
//   top     : largest x first, ties to the lowest index
// The sums are fp32.  One CTA per row.
#include "nie_common.cuh"

namespace nie {

constexpr int kLpThreads = 512;
constexpr int kLpMaxTop = 32;

struct LogprobArgs {
  const void* logits;
  int64_t stride, cols;
  const int64_t* tokens;
  int top;
  float* logprobs;
  float* entropy;
  float* top_logprobs;  // [rows, top]
  int64_t* top_ids;
  int32_t* err;
};

// (av, ai) ranks before (bv, bi): larger value (NaN largest), then smaller index.
__device__ __forceinline__ bool lp_before(float av, int64_t ai, float bv, int64_t bi) {
  const bool an = av != av, bn = bv != bv;
  if (an || bn) return an && (!bn || ai < bi);
  return av > bv || (av == bv && ai < bi);
}

__device__ __forceinline__ float block_sum(float x, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < kLpThreads / 32; ++w) s += red[w];
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(LogprobArgs a) {
  using N = Num<T>;
  __shared__ float red[kLpThreads / 32];
  __shared__ int64_t red_i[kLpThreads / 32];
  const int64_t r = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.logits) + r * a.stride;
  float m = -INFINITY;
  for (int64_t c = threadIdx.x; c < a.cols; c += kLpThreads) m = fmaxf(m, N::to_f(x[c]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int w = 0; w < kLpThreads / 32; ++w) m = fmaxf(m, red[w]);
  float z = 0.f, s = 0.f;
  for (int64_t c = threadIdx.x; c < a.cols; c += kLpThreads) {
    const float d = N::to_f(x[c]) - m;
    const float e = expf(d);
    z += e;
    if (e != 0.f) s = fmaf(d, e, s);
  }
  z = block_sum(z, red);
  s = block_sum(s, red);
  const float log_z = logf(z);
  if (threadIdx.x == 0) {
    const int64_t t = a.tokens[r];
    const bool ok = t >= 0 && t < a.cols;
    if (!ok) raise_flag(a.err, NIE_DEV_ERR_INDEX_RANGE);
    a.logprobs[r] = ok ? N::to_f(x[t]) - m - log_z : __int_as_float(0x7fc00000);
    a.entropy[r] = log_z - s / z;
  }
  float pv = 0.f;
  int64_t pi = -1;  // the alternative found last (-1: none yet)
  for (int k = 0; k < a.top; ++k) {
    float bv = -INFINITY;
    int64_t bi = INT64_MAX;
    for (int64_t c = threadIdx.x; c < a.cols; c += kLpThreads) {
      const float v = N::to_f(x[c]);
      if ((pi < 0 || lp_before(pv, pi, v, c)) && lp_before(v, c, bv, bi)) bv = v, bi = c;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int64_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (lp_before(ov, oi, bv, bi)) bv = ov, bi = oi;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = bv, red_i[threadIdx.x >> 5] = bi;
    __syncthreads();
    for (int w = 0; w < kLpThreads / 32; ++w)
      if (lp_before(red[w], red_i[w], bv, bi)) bv = red[w], bi = red_i[w];
    pv = bv, pi = bi;
    if (threadIdx.x == 0) {
      a.top_logprobs[r * a.top + k] = bv - m - log_z;
      a.top_ids[r * a.top + k] = bi;
    }
  }
}

}  // namespace nie

using namespace nie;

extern "C" int nie_token_logprobs(const void* logits, int64_t rows, int64_t cols, int64_t row_stride, int32_t dtype,
                                  const int64_t* tokens, int32_t top, float* logprobs, float* entropy,
                                  float* top_logprobs, int64_t* top_ids, int32_t* err_flag, void* stream) {
  NIE_REQUIRE(logits && tokens && logprobs && entropy, "null pointer argument");
  NIE_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31), "rows out of range");
  NIE_REQUIRE(cols >= 1 && cols < (int64_t(1) << 31) && row_stride >= cols, "bad shape");
  NIE_REQUIRE(top >= 0 && top <= kLpMaxTop && top <= cols, "top must be in [0, %d] and at most the vocabulary", kLpMaxTop);
  NIE_REQUIRE(top == 0 || (top_logprobs && top_ids), "null pointer argument");
  NIE_REQUIRE(dtype_size(dtype) > 0, "unknown dtype %d", dtype);
  if (rows == 0) return NIE_OK;
  LogprobArgs a{logits, row_stride, cols, tokens, top, logprobs, entropy, top_logprobs, top_ids, err_flag};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case NIE_DTYPE_BF16: logprobs_kernel<__nv_bfloat16><<<(unsigned)rows, kLpThreads, 0, s>>>(a); break;
    case NIE_DTYPE_F32: logprobs_kernel<float><<<(unsigned)rows, kLpThreads, 0, s>>>(a); break;
    default: logprobs_kernel<__half><<<(unsigned)rows, kLpThreads, 0, s>>>(a); break;
  }
  return check_launch("logprobs_kernel");
}
