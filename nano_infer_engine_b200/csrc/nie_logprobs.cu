// Log probability of a given token per row of logits, entropy of the row, and
// its top alternatives:
//   m = max x, Z = sum e^(x - m), S = sum (x - m) e^(x - m)  (0 where x = -inf)
//   logprob = x[token] - m - log Z
//   entropy = log Z - S / Z
//   top     : largest x first, ties to the lowest index
//
// What bounds it: the row is read once, 16 bytes a load; at 12 bf16 values a clock
// and SM the exponentials (16 a clock) are close behind.  So everything comes from
// one pass.
//
// Sums: every thread keeps (reference, Z, S) of its own values in fp32; the
// reference is raised only when 8 are exceeded (e^8 leaves fp32 room enough), and
// the triples are merged in a fixed order.
//
// Top: 32 groups of threads each bring the largest value of the first round; the
// k-th largest of those 32 is a lower bound of the k-th largest of all, so that only
// about a hundred values per row pass it.  They go to a buffer of (value, index)
// keys, from which the bound is raised when it fills; the k largest are ranked by
// counting.  A round that overflows the buffer raises the bound from what the buffer
// holds and offers its values again.
//
// Few rows are split over a cluster of up to 8 CTAs; the first one merges the
// others' sums and keys through distributed shared memory.
#include <cooperative_groups.h>

#include <algorithm>

#include "nie_common.cuh"

namespace cg = cooperative_groups;

namespace nie {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;
constexpr int kLpCap = 1024;      // keys of the buffer
constexpr int kLpPrune = 384;     // keys from which the bound is raised
constexpr int kLpMaxCluster = 8;
constexpr float kLpLowest = -3.402823466e38f;
constexpr float kLpLog2e = 1.4426950408889634f;

struct LogprobArgs {
  const void* logits;
  int64_t stride;
  int cols;
  const int64_t* tokens;
  int top;
  float* logprobs;
  float* entropy;
  float* top_logprobs;  // [rows, top]
  int64_t* top_ids;
  int32_t* err;
};

// Larger is better: value (NaN above all, -0 as 0), then the lower index.
__device__ __forceinline__ uint64_t lp_key(float x, int index) {
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t order = x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return ((uint64_t)order << 32) | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ float lp_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0xffffffffu ? __int_as_float(0x7fc00000) : __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int lp_index(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }

// Sums against a reference: m >= every x - 8 so far.
struct LpSums {
  float m, z, s;
  __device__ __forceinline__ void raise(float to) {
    const float f = exp2f((m - to) * kLpLog2e);  // 0 from the lowest reference
    s = f == 0.f ? 0.f : f * (s + (m - to) * z);
    z *= f;
    m = to;
  }
  __device__ __forceinline__ void add(float x) {
    const float d = x - m;
    const float e = fast_exp2(d * kLpLog2e);
    z += e;
    s = fmaf(fmaxf(d, -200.f), e, s);  // e is 0 long before -200, and -inf * 0 is no number
  }
  __device__ __forceinline__ void merge(const LpSums& o) {
    const float to = fmaxf(m, o.m);
    LpSums b = o;
    if (m != to) raise(to);
    if (b.m != to) b.raise(to);
    z += b.z;
    s += b.s;
  }
};

struct LpShared {
  uint64_t keys[kLpCap];
  uint64_t best[kLpMaxTop];     // the k largest so far, sorted
  float groups[2 * kLpWarps];
  LpSums sums[kLpWarps];
  uint64_t bound;               // keys below it are not among the k largest
  int count;                    // keys offered; those past kLpCap are lost
  // what a cluster's first CTA reads
  LpSums total;
  int found;                    // entries of best
};

// The k largest of keys[0, n) to best, sorted; returns how many there are.  Called by the CTA.
__device__ __forceinline__ int lp_rank(LpShared& sh, int n, int k) {
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const uint64_t key = sh.keys[i];
    int rank = 0;
    for (int j = 0; j < n && rank < k; ++j) rank += sh.keys[j] > key;
    if (rank < k) sh.best[rank] = key;
  }
  __syncthreads();
  return min(n, k);
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 2) logprobs_kernel(const __grid_constant__ LogprobArgs a) {
  using N = Num<T>;
  constexpr int V = 16 / (int)sizeof(T);  // values of a load
  constexpr int U = 4;                    // loads of a round
  __shared__ LpShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int part = (int)cluster.block_rank(), parts = (int)cluster.num_blocks();
  const int64_t r = blockIdx.x / parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.stride;
  const int k = a.top;

  // whole 16-byte vectors [0, nvec) behind `head` values; this CTA has [v0, v1) of them
  const int head = min(a.cols, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
  const int nvec = (a.cols - head) / V;
  const int share = (nvec + parts - 1) / parts;
  const int v0 = min(nvec, part * share), v1 = min(nvec, v0 + share);
  const uint4* vec = reinterpret_cast<const uint4*>(row + head);

  if (tid == 0) {
    sh.bound = 0;
    sh.count = 0;
  }
  __syncthreads();

  LpSums mine{kLpLowest, 0.f, 0.f};
  uint64_t bound = 0;
  float floor_v = -INFINITY;  // the bound's value: smaller ones need no key
  auto offer = [&](float x, int index) {
    if (x == -INFINITY) return;  // never a candidate; filled in at the end where others are missing
    const uint64_t key = lp_key(x, index);
    if (key < bound) return;
    const int at = atomicAdd(&sh.count, 1);
    if (at < kLpCap) sh.keys[at] = key;
  };
  auto values = [&](const uint4& raw, float (&x)[V]) {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = N::to_f(e[i]);
  };

  uint4 next[U];
  auto fetch = [&](int from) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = from + u * kLpThreads + tid;
      if (v < v1) next[u] = __ldcs(vec + v);
    }
  };
  fetch(v0);
  for (int from = v0; from < v1; from += U * kLpThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
    fetch(from + U * kLpThreads);
    float top[U], most = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      top[u] = -INFINITY;
      if (from + u * kLpThreads + tid < v1) {
        float x[V];
        values(raw[u], x);
        float mx = x[0];
        bool nan = x[0] != x[0];
#pragma unroll
        for (int i = 1; i < V; ++i) {
          mx = fmaxf(mx, x[i]);
          nan |= x[i] != x[i];
        }
        if (mx > mine.m + 8.f) mine.raise(mx);
#pragma unroll
        for (int i = 0; i < V; ++i) mine.add(x[i]);
        top[u] = nan ? INFINITY : mx;
        most = fmaxf(most, top[u]);
      }
    }
    if (k == 0) continue;
    if (from == v0) {
      // the first bound: the k-th largest of 32 half warps' largest
      float h = most;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, o));
      if ((lane & 15) == 0) sh.groups[2 * warp + (lane >> 4)] = h;
      __syncthreads();
      const float g = sh.groups[lane];
      int above = 0;
      for (int j = 0; j < 32; ++j) above += sh.groups[j] > g || (sh.groups[j] == g && j < lane);
      const unsigned at = __ballot_sync(0xffffffffu, above == k - 1);
      floor_v = __shfl_sync(0xffffffffu, g, __ffs(at) - 1);
      // the key of the value behind any index
      bound = floor_v == -INFINITY ? 0 : (lp_key(floor_v, 0) >> 32) << 32;
      if (floor_v == INFINITY) bound = 0xff800000ull << 32;  // +inf or NaN
    }
    const int kept = sh.count;  // before this round; every thread is past the barrier behind the last one
    __syncthreads();
    auto offer_round = [&]() {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = from + u * kLpThreads + tid;
        if (v < v1 && top[u] >= floor_v) {
          float x[V];
          values(raw[u], x);
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (!(x[i] < floor_v)) offer(x[i], head + v * V + i);
        }
      }
    };
    offer_round();
    __syncthreads();
    while (sh.count > kLpPrune) {  // the same for all threads
      const int n = min(sh.count, kLpCap);
      const bool lost = sh.count > kLpCap;
      lp_rank(sh, n, k);  // n > k: the k-th best of what is there bounds the k-th best of all
      bound = sh.best[k - 1];
      floor_v = lp_value(bound);
      if (floor_v != floor_v) floor_v = INFINITY;
      __syncthreads();
      if (!lost) {
        if (tid < k) sh.keys[tid] = sh.best[tid];
        if (tid == 0) sh.count = k;
        __syncthreads();
        break;
      }
      // the round's keys go, its values are offered again to the higher bound
      if (tid == 0) sh.count = kept;
      __syncthreads();
      offer_round();
      __syncthreads();
    }
  }
  // values in front of the first vector (first CTA) and behind the last one (last CTA)
  {
    const int tail = a.cols - head - nvec * V;
    int index = -1;
    if (part == 0 && tid < head) index = tid;
    else if (part == parts - 1 && tid >= 32 && tid - 32 < tail) index = head + nvec * V + tid - 32;
    if (index >= 0) {
      const float x = N::to_f(row[index]);
      if (x > mine.m + 8.f) mine.raise(x);
      mine.add(x);
      if (k > 0) offer(x, index);  // at most 14 more than the buffer is pruned to
    }
  }
  // sums of the CTA, its best keys
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpSums other{__shfl_down_sync(0xffffffffu, mine.m, o), __shfl_down_sync(0xffffffffu, mine.z, o),
                 __shfl_down_sync(0xffffffffu, mine.s, o)};
    mine.merge(other);
  }
  if (lane == 0) sh.sums[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    LpSums t = sh.sums[0];
    for (int w = 1; w < kLpWarps; ++w) t.merge(sh.sums[w]);
    sh.total = t;
  }
  const int found = k > 0 ? lp_rank(sh, sh.count, k) : 0;
  if (tid == 0) sh.found = found;
  if (parts > 1) {
    cluster.sync();
    if (part == 0) {
      int n = found;
      if (tid < found) sh.keys[tid] = sh.best[tid];
      for (int p = 1; p < parts; ++p) {
        const LpShared* o = cluster.map_shared_rank(&sh, p);
        const int f = o->found;
        if (tid < f) sh.keys[n + tid] = o->best[tid];
        n += f;
        if (tid == 0) sh.total.merge(o->total);
      }
      __syncthreads();
      if (k > 0) {
        const int f = lp_rank(sh, n, k);
        if (tid == 0) sh.found = f;
      }
    }
    cluster.sync();  // the others stay until their shared memory has been read
    if (part != 0) return;
  }
  __syncthreads();
  const LpSums t = sh.total;
  const float nan = __int_as_float(0x7fc00000);
  // a row of nothing but -inf has no distribution
  const float log_z = t.z == 0.f ? nan : logf(t.z);
  if (tid == 0) {
    const int64_t token = a.tokens[r];
    const bool ok = token >= 0 && token < a.cols;
    if (!ok) raise_flag(a.err, NIE_DEV_ERR_INDEX_RANGE);
    a.logprobs[r] = ok ? N::to_f(row[token]) - t.m - log_z : nan;
    a.entropy[r] = log_z - t.s / t.z;
  }
  if (tid < sh.found) {
    const uint64_t key = sh.best[tid];
    a.top_logprobs[r * k + tid] = lp_value(key) - t.m - log_z;
    a.top_ids[r * k + tid] = lp_index(key);
  }
  if (warp == 0 && sh.found < k) {
    // fewer tokens than asked for have any probability: the first of the others
    int at = sh.found;
    for (int c0 = 0; c0 < a.cols && at < k; c0 += 32) {
      const int c = c0 + lane;
      const bool none = c < a.cols && N::to_f(row[c]) == -INFINITY;
      const unsigned all = __ballot_sync(0xffffffffu, none);
      const int mine_at = at + __popc(all & ((1u << lane) - 1u));
      if (none && mine_at < k) {
        a.top_logprobs[r * k + mine_at] = -INFINITY - t.m - log_z;
        a.top_ids[r * k + mine_at] = c;
      }
      at += __popc(all);
    }
  }
}

template <typename T>
static int launch_logprobs(const LogprobArgs& a, int64_t rows, int parts, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, a);
  if (e != cudaSuccess) return fail(NIE_ERR_CUDA, "logprobs_kernel launch: %s", cudaGetErrorString(e));
  return check_launch("logprobs_kernel");
}

}  // namespace nie

using namespace nie;

extern "C" int nie_token_logprobs(const void* logits, int64_t rows, int64_t cols, int64_t row_stride, int32_t dtype,
                                  const int64_t* tokens, int32_t top, float* logprobs, float* entropy,
                                  float* top_logprobs, int64_t* top_ids, int32_t* err_flag, void* stream) {
  NIE_REQUIRE(rows >= 0 && rows < (int64_t(1) << 28), "rows out of range");
  NIE_REQUIRE(cols >= 1 && cols < (int64_t(1) << 31) - 65536 && row_stride >= cols, "bad shape");
  NIE_REQUIRE(top >= 0 && top <= kLpMaxTop && top <= cols, "top must be in [0, %d] and at most the vocabulary", kLpMaxTop);
  NIE_REQUIRE(dtype_size(dtype) > 0, "unknown dtype %d", dtype);
  if (rows == 0) return NIE_OK;
  NIE_REQUIRE(logits && tokens && logprobs && entropy, "null pointer argument");
  NIE_REQUIRE(top == 0 || (top_logprobs && top_ids), "null pointer argument");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int sms = sm_count(stream_device(s));
  NIE_REQUIRE(sms > 0, "cannot query the SM count");
  // rows that do not fill the SMs (two CTAs each) are split, down to a round's worth of values
  const int64_t round = (int64_t)kLpThreads * 4 * (16 / dtype_size(dtype));
  int parts = 1;
  while (parts < kLpMaxCluster && rows * parts * 2 <= 2 * sms && cols > parts * round) parts *= 2;
  LogprobArgs a{logits, row_stride, (int)cols, tokens, top, logprobs, entropy, top_logprobs, top_ids, err_flag};
  switch (dtype) {
    case NIE_DTYPE_BF16: return launch_logprobs<__nv_bfloat16>(a, rows, parts, s);
    case NIE_DTYPE_F32: return launch_logprobs<float>(a, rows, parts, s);
    default: return launch_logprobs<__half>(a, rows, parts, s);
  }
}
