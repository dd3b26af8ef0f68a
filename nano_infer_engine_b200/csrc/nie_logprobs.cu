// Log probability of a given token per row of logits, entropy of the row, and
// its top alternatives:
//   m = max x, Z = sum e^(x - m), S = sum (x - m) e^(x - m)  (0 where x = -inf)
//   logprob = x[token] - m - log Z
//   entropy = log Z - S / Z
//   top     : largest x first, ties to the lowest index
//
// What bounds it: the row is read once, 16 bytes a load; at 12 bf16 values a clock
// and SM the exponentials (16 a clock) and the instructions around them (5 to a
// value) are close behind.  So everything comes from one pass, in pairs of values.
// Measured: 4096 rows of 128256 bf16 values with 20 alternatives 244 us (4.3 TB/s), without
// any 164 (6.4 TB/s), 333 of 50257 fp32 values with 3 20 us (3.3 TB/s), one row with 5 11.7
// us, without any 6.6.
//
// Sums: every thread keeps (reference, Z, S) of its own values in fp32; the
// reference is raised only when exceeded by 8 (e^8 leaves fp32 room enough), and the
// triples are merged in a fixed order.  Rows that touch the ends of the range, where
// x - m may have no fp32 form, get a pass of their own.
//
// Top: 32 groups of threads each bring the largest value of the first round of loads;
// the k-th largest of those 32 is a lower bound of the k-th largest of all.  What
// passes it goes to a buffer of (value, index) keys, whose k-th best, found by
// counting, is the bound of the next rounds.  It is raised behind rounds 1, 2, 4, 8,
// ..., so that about k values of each doubling pass it and most rounds need no
// barrier.  Loads of nothing but forbidden tokens bring no key: a mask may leave fewer
// values than a bound takes.  Rows that overflow the buffer (values that rise all the way), or
// have fewer than k values above the lowest that the maxima know and some below, are
// gone through again, with the bound raised after every load.
//
// Few rows are split over a cluster of up to 4 CTAs; the first one merges the
// others' sums and keys through distributed shared memory.
#include <cooperative_groups.h>

#include <algorithm>

#include "nie_common.cuh"

namespace cg = cooperative_groups;

namespace nie {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;
constexpr int kLpCap = 1024;      // keys of the buffer (a load of every thread and the k best fit)
constexpr int kLpQueue = 512;     // loads that hold a value above the bound
constexpr int kLpMaxCluster = 4;
// Rows with larger values, or with none above its negative, are taken apart; a reference starts below.
constexpr float kLpRange = 1.3e38f;
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

// d = a + b, a * b, a * b + c on two fp32 lanes in one instruction.
__device__ __forceinline__ float2 lp_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 ra, rb, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %5};\nadd.rn.f32x2 rd, ra, rb;\n"
      "mov.b64 {%0, %1}, rd;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 lp_mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 ra, rb, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %5};\nmul.rn.f32x2 rd, ra, rb;\n"
      "mov.b64 {%0, %1}, rd;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 lp_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 ra, rb, rc, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %5};\nmov.b64 rc, {%6, %7};\n"
      "fma.rn.f32x2 rd, ra, rb, rc;\nmov.b64 {%0, %1}, rd;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// Two neighbouring values of a load: -inf brought to a low finite value, kLowest (its
// exponential is 0 all the same, and 0 times it is 0), NaN kept; as fp32; larger of
// two pairs with NaN winning.
template <typename T>
struct LpPair;
template <>
struct LpPair<__nv_bfloat16> {
  static constexpr float kLowest = -1.2959972171045839e38f;  // 0xfec3
  static constexpr uint32_t kNone = 0xff80ff80u;  // -inf, -inf
  static __device__ __forceinline__ uint32_t finite(uint32_t a) { return larger(a, 0xfec3fec3u); }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float2 floats(uint32_t a) {
    return make_float2(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
  }
};
template <>
struct LpPair<__half> {
  static constexpr float kLowest = -65504.f;
  static constexpr uint32_t kNone = 0xfc00fc00u;
  static __device__ __forceinline__ uint32_t finite(uint32_t a) { return larger(a, 0xfbfffbffu); }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float2 floats(uint32_t a) { return __half22float2(*reinterpret_cast<const __half2*>(&a)); }
};
template <>
struct LpPair<float> {
  static constexpr float kLowest = -kLpRange;
  static constexpr uint32_t kNone = 0xff800000u;
};
__device__ __forceinline__ float lp_max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Sums against a reference m, none of the values more than 8 above it; two
// partial sums, of the even and the odd values.
struct LpSums {
  float m;
  float2 z, s;
  __device__ __forceinline__ void raise(float to) {
    const float by = fmaxf(m - to, -200.f);  // e^-200 is 0
    const float f = fast_exp2(by * kLpLog2e);
    s = make_float2(f * fmaf(by, z.x, s.x), f * fmaf(by, z.y, s.y));
    z = make_float2(z.x * f, z.y * f);
    m = to;
  }
  // x: finite or NaN or +inf
  __device__ __forceinline__ void add(float2 x) {
    const float2 d = lp_add2(x, make_float2(-m, -m));
    const float2 t = lp_mul2(d, make_float2(kLpLog2e, kLpLog2e));
    const float2 e = make_float2(fast_exp2(t.x), fast_exp2(t.y));
    z = lp_add2(z, e);
    s = lp_fma2(d, e, s);
  }
  __device__ __forceinline__ void see(float mx) {  // before values up to mx are added
    if (mx > m + 8.f) raise(mx);
  }
  // The largest of the values of a load, +inf for NaN, after they were added.
  template <typename T>
  __device__ __forceinline__ float add_load(const uint4& raw) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (sizeof(T) == 4) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = lp_max_nan(__uint_as_float(w[i]), -kLpRange);
      const float mx = lp_max_nan(lp_max_nan(x[0], x[1]), lp_max_nan(x[2], x[3]));
      see(mx);
      add(make_float2(x[0], x[1]));
      add(make_float2(x[2], x[3]));
      return mx != mx ? INFINITY : mx;
    } else {
      using P = LpPair<T>;
      uint32_t f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = P::finite(w[i]);
      const float2 h = P::floats(P::larger(P::larger(f[0], f[1]), P::larger(f[2], f[3])));
      const float mx = lp_max_nan(h.x, h.y);
      see(mx);
#pragma unroll
      for (int i = 0; i < 4; ++i) add(P::floats(f[i]));
      return mx != mx ? INFINITY : mx;
    }
  }
  __device__ __forceinline__ void merge(const LpSums& o) {
    const float to = fmaxf(m, o.m);
    LpSums b = o;
    if (m != to) raise(to);
    if (b.m != to) b.raise(to);
    z = lp_add2(z, b.z);
    s = lp_add2(s, b.s);
  }
};

struct __align__(16) LpShared {
  uint64_t keys[kLpCap];
  uint64_t best[kLpMaxTop];     // the k largest so far, sorted
  uint4 queue[kLpQueue];
  int queue_at[kLpQueue];       // their places in the row, in loads
  int queued;
  int low;                      // a load of nothing but values up to kLowest, not all of them -inf, was left out
  float groups[32];
  LpSums sums[kLpWarps];
  int count;                    // keys offered; those past kLpCap are lost
  // what a cluster's first CTA reads
  LpSums total;
  int found;                    // entries of best
};

// The k largest of keys[0, n) to best, sorted; returns how many there are.  Called
// by the CTA; eight lanes count for a key.
__device__ __forceinline__ int lp_rank(LpShared& sh, int n, int k) {
  const int part = threadIdx.x & 7;
  for (int i0 = 0; i0 < n; i0 += kLpThreads / 8) {
    const int i = i0 + threadIdx.x / 8;
    const uint64_t key = i < n ? sh.keys[i] : 0;
    int rank = 0;
#pragma unroll 4
    for (int j = part; j < n; j += 8) rank += sh.keys[j] > key;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (part == 0 && i < n && rank < k) sh.best[rank] = key;
  }
  __syncthreads();
  return min(n, k);
}

// x of all threads brought together, in a fixed order.
template <typename F>
__device__ __forceinline__ float lp_block(LpShared& sh, float x, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.groups[threadIdx.x >> 5] = x;
  __syncthreads();
  x = sh.groups[0];
  for (int w = 1; w < kLpWarps; ++w) x = f(x, sh.groups[w]);
  return x;
}

// TOP: alternatives are wanted.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4) logprobs_kernel(const __grid_constant__ LogprobArgs a) {
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

  if (tid == 0) sh.count = sh.queued = sh.low = 0;
  __syncthreads();

  LpSums mine{-1.5f * kLpRange, make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  uint64_t bound = 0;         // keys below it are not among the k largest
  float floor_v = -INFINITY;  // the bound's value: smaller ones need no key
  auto set_bound = [&](uint64_t key) {
    bound = key;
    floor_v = lp_value(key);
    if (!(floor_v > LpPair<T>::kLowest)) floor_v = -INFINITY;  // among values that the maxima below are too high for
    if (floor_v != floor_v) floor_v = INFINITY;                // NaN: only what ranks as +inf or NaN comes near
  };
  auto offer = [&](float x, int index) {
    if (x == -INFINITY) return;  // never a candidate; filled in at the end where others are missing
    const uint64_t key = lp_key(x, index);
    if (key < bound) return;
    const int at = atomicAdd(&sh.count, 1);
    if (at < kLpCap) sh.keys[at] = key;
  };
  // the values of the loads in the queue; between barriers
  auto drain = [&]() {
    const int n = min(sh.queued, kLpQueue) * V;
    for (int i = tid; i < n; i += kLpThreads) {
      const float x = N::to_f(reinterpret_cast<const T*>(sh.queue)[i]);
      if (!(x < floor_v)) offer(x, head + sh.queue_at[i / V] * V + i % V);
    }
  };
  // the k best of the buffer alone stay in it, and bound what may come
  auto prune = [&]() {
    const int n = min(sh.count, kLpCap);
    if (n >= k) {
      lp_rank(sh, n, k);
      set_bound(sh.best[k - 1]);
      if (tid < k) sh.keys[tid] = sh.best[tid];
      if (tid == 0) sh.count = k;
    }
    __syncthreads();
  };

  uint4 next[U];
  auto fetch = [&](int from) {
    if (from + U * kLpThreads <= v1) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = __ldcs(vec + from + u * kLpThreads + tid);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = from + u * kLpThreads + tid;
        if (v < v1) next[u] = __ldcs(vec + v);
      }
    }
  };
  fetch(v0);
  for (int from = v0; from < v1; from += U * kLpThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
    fetch(from + U * kLpThreads);
    float top[U];
    if (from + U * kLpThreads <= v1) {
#pragma unroll
      for (int u = 0; u < U; ++u) top[u] = mine.template add_load<T>(raw[u]);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        top[u] = from + u * kLpThreads + tid < v1 ? mine.template add_load<T>(raw[u]) : -INFINITY;
    }
    if constexpr (TOP) {
      float most = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) most = fmaxf(most, top[u]);
      if (from == v0) {
        // the first bound: the k-th largest of 32 groups' largest
        float h = most;
#pragma unroll
        for (int o = 1; o < kLpThreads / 32; o <<= 1) h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, o));
        if (tid % (kLpThreads / 32) == 0) sh.groups[tid / (kLpThreads / 32)] = h;
        __syncthreads();
        const float g = sh.groups[lane];
        int above = 0;
        for (int j = 0; j < 32; ++j) above += sh.groups[j] > g || (sh.groups[j] == g && j < lane);
        const unsigned at = __ballot_sync(0xffffffffu, above == k - 1);
        const float b = __shfl_sync(0xffffffffu, g, __ffs(at) - 1);
        if (b > LpPair<T>::kLowest) set_bound((lp_key(b, 0) >> 32) << 32);  // that value at any index
      }
      // loads that hold something above kLowest, and above the bound where there is one
      const float gate = fmaxf(floor_v, __uint_as_float(__float_as_uint(LpPair<T>::kLowest) - 1u));
      if (most >= gate) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int v = from + u * kLpThreads + tid;
          if (v < v1 && top[u] >= gate) {
            const int at = atomicAdd(&sh.queued, 1);
            if (at < kLpQueue) {
              sh.queue[at] = raw[u];
              sh.queue_at[at] = v;
            }
          }
        }
      }
      if (floor_v == -INFINITY) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (from + u * kLpThreads + tid < v1 && top[u] < gate &&
              (raw[u].x != LpPair<T>::kNone || raw[u].y != LpPair<T>::kNone || raw[u].z != LpPair<T>::kNone ||
               raw[u].w != LpPair<T>::kNone))
            sh.low = 1;
        }
      }
      // behind rounds 1, 2, 4, 8, ...: about k values of each doubling pass the bound
      const int round = (from - v0) / (U * kLpThreads) + 1;
      if ((round & (round - 1)) == 0) {
        __syncthreads();
        if (sh.queued <= kLpQueue) {  // the same for all threads
          drain();
          __syncthreads();
          const bool fit = sh.count <= kLpCap;
          __syncthreads();
          if (fit) {
            if (tid == 0) sh.queued = 0;
            prune();
          }
        }
      }
    }
  }
  if constexpr (TOP) {
    __syncthreads();
    drain();
  }
  // the value in front of the first vector (first CTA) or behind the last one (last CTA) that this thread has
  const int tail = a.cols - head - nvec * V;
  int lone = -1;
  if (part == 0 && tid < head) lone = tid;
  else if (part == parts - 1 && tid >= 32 && tid - 32 < tail) lone = head + nvec * V + tid - 32;
  if (lone >= 0) {
    const float x = N::to_f(row[lone]), y = lp_max_nan(x, LpPair<T>::kLowest);
    mine.see(y);
    const LpSums before = mine;
    mine.add(make_float2(y, y));
    mine.z.y = before.z.y, mine.s.y = before.s.y;  // one value, not two
    if (TOP) offer(x, lone);
  }
  if constexpr (TOP) {
    __syncthreads();
    bool again = sh.count > kLpCap || sh.queued > kLpQueue;  // some were lost
    if (!again && sh.low) {  // some were left out: needed if one of their kind is among the k best
      const int n = sh.count;
      if (n >= k) lp_rank(sh, n, k);
      again = n < k || !(lp_value(sh.best[k - 1]) > LpPair<T>::kLowest);
    }
    if (again) {
      // all again, the bound raised on the way; a round's 256 values and 512 keys fit
      __syncthreads();
      if (tid == 0) sh.count = 0;
      set_bound(0);
      __syncthreads();
      if (lone >= 0) offer(N::to_f(row[lone]), lone);
      for (int64_t c0 = (int64_t)v0 * V; c0 < (int64_t)v1 * V; c0 += kLpThreads) {
        if (c0 + tid < (int64_t)v1 * V) offer(N::to_f(row[head + c0 + tid]), (int)(head + c0) + tid);
        __syncthreads();
        const bool long_enough = sh.count > kLpCap / 2;
        __syncthreads();
        if (long_enough) prune();
      }
      prune();
    }
  }
  // sums of the CTA, its best keys
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpSums other{__shfl_down_sync(0xffffffffu, mine.m, o),
                 make_float2(__shfl_down_sync(0xffffffffu, mine.z.x, o), __shfl_down_sync(0xffffffffu, mine.z.y, o)),
                 make_float2(__shfl_down_sync(0xffffffffu, mine.s.x, o), __shfl_down_sync(0xffffffffu, mine.s.y, o))};
    mine.merge(other);
  }
  if (lane == 0) sh.sums[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    LpSums t = sh.sums[0];
    for (int w = 1; w < kLpWarps; ++w) t.merge(sh.sums[w]);
    sh.total = t;
  }
  const int found = TOP ? lp_rank(sh, sh.count, k) : 0;
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
      if (TOP) {
        const int f = lp_rank(sh, n, k);
        if (tid == 0) sh.found = f;
      }
    }
    cluster.sync();  // the others stay until their shared memory has been read
    if (part != 0) return;
  }
  __syncthreads();
  const float nan = __int_as_float(0x7fc00000);
  float m = sh.total.m, z = sh.total.z.x + sh.total.z.y, s = sh.total.s.x + sh.total.s.y;
  float log_z = logf(z);
  const bool usual = m > LpPair<T>::kLowest && m < kLpRange && z == z;
  if (!usual) {
    bool none = true, bad = false;  // nothing but -inf; NaN or +inf somewhere
    float mx = -INFINITY;
    for (int i = tid; i < a.cols; i += kLpThreads) {
      const float x = N::to_f(row[i]);
      mx = fmaxf(mx, x);
      none = none && x == -INFINITY;
      bad = bad || !(x < INFINITY);
    }
    none = __syncthreads_and(none);
    bad = __syncthreads_or(bad);
    mx = lp_block(sh, mx, [](float p, float q) { return fmaxf(p, q); });
    z = s = 0.f;
    for (int i = tid; i < a.cols; i += kLpThreads) {
      const float d = N::to_f(row[i]) - mx, e = expf(d);
      z += e;
      if (e != 0.f) s = fmaf(d, e, s);
    }
    z = lp_block(sh, z, [](float p, float q) { return p + q; });
    s = lp_block(sh, s, [](float p, float q) { return p + q; });
    m = mx;
    log_z = none || bad ? nan : logf(z);
  }
  if (tid == 0) {
    const int64_t token = a.tokens[r];
    const bool ok = token >= 0 && token < a.cols;
    if (!ok) raise_flag(a.err, NIE_DEV_ERR_INDEX_RANGE);
    a.logprobs[r] = ok ? N::to_f(row[token]) - m - log_z : nan;
    a.entropy[r] = log_z - s / z;
  }
  if (tid < sh.found) {
    const uint64_t key = sh.best[tid];
    a.top_logprobs[r * k + tid] = lp_value(key) - m - log_z;
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
        a.top_logprobs[r * k + mine_at] = -INFINITY - m - log_z;
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
  const cudaError_t e = a.top > 0 ? cudaLaunchKernelEx(&cfg, logprobs_kernel<T, true>, a)
                                  : cudaLaunchKernelEx(&cfg, logprobs_kernel<T, false>, a);
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
  // Rows that do not bring a CTA to each SM are split, down to a round's worth of values.  128256 bf16 values, 5
  // alternatives, in 1, 2, 4 and 8 parts: one row 17.4, 13.5, 11.5 and 11.4 us, 64 rows 17.8, 14.5, 13.5 and 16.2,
  // 128 rows 17.9, 16.6, 18.3 and 29, 256 rows 22, 24, 33 and 54.
  const int64_t round = (int64_t)kLpThreads * 4 * (16 / dtype_size(dtype));
  int parts = 1;
  while (parts < kLpMaxCluster && rows * parts <= sms && cols > parts * round) parts *= 2;
  LogprobArgs a{logits, row_stride, (int)cols, tokens, top, logprobs, entropy, top_logprobs, top_ids, err_flag};
  switch (dtype) {
    case NIE_DTYPE_BF16: return launch_logprobs<__nv_bfloat16>(a, rows, parts, s);
    case NIE_DTYPE_F32: return launch_logprobs<float>(a, rows, parts, s);
    default: return launch_logprobs<__half>(a, rows, parts, s);
  }
}
