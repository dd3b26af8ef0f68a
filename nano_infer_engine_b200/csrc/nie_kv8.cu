// Appending to and reading back the 8-bit paged cache.
//
//   rope_write_kv8 : q' = rope(q); k' = rope(k); k' and v go to the cache
//                    slots in e4m3 with one scale per (block, kv head)
//   write_kv8      : the same without the rotation (k stored as given)
//   gather_kv8     : a table's tokens as values (code * scale)
//
// Rotation: (a, b) -> (a c - b s, b c + a s) on the halves of a head, in fp32
// without fused multiply-add, rounded once: q' to the activation type, k'
// straight to 8 bits.
//
// Scale of a block: tokens of one call that are neighbours, lie in one block
// and have slots that follow one another ("a run") share s = 2^e, the least power of
// two with max|x| <= 448 s.  A run that continues a block (its first slot is
// not the block's first) never lowers the block's scale; where it raises it,
// the codes before the run are brought to the new scale; those behind it are not
// looked at, and a run that begins a block replaces the scale: a block is appended to.  A power of two
// costs no precision in a floating format and makes that step exact except
// for codes that become subnormal.  Scales stay in [2^-48, 2^48]; values
// beyond 448 * 2^48 saturate.  Non-finite values are stored as NaN and do not
// count for the scale.
//
// What bounds it: each byte in and out once, some 60 operations to 16 of them, so
// bandwidth from a few thousand tokens on and latency below.  One kernel does all:
// some CTAs rotate queries, the others store; rows move in 16-byte pieces, and a lane's
// first pair of them stays in registers between the run's maximum and its codes.
// Registers decide: with two pairs and four CTAs to an SM the loops' state went to
// memory and 16384 tokens (32 + 2 x 8 heads of 64, bf16) took 55 us; with one and
// three CTAs 43 us, 185 MB at 4.3 TB/s, of which the queries' 134 MB take 24.  fp32
// rows 68 us.  Other sizes and alignments take the plain kernel: 2048 tokens of heads of
// 72 62 us, where those of 64 take 7.
//
// One warp owns a (block, kv head, K or V) and takes the block's runs in turn,
// as calls of their own would be, so no two warps write one scale or one code
// and the result does not depend on the order of the warps.
#include "nie_kv8.cuh"

#include <algorithm>

namespace nie {

struct AppendArgs {
  const void* q;  // null: no queries to rotate
  const void* k;
  const void* v;
  int64_t q_stride, k_stride, v_stride;  // elements between token rows
  const void* sin;  // null: k is stored as given
  const void* cos;
  int64_t tokens;
  int hq, hkv, hd, bs;
  void* q_out;
  uint8_t* codes[2];   // K, V codes of the layer
  float* scales[2];    // K, V scales of the layer
  int64_t total_slots;
  const int64_t* slots;
  int32_t* err;
};

// The block of a token's slot; -1 for a token that is not stored.
__device__ __forceinline__ int64_t block_of(const AppendArgs& a, int64_t t) {
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.total_slots) return -1;
  // a 32-bit division is a fifth of a 64-bit one
  return slot <= 0xffffffffll ? (int64_t)((uint32_t)slot / (uint32_t)a.bs) : slot / a.bs;
}

// The nearest stored token from t on, forwards (dir 1) or backwards (-1), or -1.  Called by a whole warp.  A padded
// call has thousands of tokens without a slot in a row: 256 are looked at together.  One token in a write of 16384
// rows takes 33 us so, 1.8 ms where they are looked at one after the other; 16384 tokens 20 us.
__device__ __forceinline__ int64_t nearest_stored(const AppendArgs& a, int64_t t, int dir) {
  constexpr int kLoads = 8;
  const int lane = threadIdx.x & 31;
  for (; t >= 0 && t < a.tokens; t += dir * 32 * kLoads) {
    int64_t slot[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int64_t i = t + dir * (j * 32 + lane);
      slot[j] = i >= 0 && i < a.tokens ? a.slots[i] : -1;
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const unsigned stored = __ballot_sync(0xffffffffu, slot[j] >= 0 && slot[j] < a.total_slots);
      if (stored) return t + dir * (j * 32 + __ffs(stored) - 1);
    }
  }
  return -1;
}

// True if token t (of block >= 0) is the first of its block's stretch: the
// stored token before it, tokens without a slot passed over, lies elsewhere.  Called by a whole warp.
__device__ __forceinline__ bool begins_block(const AppendArgs& a, int64_t t, int64_t block) {
  if (t == 0) return true;
  int64_t b = block_of(a, t - 1);
  if (b < 0) {
    const int64_t p = nearest_stored(a, t - 1, -1);
    if (p >= 0) b = block_of(a, p);
  }
  return b != block;
}

// Number of tokens of the run that starts at t: slots that follow one another in
// one block.  Called by a whole warp.
__device__ __forceinline__ int run_length(const AppendArgs& a, int64_t t, int64_t block) {
  const int64_t slot = a.slots[t];
  const int most = (int)min(a.tokens - t, (block + 1) * a.bs - slot);
  for (int n = 0; n < most; n += 32) {
    const int i = n + (int)(threadIdx.x & 31);
    const unsigned same = __ballot_sync(0xffffffffu, i < most && a.slots[t + i] == slot + i);
    if (same != 0xffffffffu) return n + __ffs(~same) - 1;
  }
  return most;
}

// First token of the block's next run from token t on, or -1: tokens without a slot are passed over.  Called by a
// whole warp.
__device__ __forceinline__ int64_t next_run(const AppendArgs& a, int64_t t, int64_t block) {
  if (t >= a.tokens) return -1;
  if (block_of(a, t) < 0) t = nearest_stored(a, t, 1);
  return t >= 0 && block_of(a, t) == block ? t : -1;
}

// A value that has no 8-bit form becomes NaN.
__device__ __forceinline__ float finite_or_nan(float x) {
  return fabsf(x) <= 3.402823466e38f ? x : __int_as_float(0x7fc00000);
}

// The least power of two whose 448-fold is not below amax, in the bounds:
// 448 = 1.75 * 2^8, so with amax = m 2^e (1 <= m < 2) it is 2^(e-8), or
// 2^(e-7) when m > 1.75.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) + ((bits & 0x7fffffu) > 0x600000u ? -7 : -8);  // biased
  if (e <= 127 - 48) return kScaleMin;
  if (e >= 127 + 48) return kScaleMax;
  return __uint_as_float((uint32_t)e << 23);
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// New scale of a block for a run whose largest magnitude is `amax`; the codes
// of the rows [0, off) are brought to it.  Called by a whole warp.
__device__ __forceinline__ float settle_scale(const AppendArgs& a, int kv, int64_t block, int head, int off, float amax,
                                              int lane) {
  float* sp = a.scales[kv] + block * a.hkv + head;
  float s = scale_for(amax);
  if (off > 0) {
    const float old = fminf(fmaxf(*sp, kScaleMin), kScaleMax);
    if (s > old) {
      const float ratio = old / s;
      const int64_t row = (int64_t)a.hkv * a.hd;
      uint8_t* base = a.codes[kv] + block * a.bs * row + (int64_t)head * a.hd;
      for (int i = lane; i < off * a.hd; i += 32) {
        uint8_t* c = base + (int64_t)(i / a.hd) * row + i % a.hd;
        *c = (uint8_t)floats_to_e4m3x2(e4m3_to_float(*c) * ratio, 0.f);
      }
    } else {
      s = old;
    }
  }
  __syncwarp();
  if (lane == 0) *sp = s;
  return s;
}

// One CTA per token: its warps rotate the token's queries and, where a run
// begins, take the run's (K / V, head) pairs in turn.  Any even head_dim, any
// alignment; a run's values are read twice.
template <typename T>
__global__ void __launch_bounds__(256) append_kv8_kernel(AppendArgs a) {
  using N = Num<T>;
  pdl_wait();     // dependent launch: q/k/v come from the projection before
  pdl_trigger();  // the kernel after this one may start its prologue
  const int64_t t = blockIdx.x;
  const int half = a.hd / 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const T* sn = reinterpret_cast<const T*>(a.sin);
  const T* cs = reinterpret_cast<const T*>(a.cos);
  if (a.q) {
    const T* q = reinterpret_cast<const T*>(a.q) + t * a.q_stride;
    T* out = reinterpret_cast<T*>(a.q_out) + t * a.hq * a.hd;
    for (int p = threadIdx.x; p < a.hq * half; p += blockDim.x) {
      const int h = p / half, i = p % half;
      const float x1 = N::to_f(q[h * a.hd + i]), x2 = N::to_f(q[h * a.hd + i + half]);
      const float c = N::to_f(cs[t * half + i]), s = N::to_f(sn[t * half + i]);
      out[h * a.hd + i] = N::from_f(__fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s)));
      out[h * a.hd + i + half] = N::from_f(__fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s)));
    }
  }
  if (a.slots[t] >= a.total_slots && threadIdx.x == 0) raise_flag(a.err, NIE_DEV_ERR_SLOT_RANGE);
  const int64_t block = block_of(a, t);
  if (block < 0 || !begins_block(a, t, block)) return;
  const int64_t row = (int64_t)a.hkv * a.hd;
  for (int task = warp; task < 2 * a.hkv; task += warps) {
    const int kv = task >= a.hkv, head = task - kv * a.hkv;
    const bool rotate = kv == 0 && a.sin != nullptr;
    const T* src = reinterpret_cast<const T*>(kv ? a.v : a.k);
    const int64_t stride = kv ? a.v_stride : a.k_stride;
    for (int64_t first = t; first >= 0;) {
      const int n = run_length(a, first, block);
      const int off = (int)(a.slots[first] - block * a.bs);
      auto value = [&](int j, int d) -> float {
        const T* x = src + (first + j) * stride + (int64_t)head * a.hd;
        if (!rotate) return finite_or_nan(N::to_f(x[d]));
        const int i = d < half ? d : d - half;
        const float x1 = N::to_f(x[i]), x2 = N::to_f(x[i + half]);
        const float c = N::to_f(cs[(first + j) * half + i]), s = N::to_f(sn[(first + j) * half + i]);
        return finite_or_nan(d < half ? __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s))
                                      : __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s)));
      };
      float amax = 0.f;
      for (int i = lane; i < n * a.hd; i += 32) amax = fmaxf(amax, fabsf(value(i / a.hd, i % a.hd)));  // skips NaN
      const float s = settle_scale(a, kv, block, head, off, warp_max(amax), lane);
      uint8_t* dst = a.codes[kv] + (block * a.bs + off) * row + (int64_t)head * a.hd;
      for (int i = lane; i < n * a.hd; i += 32)
        dst[(int64_t)(i / a.hd) * row + i % a.hd] = (uint8_t)floats_to_e4m3x2(value(i / a.hd, i % a.hd) / s, 0.f);
      __syncwarp();
      first = next_run(a, first + n, block);
    }
  }
}

// ------------------------------------------------ 16-byte variants
// The same arithmetic for rows whose halves are whole 16-byte pieces at 16-byte
// boundaries, and head_dim a multiple of 16 (that of the codes' pieces).
template <typename T>
struct Piece {
  static constexpr int V = 16 / (int)sizeof(T);
  float f[V];
  __device__ __forceinline__ void load(const T* p) { expand(*reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void expand(const uint4 u) {
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = Num<T>::to_f(e[i]);
  }
  __device__ __forceinline__ void store(T* p) const {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = Num<T>::from_f(f[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
  // V codes of f / s; s a power of two: f * inv is the quotient
  __device__ __forceinline__ void store_codes(uint8_t* p, float s, float inv) const {
    uint16_t c[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      c[i] = inv != 0.f ? floats_to_e4m3x2(f[2 * i] * inv, f[2 * i + 1] * inv) : floats_to_e4m3x2(f[2 * i] / s, f[2 * i + 1] / s);
    if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(c);
    else *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(c);
  }
};

// Rotation of a pair of pieces from the loaded words, so that no more of them than needed are values at a time.
template <typename T>
__device__ __forceinline__ void rotate_raw(const uint4& a, const uint4& b, const uint4& c, const uint4& s, Piece<T>& x, Piece<T>& y) {
  const T *pa = reinterpret_cast<const T*>(&a), *pb = reinterpret_cast<const T*>(&b);
  const T *pc = reinterpret_cast<const T*>(&c), *ps = reinterpret_cast<const T*>(&s);
#pragma unroll
  for (int i = 0; i < Piece<T>::V; ++i) {
    const float u = Num<T>::to_f(pa[i]), v = Num<T>::to_f(pb[i]), co = Num<T>::to_f(pc[i]), si = Num<T>::to_f(ps[i]);
    x.f[i] = __fsub_rn(__fmul_rn(u, co), __fmul_rn(v, si));
    y.f[i] = __fadd_rn(__fmul_rn(v, co), __fmul_rn(u, si));
  }
}

// The codes of a block's rows [0, off) times ratio, 16 a lane.
__device__ __noinline__ void rescale_codes(uint8_t* base, int64_t row, int hd, int off, float ratio) {
  const int per_row = hd / 16;
  for (int i = threadIdx.x & 31; i < off * per_row; i += 32) {
    uint4* p = reinterpret_cast<uint4*>(base + (int64_t)(i / per_row) * row + i % per_row * 16);
    uint4 u = *p;
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 lo = f16x2_to_float2(e4m3x2_to_f16x2((uint16_t)(w[e] & 0xffffu)));
      const float2 hi = f16x2_to_float2(e4m3x2_to_f16x2((uint16_t)(w[e] >> 16)));
      w[e] = (uint32_t)floats_to_e4m3x2(lo.x * ratio, lo.y * ratio) |
             ((uint32_t)floats_to_e4m3x2(hi.x * ratio, hi.y * ratio) << 16);
    }
    *p = u;
  }
}

// settle_scale() on it.
__device__ __forceinline__ float settle_scale_vec(const AppendArgs& a, int kv, int64_t block, int head, int off, float amax,
                                                  int lane) {
  float* sp = a.scales[kv] + block * a.hkv + head;
  float s = scale_for(amax);
  if (off > 0) {
    const float old = fminf(fmaxf(*sp, kScaleMin), kScaleMax);
    if (s > old) {
      const int64_t row = (int64_t)a.hkv * a.hd;
      rescale_codes(a.codes[kv] + block * a.bs * row + (int64_t)head * a.hd, row, a.hd, off, old / s);
    } else {
      s = old;
    }
  }
  __syncwarp();
  if (lane == 0) *sp = s;
  return s;
}

constexpr int kQHeads = 4;  // query heads that a thread rotates with one piece of sin and cos

// CTAs [0, kv_ctas): `tile` tokens each and K (even) or V (odd), the heads of whose
// blocks the warps take in turn; first, since theirs is the longer chain of loads.
// The others: a thread rotates one pair of pieces of kQHeads heads of a token.
template <typename T>
__global__ void __launch_bounds__(256, 3) append_kv8_vec_kernel(const __grid_constant__ AppendArgs a, int kv_ctas, int tile) {
  constexpr int V = Piece<T>::V;
  pdl_wait();     // dependent launch: q/k/v come from the projection before
  pdl_trigger();  // the kernel after this one may start its prologue
  const int half = a.hd / 2, per_half = half / V;
  const T* sn = reinterpret_cast<const T*>(a.sin);
  const T* cs = reinterpret_cast<const T*>(a.cos);
  if ((int)blockIdx.x >= kv_ctas) {
    const int sets = (a.hq + kQHeads - 1) / kQHeads, per_token = per_half * sets;
    const int64_t x = (int64_t)(blockIdx.x - kv_ctas) * 256 + threadIdx.x;
    const int64_t t = x <= 0xffffffffll ? (int64_t)((uint32_t)x / (uint32_t)per_token) : x / per_token;
    if (t >= a.tokens) return;
    const int e = (int)(x - t * per_token);
    const int c = e % per_half * V, h0 = e / per_half * kQHeads;
    const T* q = reinterpret_cast<const T*>(a.q) + t * a.q_stride + (int64_t)h0 * a.hd + c;
    T* out = reinterpret_cast<T*>(a.q_out) + (t * a.hq + h0) * a.hd + c;
    uint4 lo[kQHeads], hi[kQHeads];  // all loads go out together
#pragma unroll
    for (int h = 0; h < kQHeads; ++h) {
      if (h0 + h < a.hq) {
        lo[h] = *reinterpret_cast<const uint4*>(q + h * a.hd);
        hi[h] = *reinterpret_cast<const uint4*>(q + h * a.hd + half);
      }
    }
    const uint4 co = *reinterpret_cast<const uint4*>(cs + t * half + c), si = *reinterpret_cast<const uint4*>(sn + t * half + c);
#pragma unroll
    for (int h = 0; h < kQHeads; ++h) {
      if (h0 + h < a.hq) {
        Piece<T> x, y;
        rotate_raw(lo[h], hi[h], co, si, x, y);
        x.store(out + h * a.hd);
        y.store(out + h * a.hd + half);
      }
    }
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kv = blockIdx.x & 1;
  const int t0 = (int)(blockIdx.x >> 1) * tile;
  // Lane i looks at token t0 - 1 + i, so that the tile's blocks and the runs at their
  // beginnings (16 tokens at least) follow from one load.
  const int seen = t0 - 1 + lane, tokens = (int)a.tokens;
  int my_block = -1, my_off = 0;  // its block, and its place in it
  if (seen >= 0 && seen < tokens) {
    my_block = (int)block_of(a, seen);
    if (my_block >= 0) my_off = (int)(a.slots[seen] - (int64_t)my_block * a.bs);
    if (lane >= 1 && lane <= tile && kv == 0 && a.slots[seen] >= a.total_slots) raise_flag(a.err, NIE_DEV_ERR_SLOT_RANGE);
  }
  const int before_off = __shfl_up_sync(0xffffffffu, my_off, 1), before_block = __shfl_up_sync(0xffffffffu, my_block, 1);
  bool begins = lane >= 1 && lane <= tile && my_block >= 0;
  // the block of the stored token before: in this window, or for its first one in front of it
  const unsigned before = __ballot_sync(0xffffffffu, my_block >= 0) & ((1u << lane) - 1);
  int last_block = __shfl_sync(0xffffffffu, my_block, before ? 31 - __clz(before) : 0);
  if (__any_sync(0xffffffffu, begins && !before) && t0 > 1) {
    const int64_t p = nearest_stored(a, t0 - 2, -1);
    if (!before) last_block = p >= 0 ? (int)block_of(a, p) : -1;
  }
  begins = begins && last_block != my_block;
  const unsigned heads = __ballot_sync(0xffffffffu, begins) >> 1;  // bit i: token t0 + i
  const unsigned goes_on = __ballot_sync(0xffffffffu, lane >= 1 && my_block >= 0 && my_block == before_block && my_off == before_off + 1);
  const int rank = __popc((heads << 1) & ((1u << lane) - 1));  // stretches that begin before this lane's token
  const int tasks = __popc(heads) * a.hkv;
  const int row_lanes = per_half, rows = 32 / row_lanes;  // lanes of a row, rows of a pass
  const int c = lane % row_lanes * V, sub = lane / row_lanes;
  const bool in = sub < rows;  // row_lanes need not divide 32
  const int64_t row = (int64_t)a.hkv * a.hd;
  for (int task = warp; task < tasks; task += 8) {
    const int nth = task / a.hkv;
    const int which = __ffs(__ballot_sync(0xffffffffu, begins && rank == nth)) - 2;  // the lane behind it is token t0 + which
    const int64_t block = __shfl_sync(0xffffffffu, my_block, which + 1);
    const int head = task - nth * a.hkv;
    const bool rotate = kv == 0 && a.sin != nullptr;
    const T* src = reinterpret_cast<const T*>(kv ? a.v : a.k) + (int64_t)head * a.hd + c;
    const int64_t stride = kv ? a.v_stride : a.k_stride;
    // the first run from the lanes, and whether another one can follow it in the block
    const unsigned stops = ~goes_on >> (which + 1) & ~1u;
    int n = stops ? __ffs(stops) - 1 : 32;
    const bool known = which + 1 + n < 32;
    int off = __shfl_sync(0xffffffffu, my_off, which + 1);
    const int behind = __shfl_sync(0xffffffffu, my_block, known ? which + 1 + n : 0);
    const bool alone = known && (t0 + which + n >= tokens || (behind >= 0 && behind != (int)block));
    if (!known) n = run_length(a, t0 + which, block);
    for (int first = t0 + which; first >= 0;) {
      bool strict = false;  // an infinite value is about: each value is looked at
      auto get = [&](int j, Piece<T>& lo, Piece<T>& hi) {
        const T* x = src + (first + j) * stride;
        const uint4 lo_raw = *reinterpret_cast<const uint4*>(x), hi_raw = *reinterpret_cast<const uint4*>(x + half);
        if (rotate) {
          const int64_t at = (int64_t)(first + j) * half + c;
          rotate_raw(lo_raw, hi_raw, *reinterpret_cast<const uint4*>(cs + at), *reinterpret_cast<const uint4*>(sn + at), lo, hi);
        } else {
          lo.expand(lo_raw);
          hi.expand(hi_raw);
        }
        if (strict) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            lo.f[i] = finite_or_nan(lo.f[i]);
            hi.f[i] = finite_or_nan(hi.f[i]);
          }
        }
      };
      Piece<T> lo, hi;  // the lane's first pair of pieces stays; further ones are read again
      float amax;
      for (;;) {
        amax = 0.f;
        auto largest = [&](const Piece<T>& p, const Piece<T>& q) {
#pragma unroll
          for (int i = 0; i < V; ++i) amax = fmaxf(amax, fmaxf(fabsf(p.f[i]), fabsf(q.f[i])));  // skips NaN
        };
        if (in && sub < n) {
          get(sub, lo, hi);
          largest(lo, hi);
        }
        for (int j = rows + sub; in && j < n; j += rows) {
          Piece<T> p, q;
          get(j, p, q);
          largest(p, q);
        }
        amax = warp_max(amax);
        if (strict || amax != INFINITY) break;
        strict = true;
      }
      const float s = settle_scale_vec(a, kv, block, head, off, amax, lane);
      const uint32_t bits = __float_as_uint(s);
      const float inv = (bits & 0x7fffffu) == 0 ? __uint_as_float((254u << 23) - bits) : 0.f;
      uint8_t* dst = a.codes[kv] + (block * a.bs + off) * row + (int64_t)head * a.hd + c;
      auto put = [&](int j, const Piece<T>& p, const Piece<T>& q) {
        p.store_codes(dst + j * row, s, inv);
        q.store_codes(dst + j * row + half, s, inv);
      };
      if (in && sub < n) put(sub, lo, hi);
      for (int j = rows + sub; in && j < n; j += rows) {
        Piece<T> p, q;
        get(j, p, q);
        put(j, p, q);
      }
      if (alone) break;
      __syncwarp();
      first = (int)next_run(a, first + n, block);
      if (first >= 0) {
        n = run_length(a, first, block);
        off = (int)(a.slots[first] - block * a.bs);
      }
    }
  }
}

// Values of a table's first n tokens, 16 of K or V to a thread: 16384 tokens of 8 heads of 64 as bf16 in 10.7 us (50
// MB at 4.7 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) gather_kv8_vec_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                             const float* __restrict__ ks, const float* __restrict__ vs,
                                                             int64_t nb, int bs, int hkv, int hd,
                                                             const int32_t* __restrict__ table, int64_t n,
                                                             T* __restrict__ ok, T* __restrict__ ov,
                                                             int32_t* __restrict__ err) {
  const int per_head = hd / 16, per_row = hkv * per_head;
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = x / per_row;
  if (t >= n) return;
  const int e = (int)(x % per_row), head = e / per_head;
  const int64_t block = table[t / bs];
  const bool there = block >= 0 && block < nb;
  if (!there) raise_flag(err, NIE_DEV_ERR_BLOCK_RANGE);
  const int64_t at = ((there ? block * bs + t % bs : 0) * per_row + e) * 16;
  const int64_t scale_at = (there ? block : 0) * hkv + head;
  const uint4 raw[2] = {*reinterpret_cast<const uint4*>(kc + at), *reinterpret_cast<const uint4*>(vc + at)};
  const float scale[2] = {ks[scale_at], vs[scale_at]};
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const uint32_t w[4] = {raw[kv].x, raw[kv].y, raw[kv].z, raw[kv].w};
    float f[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 p = f16x2_to_float2(e4m3x2_to_f16x2((uint16_t)(w[i / 2] >> (16 * (i & 1)))));
      f[2 * i] = there ? p.x * scale[kv] : 0.f;
      f[2 * i + 1] = there ? p.y * scale[kv] : 0.f;
    }
    T* out = (kv ? ov : ok) + x * 16;
#pragma unroll
    for (int i = 0; i < 16; i += Piece<T>::V) {
      Piece<T> p;
#pragma unroll
      for (int u = 0; u < Piece<T>::V; ++u) p.f[u] = f[i + u];
      p.store(out + i);
    }
  }
}

// Values of a table's first T tokens, one element per thread and step.
template <typename T>
__global__ void __launch_bounds__(256) gather_kv8_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                         const float* __restrict__ ks, const float* __restrict__ vs,
                                                         int64_t nb, int bs, int hkv, int hd,
                                                         const int32_t* __restrict__ table, int64_t n,
                                                         T* __restrict__ ok, T* __restrict__ ov,
                                                         int32_t* __restrict__ err) {
  const int64_t row = (int64_t)hkv * hd;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n * row; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / row;
    const int e = (int)(i % row);
    const int64_t block = table[t / bs];
    float k = 0.f, v = 0.f;
    if (block < 0 || block >= nb) {
      raise_flag(err, NIE_DEV_ERR_BLOCK_RANGE);
    } else {
      const int64_t at = (block * bs + t % bs) * row + e;
      k = e4m3_to_float(kc[at]) * ks[block * hkv + e / hd];
      v = e4m3_to_float(vc[at]) * vs[block * hkv + e / hd];
    }
    ok[i] = Num<T>::from_f(k);
    ov[i] = Num<T>::from_f(v);
  }
}

static bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
static void launch_append(const AppendArgs& a, cudaStream_t s) {
  constexpr int V = Piece<T>::V;
  if (a.hd % 16 == 0 && a.hd / 2 % V == 0 && a.hd / 2 / V <= 32 && a.k_stride % V == 0 && a.v_stride % V == 0 &&
      (!a.q || a.q_stride % V == 0) && at16(a.q) && at16(a.k) && at16(a.v) && at16(a.sin) && at16(a.cos) && at16(a.q_out) &&
      at16(a.codes[0]) && at16(a.codes[1]) && a.tokens <= (1 << 30) && a.total_slots / a.bs < (int64_t(1) << 31)) {
    const int64_t threads = a.q ? a.tokens * (a.hd / 2 / V) * ((a.hq + kQHeads - 1) / kQHeads) : 0;
    const int64_t q_ctas = (threads + 255) / 256;
    // Tokens to a CTA.  Few are likely to be of as many requests and lie in as many blocks, which a CTA takes in
    // turn; many are of prompts, whose neighbours share blocks.  With 1, 8 and 16 to a CTA (8 kv heads of 64):
    // 64 tokens of as many requests 3.6, 15 and 28 us, 512 9.4, 16 and 28, 4096 56, 46 and 57; of one prompt 512
    // tokens 6.8, 5.4 and 4.5 us, 2048 14.8, 7.2 and 6.7, 16384 116, 49 and 44.
    const int tile = a.tokens <= 512 ? 1 : a.tokens <= 4096 ? 8 : 16;
    const int64_t kv_ctas = 2 * ((a.tokens + tile - 1) / tile);
    if (q_ctas + kv_ctas < (int64_t(1) << 31)) {
      pdl_launch(append_kv8_vec_kernel<T>, dim3((unsigned)(q_ctas + kv_ctas)), dim3(256), s, a, (int)kv_ctas, tile);
      return;
    }
  }
  pdl_launch(append_kv8_kernel<T>, dim3((unsigned)a.tokens), dim3(256), s, a);
}

static int append(AppendArgs a, void* key_codes, void* value_codes, float* key_scales, float* value_scales,
                  int32_t dtype, int32_t layer, int64_t num_layers, int64_t num_blocks, cudaStream_t s) {
  NIE_REQUIRE(a.k && a.v && key_codes && value_codes && key_scales && value_scales && a.slots, "null pointer argument");
  NIE_REQUIRE(a.tokens >= 0 && a.tokens < (int64_t(1) << 31), "num_tokens out of range");
  NIE_REQUIRE(layer >= 0 && layer < num_layers, "layer %d out of range", layer);
  NIE_REQUIRE(a.hkv > 0 && a.hd > 0 && a.bs > 0 && num_blocks > 0, "bad cache geometry");
  NIE_REQUIRE(dtype_size(dtype) > 0, "unknown dtype %d", dtype);
  if (a.tokens == 0) return NIE_OK;
  a.total_slots = num_blocks * a.bs;
  const int64_t codes = (int64_t)layer * a.total_slots * a.hkv * a.hd, scales = (int64_t)layer * num_blocks * a.hkv;
  a.codes[0] = (uint8_t*)key_codes + codes;
  a.codes[1] = (uint8_t*)value_codes + codes;
  a.scales[0] = key_scales + scales;
  a.scales[1] = value_scales + scales;
  switch (dtype) {
    case NIE_DTYPE_BF16: launch_append<__nv_bfloat16>(a, s); break;
    case NIE_DTYPE_F32: launch_append<float>(a, s); break;
    default: launch_append<__half>(a, s); break;
  }
  return check_launch("append_kv8_kernel");
}

}  // namespace nie

using namespace nie;

extern "C" int nie_rope_write_kv8(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                  int64_t v_stride, const void* sin, const void* cos, int64_t num_tokens,
                                  int32_t q_heads, int32_t kv_heads, int32_t head_dim, void* q_out, void* key_cache,
                                  void* value_cache, float* key_scales, float* value_scales, int32_t dtype,
                                  int32_t layer, int64_t num_layers, int64_t num_blocks, int32_t block_size,
                                  const int64_t* slot_mapping, int32_t* err_flag, void* stream) {
  NIE_REQUIRE(q && sin && cos && q_out, "null pointer argument");
  NIE_REQUIRE(q_heads > 0, "bad geometry");
  NIE_REQUIRE(head_dim > 0 && head_dim % 2 == 0, "head_dim must be even");
  AppendArgs a{};
  a.q = q, a.k = k, a.v = v;
  a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
  a.sin = sin, a.cos = cos;
  a.tokens = num_tokens;
  a.hq = q_heads, a.hkv = kv_heads, a.hd = head_dim, a.bs = block_size;
  a.q_out = q_out;
  a.slots = slot_mapping;
  a.err = err_flag;
  return append(a, key_cache, value_cache, key_scales, value_scales, dtype, layer, num_layers, num_blocks,
                reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int nie_write_kv8(const void* keys, int64_t k_stride, const void* values, int64_t v_stride,
                             int64_t num_tokens, void* key_cache, void* value_cache, float* key_scales,
                             float* value_scales, int32_t dtype, int32_t layer, int64_t num_layers, int64_t num_blocks,
                             int32_t block_size, int32_t kv_heads, int32_t head_dim, const int64_t* slot_mapping,
                             int32_t* err_flag, void* stream) {
  AppendArgs a{};
  a.k = keys, a.v = values;
  a.k_stride = k_stride, a.v_stride = v_stride;
  a.tokens = num_tokens;
  a.hkv = kv_heads, a.hd = head_dim, a.bs = block_size;
  a.slots = slot_mapping;
  a.err = err_flag;
  return append(a, key_cache, value_cache, key_scales, value_scales, dtype, layer, num_layers, num_blocks,
                reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int nie_gather_kv8(const void* key_cache, const void* value_cache, const float* key_scales,
                              const float* value_scales, int32_t layer, int64_t num_layers, int64_t num_blocks,
                              int32_t block_size, int32_t kv_heads, int32_t head_dim, const int32_t* block_table,
                              int64_t num_tokens, void* out_keys, void* out_values, int32_t out_dtype,
                              int32_t* err_flag, void* stream) {
  NIE_REQUIRE(layer >= 0 && layer < num_layers, "layer %d out of range", layer);
  NIE_REQUIRE(key_cache && value_cache && key_scales && value_scales && block_table && out_keys && out_values,
              "null pointer argument");
  NIE_REQUIRE(num_blocks > 0 && block_size > 0 && kv_heads > 0 && head_dim > 0, "bad cache geometry");
  NIE_REQUIRE(dtype_size(out_dtype) > 0, "unknown dtype %d", out_dtype);
  if (num_tokens <= 0) return NIE_OK;
  const int64_t codes = (int64_t)layer * num_blocks * block_size * kv_heads * head_dim;
  const int64_t scales = (int64_t)layer * num_blocks * kv_heads;
  const uint8_t* kc = (const uint8_t*)key_cache + codes;
  const uint8_t* vc = (const uint8_t*)value_cache + codes;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int64_t n = num_tokens * kv_heads * head_dim;
  const int64_t pieces = n / 16;
  if (head_dim % 16 == 0 && at16(kc) && at16(vc) && at16(out_keys) && at16(out_values) && pieces < (int64_t(1) << 38)) {
    const unsigned ctas = (unsigned)((pieces + 255) / 256);
    const float *sk = key_scales + scales, *sv = value_scales + scales;
    switch (out_dtype) {
      case NIE_DTYPE_BF16:
        gather_kv8_vec_kernel<<<ctas, 256, 0, s>>>(kc, vc, sk, sv, num_blocks, block_size, kv_heads, head_dim, block_table,
                                                   num_tokens, (__nv_bfloat16*)out_keys, (__nv_bfloat16*)out_values, err_flag);
        break;
      case NIE_DTYPE_F32:
        gather_kv8_vec_kernel<<<ctas, 256, 0, s>>>(kc, vc, sk, sv, num_blocks, block_size, kv_heads, head_dim, block_table,
                                                   num_tokens, (float*)out_keys, (float*)out_values, err_flag);
        break;
      default:
        gather_kv8_vec_kernel<<<ctas, 256, 0, s>>>(kc, vc, sk, sv, num_blocks, block_size, kv_heads, head_dim, block_table,
                                                   num_tokens, (__half*)out_keys, (__half*)out_values, err_flag);
        break;
    }
    return check_launch("gather_kv8_vec_kernel");
  }
  const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 148 * 32);
  switch (out_dtype) {
    case NIE_DTYPE_BF16:
      gather_kv8_kernel<<<grid, 256, 0, s>>>(kc, vc, key_scales + scales, value_scales + scales, num_blocks, block_size,
                                             kv_heads, head_dim, block_table, num_tokens, (__nv_bfloat16*)out_keys,
                                             (__nv_bfloat16*)out_values, err_flag);
      break;
    case NIE_DTYPE_F32:
      gather_kv8_kernel<<<grid, 256, 0, s>>>(kc, vc, key_scales + scales, value_scales + scales, num_blocks, block_size,
                                             kv_heads, head_dim, block_table, num_tokens, (float*)out_keys,
                                             (float*)out_values, err_flag);
      break;
    default:
      gather_kv8_kernel<<<grid, 256, 0, s>>>(kc, vc, key_scales + scales, value_scales + scales, num_blocks, block_size,
                                             kv_heads, head_dim, block_table, num_tokens, (__half*)out_keys,
                                             (__half*)out_values, err_flag);
      break;
  }
  return check_launch("gather_kv8_kernel");
}
