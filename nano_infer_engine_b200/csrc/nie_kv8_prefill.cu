// Ragged causal attention over the 8-bit paged cache on tcgen05 / TMEM, for
// bf16 / f16 queries, head_dim 64 or 128, blocks of a multiple of 16 tokens.
//
// What bounds it: a score costs 4 head_dim flops and one exp2; at 16 exp2 per
// clock and SM against 8192 flops of f16 MMA, head_dim 64 spends twice the MMA's
// time in exp2 and head_dim 128 the same.  So the MMAs run behind the softmax, and
// all else (loads, 8 bit to f16) is done by warps of its own.  Measured: 8192 tokens
// of one prompt, 32 heads on 8 of 64, bf16: 586 us, 470 TFLOP/s of causal work, of
// which exp2 alone is 240 us and the MMAs 185; 6 x 513 tokens behind up to 4000, 16
// on 4 of 128, f16: 87 us, 453 TFLOP/s.  What is left is the latency of a row's chain.
//
// Rows.  The query heads of a kv head share its codes, so the rows of a tile are
// (token, head of the group) pairs in that order, of one kv head, in MMA tiles of
// 128 ("parts"): four at head_dim 64, two at 128.  A "segment" is one such tile of
// a request and kv head against all keys that its last token sees.
//
// Split.  All segments lie end to end, each weighted as its key tiles plus a
// fixed part; every CTA takes an equal stretch.  A segment cut by a border leaves
// (max, sum, unnormalised output) of each part for a merging kernel; which parts
// and in which order follows from the lengths alone.
//
// Latency is what the chain of a row costs (S, its softmax, P V, the next S, each
// waiting for the one before), so several chains share an SM: four parts at
// head_dim 64; two at 128, where TMEM holds no more, with two S buffers each, so that
// the next tile's S is there when a softmax ends.
//
// Roles:
//   softmax   four warps a part: a thread owns a row, and brings its row of the
//             next segment's queries to shared memory under the last tile
//   issuers   a warp a part, of which one thread issues S = Q K^T and O += P V (P
//             from TMEM); an issuing thread is slow, some ten instructions to an MMA
//   loaders   four warps: codes to 16 bits (exact: K in the queries' type, V in
//             f16) into 128-byte swizzled shared memory; they come two tiles
//             ahead by cp.async into a thread's own bytes
//
// Softmax with scales as in the single-token kernel: y = S c + log2 vs per block
// of 16 keys, p = 2^(y - m) in f16 for the product (an error of 2^-12 of it), O = sum
// p vcode, l = sum p / vs from the unrounded p.  (A second product for what the rounding
// leaves would bring f16 outputs from 2.9e-4 to 2.1e-4 of 64 bits and bf16 ones nowhere, and
// take 13 % and 25 % more time in the two workloads above.)  m is raised (and O and l rescaled) only
// when a p would pass 2^15, which leaves the largest 2^9: weights (times vs) under 2^-23
// of the largest lose bits, those under 2^-34 are in l alone.
//
// TMEM columns: the parts' S buffers 0-255 (P takes the place of the scores it
// came from), their O 256-511.  Waits are bounded; one that runs out raises
// NIE_DEV_ERR_TIMEOUT and ends the CTA.
#include <algorithm>
#include <type_traits>

#include "nie_kv8_attn.cuh"

namespace nie {

constexpr int kF8MaxReq = 256;     // requests of one launch
constexpr int kF8MaxStages = 4;
constexpr uint32_t kF8OCol = 256;
// A segment's fixed part (its queries, its first and last waits, its output), in key tiles.  With 2, 5 and 10: 6 x
// 513 tokens behind up to 4000 take 93.7, 88.5 and 95.2 us, 8192 of one prompt 597, 589 and 602; less even loads
// differ: 513 tokens behind 487 35, 37 and 40, 16 x 128 behind 2872 133, 136 and 141, 90 x 65 behind 5 43, 48 and 43.
constexpr int kF8SegCost = 5;
constexpr uint32_t kF8Wait = 1u << 22;
constexpr float kF8Log2e = 1.4426950408889634f;
constexpr float kF8Most = 15.f, kF8Up = 9.f;  // log2 of p: its most, and that of the key that raised m

// What the merging kernel needs about the segment that begins in a CTA's
// stretch and goes on behind it (parts: CTAs after it that hold some of it).
struct F8Cut {
  int64_t row0;   // first row of the tile: (token, head) pairs of the request
  int64_t first;  // the request's first query row
  int32_t rows, kvh, parts, pad;
};

struct F8Plan {
  int num_req;
  float* partials;  // [2 * ctas][2 + hd][rows of a tile]: a CTA's first segment (cut in front), its last (cut behind)
  F8Cut* cuts;      // [ctas]
};

template <int HD>
struct F8Cfg {
  static constexpr int BN = 64;                           // keys of a tile
  static constexpr int Subs = BN / 16;
  static constexpr int Parts = HD == 64 ? 4 : 2;
  static constexpr int Rows = 128 * Parts;
  static constexpr int SBufs = HD == 64 ? 1 : 2;          // S buffers of a part
  static constexpr int Stages = HD == 64 ? 4 : 3;         // 16-bit key tiles in shared memory
  static constexpr int Loaders = 128;                     // threads
  static constexpr int IssueWarp = 4 * Parts, LoadWarp = 5 * Parts;
  static constexpr int Threads = LoadWarp * 32 + Loaders;
  static constexpr int PartBytes = 128 * HD * 2;          // queries of a part
  static constexpr int TileBytes = BN * HD * 2;           // K or V of a tile in 16 bits
  static constexpr int StageBytes = 2 * TileBytes;
  static constexpr int CodeBytes = 2 * BN * HD;           // codes of a tile
};

// A key tile of a segment: its first in this CTA, its last; the end of the stretch; above them the parts with rows.
enum F8Flag { kF8First = 1, kF8Last = 2, kF8End = 4, kF8PartShift = 4 };

struct F8Bars {
  uint64_t q_full[4];
  uint64_t kv_full[kF8MaxStages], kv_empty[kF8MaxStages];
  uint64_t s_full[4][2], p_full[4][2];   // of a part's S buffers
  uint64_t o_done[4];                    // a part's product is done
  uint64_t o_full[4], o_free[4];         // a segment's last one; its output has been read
  uint64_t done;
  uint32_t tmem_base;
  int abort;
  int nan_codes;                         // a NaN of V has been kept out of a product
  int4 row_of[16];                       // of a softmax warp's segment: its table row, kv head, first key of a NaN search
  int start_req, start_tile, start_head;
  int64_t start_pos;
  int flags[kF8MaxStages];                  // of a stage's tile: kF8First, ...
  float4 info[kF8MaxStages][4];             // of 16 keys: score factor, log2 vs, 1 / vs
  int64_t cum[kF8MaxReq + 1];            // cost before each request
};

__device__ __forceinline__ bool f8_wait(F8Bars* b, uint64_t* bar, uint32_t parity, int32_t* err) {
  for (uint32_t i = 0; i < kF8Wait; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 1023u) == 1023u && *reinterpret_cast<volatile int*>(&b->abort)) return false;
  }
  *reinterpret_cast<volatile int*>(&b->abort) = 1;
  raise_flag(err, NIE_DEV_ERR_TIMEOUT);
  return false;
}

// The same out of line, for a wait outside the loops: their code fills the instruction caches as it is.
__device__ __noinline__ bool f8_wait_call(F8Bars* b, uint64_t* bar, uint32_t parity, int32_t* err) {
  return f8_wait(b, bar, parity, err);
}

// The same for warps that run ahead: they sleep between probes, since every probe
// goes through the queue that the exponentials of the softmax warps use.
__device__ __forceinline__ bool f8_wait_idle(F8Bars* b, uint64_t* bar, uint32_t parity, int32_t* err) {
  for (uint32_t i = 0; i < kF8Wait; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    __nanosleep(100);
    if ((i & 1023u) == 1023u && *reinterpret_cast<volatile int*>(&b->abort)) return false;
  }
  *reinterpret_cast<volatile int*>(&b->abort) = 1;
  raise_flag(err, NIE_DEV_ERR_TIMEOUT);
  return false;
}

__device__ __forceinline__ float f8_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ void f8_fma2(float& d0, float& d1, float a0, float a1, float b, float c) {
  asm("{\n.reg .b64 ra, rb, rc, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %4};\nmov.b64 rc, {%5, %5};\n"
      "fma.rn.f32x2 rd, ra, rb, rc;\nmov.b64 {%0, %1}, rd;\n}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void f8_add2(float& d0, float& d1, float b0, float b1) {
  asm("{\n.reg .b64 ra, rb, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %5};\n"
      "add.rn.f32x2 rd, ra, rb;\nmov.b64 {%0, %1}, rd;\n}"
      : "=f"(d0), "=f"(d1)
      : "f"(d0), "f"(d1), "f"(b0), "f"(b1));
}

// kind::f16 with f16 (or bf16) A and B, f32 D.
constexpr uint32_t f8_idesc(int m, int n, bool b_mn_major, bool bf16) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// A request of the call; none of its fields depend on the kv head.
struct F8Req {
  int first;  // first query row
  int rows;   // query tokens * heads of a group
  int ctx;    // keys before its first token (negative: the first tokens see none)
  int n;      // keys
  int trow;
};

__device__ __noinline__ F8Req f8_request(const Kv8Args& a, int i, int32_t* err) {
  F8Req x{};
  const int r = a.req_list ? a.req_list[i] : i;
  const int tr = r < 0 || r >= a.num_seqs ? -1 : a.table_rows ? a.table_rows[r] : r;
  if (tr < 0 || tr >= a.num_table_rows) {
    raise_flag(err, NIE_DEV_ERR_CAPACITY);
    return x;
  }
  const Kv8Rows rows = kv8_rows(a, r, err);
  if (rows.count <= 0) return x;
  x.first = (int)rows.first;
  x.rows = (int)rows.count * a.group;
  x.ctx = (int)rows.keys;
  // keys past the end of the table have no block
  const int64_t most = min(a.twidth * a.bs, (int64_t)1 << 30), n = max(a.seq_lens[r], 0);
  if (n > most) raise_flag(err, NIE_DEV_ERR_BLOCK_RANGE);
  x.n = (int)min(n, most);
  x.trow = tr;
  return x;
}

// Tiles of a request; keys that the last token of a tile sees, and the tiles of BN
// keys they fill (at least one: rows that see no key still get their zeros from a
// masked tile).
template <class C>
__device__ __forceinline__ int f8_tiles(const F8Req& x) {
  return (x.rows + C::Rows - 1) / C::Rows;
}
template <class C>
__device__ __forceinline__ int f8_keys(const F8Req& x, int group, int tile) {
  return min(x.n, max(0, x.ctx + (min(x.rows, (tile + 1) * C::Rows) - 1) / group + 1));
}
template <class C>
__device__ __forceinline__ int f8_key_tiles(int keys) {
  return max(1, (keys + C::BN - 1) / C::BN);
}

// Walks the segments of a CTA's stretch: requests, tiles, kv heads.  Positions
// are costs from the stretch's beginning; it ends at `hi`.
template <class C>
struct F8Walk {
  int hi, start;  // start: position of the segment's first key tile (may be negative)
  int i, tile, h, keys, n;
  F8Req x;

  __device__ __forceinline__ void load(const Kv8Args& a) {
    keys = f8_keys<C>(x, a.group, tile);
    n = f8_key_tiles<C>(keys);
  }
  __device__ __forceinline__ void init(const Kv8Args& a, const F8Bars* b, int64_t lo, int64_t end) {
    hi = (int)(end - lo);
    i = b->start_req;
    tile = b->start_tile;
    h = b->start_head;
    x = f8_request(a, i, nullptr);
    load(a);
    start = (int)(b->start_pos - lo) + kF8SegCost;
  }
  __device__ __forceinline__ bool valid() const { return start < hi; }
  __device__ __forceinline__ int t_lo() const { return max(0, -start); }
  __device__ __forceinline__ int t_hi() const { return min(hi - start, n); }
  __device__ __forceinline__ int rows() const { return min(C::Rows, x.rows - tile * C::Rows); }
  __device__ __forceinline__ void next(const Kv8Args& a, int num_req) {
    start += n;
    if (++h == a.hkv) {
      h = 0;
      if (++tile >= f8_tiles<C>(x)) {
        tile = 0;
        do {
          if (++i >= num_req) {
            start = hi;
            return;
          }
          x = f8_request(a, i, nullptr);
        } while (x.rows == 0);
      }
      load(a);
    }
    start += kF8SegCost;
  }
};

// D[tmem] (+)= A[smem] * B[smem] and A[tmem] * B[smem], kind::f16.  Only the low words
// of the operands' descriptors differ: 128-byte swizzle, 1024 bytes between groups of 8 rows.
constexpr uint32_t kF8DescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void f8_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 da, db;\nmov.b64 da, {%1, %5};\nmov.b64 db, {%2, %5};\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "n"(kF8DescHi)
      : "memory");
}
__device__ __forceinline__ void f8_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 db;\nmov.b64 db, {%2, %5};\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "n"(kF8DescHi)
      : "memory");
}
__device__ __forceinline__ uint32_t f8_desc(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | ((lbo >> 4) << 16); }

// First tile of a segment that some row does not see all of.  There the loaders put
// zeros for NaN codes of V: 0 * NaN would reach the rows that do not see the key.
template <class C>
__device__ __forceinline__ int f8_masked_from(const Kv8Args& a, const F8Walk<C>& s) {
  return max(0, s.x.ctx + s.tile * C::Rows / a.group + 1) / C::BN;
}

// The NaN that were left out, for one row that sees the keys [from, to): out + d * step gets one for
// each dimension d in which one of them has it.
template <typename T>
__device__ __noinline__ void f8_put_nan(const Kv8Args& a, int trow, int h, int from, int to, T* out, int step) {
  for (int key = from; key < to; ++key) {
    const int lb = key / a.bs;
    const int64_t block = lb < a.twidth ? (int64_t)a.tables[(int64_t)trow * a.tstride + lb] : -1;
    if (block < 0 || block >= a.nb) continue;
    const uint8_t* codes = a.vc + ((block * a.bs + key % a.bs) * a.hkv + h) * a.hd;
    for (int d = 0; d < a.hd; ++d)
      if ((codes[d] & 0x7f) == 0x7f) out[(int64_t)d * step] = Num<T>::from_f(__int_as_float(0x7fffffff));
  }
}

template <int HD, typename T>
__global__ void __launch_bounds__(F8Cfg<HD>::Threads, 1)
    kv8_prefill_kernel(const __grid_constant__ Kv8Args a, const __grid_constant__ F8Plan p) {
  using C = F8Cfg<HD>;
  constexpr int BN = C::BN;
  extern __shared__ uint8_t f8_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(f8_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = sm;
  uint8_t* skv = sq + C::Parts * C::PartBytes;
  uint8_t* scode = skv + C::Stages * C::StageBytes;
  F8Bars* b = reinterpret_cast<F8Bars*>(scode + 2 * C::CodeBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = p.num_req;

  pdl_wait();
  pdl_trigger();
  // ---- cost of each request (a warp each), then of all before it
  for (int i = warp; i < R; i += C::Threads / 32) {
    const F8Req x = f8_request(a, i, blockIdx.x == 0 && lane == 0 ? a.err : nullptr);
    int64_t cost = 0;
    for (int tile = lane; tile < f8_tiles<C>(x); tile += 32) cost += f8_key_tiles<C>(f8_keys<C>(x, a.group, tile)) + kF8SegCost;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) cost += __shfl_xor_sync(0xffffffffu, cost, o);
    if (lane == 0) b->cum[i + 1] = cost * a.hkv;
  }
  if (threadIdx.x == 0) {
    b->cum[0] = 0;
    for (int i = 0; i < C::Parts; ++i) {
      mbar_init(&b->q_full[i], 4);
      for (int u = 0; u < 2; ++u) {
        mbar_init(&b->s_full[i][u], 1);
        mbar_init(&b->p_full[i][u], 4);
      }
      mbar_init(&b->o_done[i], 1);
      mbar_init(&b->o_full[i], 1);
      mbar_init(&b->o_free[i], 4);
    }
    for (int s = 0; s < C::Stages; ++s) {
      mbar_init(&b->kv_full[s], C::Loaders);
      mbar_init(&b->kv_empty[s], C::Parts);
    }
    mbar_init(&b->done, C::Parts);
    b->abort = 0;
    b->nan_codes = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (warp == 0) {
    // prefix sums by one warp, 32 requests at a time
    int64_t before = 0;
    for (int i0 = 0; i0 < R; i0 += 32) {
      int64_t v = i0 + lane < R ? b->cum[i0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
      }
      v += before;
      if (i0 + lane < R) b->cum[i0 + lane + 1] = v;
      before = __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const int64_t total = b->cum[R];
  const int64_t W = (total + gridDim.x - 1) / gridDim.x;
  const int64_t lo = min((int64_t)blockIdx.x * W, total), hi = min(total, lo + W);
  if (threadIdx.x == 0) p.cuts[blockIdx.x].parts = 0;
  if (lo >= hi) return;  // the whole CTA: nothing left for it
  if (warp == 0) {
    // the segment that holds position lo
    int l = 0, r = R;  // cum[l] <= lo < cum[r]
    while (r - l > 1) {
      const int mid = (l + r) >> 1;
      if (b->cum[mid] <= lo) l = mid; else r = mid;
    }
    const F8Req x = f8_request(a, l, nullptr);
    int64_t pos = b->cum[l];
    const int tiles = f8_tiles<C>(x);
    for (int t0 = 0; t0 < tiles; t0 += 32) {
      const int64_t c = t0 + lane < tiles ? f8_key_tiles<C>(f8_keys<C>(x, a.group, t0 + lane)) + kF8SegCost : 0;
      int64_t v = c * a.hkv;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
      }
      const int64_t end = pos + v, begin = end - c * a.hkv;
      if (begin <= lo && lo < end) {  // one lane of one round
        b->start_req = l;
        b->start_tile = t0 + lane;
        b->start_head = (int)((lo - begin) / c);
        b->start_pos = begin + (int64_t)b->start_head * c;
      }
      pos = __shfl_sync(0xffffffffu, end, 31);
      if (lo < pos) break;
    }
  }
  if (warp == C::IssueWarp) {
    tmem_alloc(&b->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = b->tmem_base;
  F8Walk<C> seg;
  seg.init(a, b, lo, hi);

  if (warp >= C::LoadWarp) {
    // ------------------------------------------------------------ loaders
    const int tid = threadIdx.x - C::LoadWarp * 32;
    constexpr int Pass = C::Loaders / 4, Passes = BN / Pass;  // rows of a copy, copies for 64 dims of all rows
    constexpr int Copies = Passes * HD / 64;                  // of K, and of V
    const int64_t row_bytes = (int64_t)a.hkv * HD;
    const float coef = fabsf(a.scale) * kF8Log2e;
    const uint32_t flip = a.scale < 0.f ? 0x80808080u : 0u;  // a negative scale's sign goes to the keys
    // tiles come two ahead: `ahead` walks in front of `seg`
    F8Walk<C> ahead = seg;
    int a_kt = ahead.valid() ? ahead.t_lo() : 0;
    // Lane s of each warp looks up the block of the tile's s-th 16 keys, a tile
    // before its codes are fetched; all rows of a warp's copy j lie in 16 keys.
    int entry = -1, offset = 0, count = 0;  // count: keys of the 16 that are there
    auto look_up = [&]() {
      count = 0;
      if (ahead.valid()) {
        const int key = a_kt * BN + 16 * lane;
        if (lane < C::Subs) count = min(16, min(ahead.keys, ahead.x.n) - key);
        const int lb = key / a.bs;
        offset = key - lb * a.bs;
        entry = count > 0 && lb < a.twidth ? a.tables[(int64_t)ahead.x.trow * a.tstride + lb] : -1;
      }
    };
    // scales of the next tile and of the one after it (first warp, lane s: the s-th 16 keys)
    float ks0 = 0.f, vs0 = 1.f, ks1 = 0.f, vs1 = 1.f;
    bool ok0 = false, ok1 = false;
    auto fetch = [&](int slot, float& p_ks, float& p_vs, bool& p_ok) {
      if (ahead.valid()) {
        const uint32_t base = smem_u32(scode + slot * C::CodeBytes) + tid * 16;
        const bool found = count > 0 && entry >= 0 && entry < a.nb;
        if (count > 0 && !found) raise_flag(a.err, NIE_DEV_ERR_BLOCK_RANGE);
        const int at = entry * a.bs + offset, here = found ? count : 0;
        if (tid < C::Subs) {
          p_ok = found;
          if (found) {
            p_ks = a.ks[(int64_t)entry * a.hkv + ahead.h];
            p_vs = a.vs[(int64_t)entry * a.hkv + ahead.h];
          }
        }
#pragma unroll
        for (int j = 0; j < Copies; ++j) {
          const int half = j / Passes;
          const int s = ((tid >> 2) + Pass * (j % Passes)) >> 4, row = (tid >> 2) & 15;  // all of a warp's rows lie in 16 keys
          const int from = __shfl_sync(0xffffffffu, at, s);
          const bool there = row < __shfl_sync(0xffffffffu, here, s);
          const int64_t off =
              there ? (int64_t)(from + row) * row_bytes + (int64_t)ahead.h * HD + half * 64 + (tid & 3) * 16 : 0;
          cp_async16(base + j * (C::Loaders * 16), a.kc + off, there ? 16 : 0);
          cp_async16(base + (Copies + j) * (C::Loaders * 16), a.vc + off, there ? 16 : 0);
        }
        if (++a_kt >= ahead.t_hi()) {
          ahead.next(a, R);
          a_kt = 0;
        }
        look_up();
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look_up();
    fetch(0, ks0, vs0, ok0);
    fetch(1, ks1, vs1, ok1);
    bool ok = true;
    int st = 0, slot = 0;
    uint32_t par = 1;  // parity of the stage's last release; the first round finds the stages free
    for (; ok && seg.valid(); seg.next(a, R)) {
      const int rows = seg.rows();
      const int thi = seg.t_hi(), masked = f8_masked_from(a, seg);
      for (int kt = seg.t_lo(); kt < thi; ++kt) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        if (!f8_wait_idle(b, &b->kv_empty[st], par, a.err)) {
          ok = false;
          break;
        }
        uint8_t* dst = skv + st * C::StageBytes;
        const uint8_t* src = scode + slot * C::CodeBytes + tid * 16;
#pragma unroll
        for (int j = 0; j < 2 * Copies; ++j) {
          const int jj = j % Copies;
          const int row = (tid >> 2) + Pass * (jj % Passes), half = jj / Passes;
          const uint4 x = *reinterpret_cast<const uint4*>(src + j * (C::Loaders * 16));
          uint32_t w[4] = {x.x, x.y, x.z, x.w}, h[8];
          if (j >= Copies && kt >= masked) {
            uint32_t any = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t nan = __vcmpeq4(w[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              w[e] &= ~nan;
              any |= nan;
            }
            if (any) *reinterpret_cast<volatile int*>(&b->nan_codes) = 1;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (j < Copies) w[e] ^= flip;
            h[2 * e] = e4m3x2_to_f16x2((uint16_t)(w[e] & 0xffffu));
            h[2 * e + 1] = e4m3x2_to_f16x2((uint16_t)(w[e] >> 16));
          }
          if (j < Copies && !std::is_same<T, __half>::value) {  // keys meet bf16 queries: 4 bits fit either type
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 f = f16x2_to_float2(h[e]);
              h[e] = pack_bf16x2(f.x, f.y);
            }
          }
          uint8_t* at = dst + j / Copies * C::TileBytes + half * (BN * 128) + row * 128;
          const int ch = 2 * (tid & 3);
          *reinterpret_cast<uint4*>(at + ((ch ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(at + (((ch + 1) ^ (row & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
        }
        if (tid < C::Subs)  // keys without a block have no weight
          {
          const float vs = fminf(fmaxf(vs0, kScaleMin), kScaleMax);
          b->info[st][tid] = ok0 ? make_float4(fminf(fmaxf(ks0, 0.f), kScaleMax) * coef, __log2f(vs), 1.f / vs, 0.f)
                                 : make_float4(0.f, -INFINITY, 0.f, 0.f);
        }
        if (tid == 0)
          b->flags[st] = (kt == seg.t_lo() ? kF8First : 0) | (kt + 1 == thi ? kF8Last : 0) | ((rows + 127) / 128) << kF8PartShift;
        fence_proxy_async_smem();
        mbar_arrive(&b->kv_full[st]);
        ks0 = ks1, vs0 = vs1, ok0 = ok1;
        fetch(slot, ks1, vs1, ok1);
        slot ^= 1;
        if (++st == C::Stages) {
          st = 0;
          par ^= 1u;
        }
      }
    }
    {  // the end, in place of a tile
      if (ok && f8_wait_idle(b, &b->kv_empty[st], par, a.err)) {
        if (tid == 0) b->flags[st] = kF8End;
        mbar_arrive(&b->kv_full[st]);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= C::IssueWarp) {
    // -------------------------------------------------------- MMA issuers
    // One thread for each part.  What it has to know of a key tile stands beside the tile.
    if (lane == 0) {
      const int x = warp - C::IssueWarp;
      const uint32_t q_desc = f8_desc(smem_u32(sq) + x * C::PartBytes, 16);
      const uint32_t k_desc = f8_desc(smem_u32(skv), 16), v_desc = f8_desc(smem_u32(skv + C::TileBytes), BN * 128);
      const uint32_t s_col = tbase + x * (BN * C::SBufs), o_col = tbase + kF8OCol + x * HD;
      constexpr uint32_t id_s = f8_idesc(128, BN, false, !std::is_same<T, __half>::value);
      constexpr uint32_t id_o = f8_idesc(128, HD, true, false);
      int flags = 0, st = 0;     // of the tile whose scores come next
      uint32_t par = 0;          // phase parity of its stage
      int tiles = 0, done = 0;   // of this part: scores and products issued
      int segs = 0, outs = 0;    // segments begun, their outputs begun
      int f0 = 0, f1 = 0, st0 = 0, st1 = 0;  // the tiles between scores and product: the older, the younger
      bool ok = true;
      auto step = [&]() {
        if (++st == C::Stages) {
          st = 0;
          par ^= 1u;
        }
      };
      auto take = [&]() {  // the next tile's flags
        ok = f8_wait(b, &b->kv_full[st], par, a.err);
        flags = ok ? *reinterpret_cast<volatile int*>(&b->flags[st]) : kF8End;
      };
      take();
      while (ok) {
        const int open = tiles - done;
        const bool mine = (flags >> kF8PartShift) > x;
        if (open == 0 && !mine && !(flags & kF8End)) {
          // a tile without rows of this part: passed over, but not before the products are issued that
          // keep stages from the loaders
          mbar_arrive(&b->kv_empty[st]);
          step();
          take();
          continue;
        }
        // S = Q K^T, as far ahead of the products as there are buffers; over a P whose product has been
        // issued: MMAs run in order.  A segment's first tile waits for the
        // products of the one before (its queries come under their softmax).
        if (mine && !(flags & kF8End) && open < C::SBufs && !((flags & kF8First) && open > 0)) {
          if (flags & kF8First) {
            ok = f8_wait(b, &b->q_full[x], (uint32_t)segs & 1u, a.err);
            if (!ok) break;
            ++segs;
          }
          tc_fence_after();
          const uint32_t kd = k_desc + (uint32_t)(st * (C::StageBytes / 16)), d = s_col + tiles % C::SBufs * BN;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            f8_mma_ss(d, q_desc + ((kk >> 2) * (128 * 128 / 16) + (kk & 3) * 2),
                      kd + ((kk >> 2) * (BN * 128 / 16) + (kk & 3) * 2), id_s, kk > 0);
          tc_commit(&b->s_full[x][tiles % C::SBufs]);
          f0 = f1, st0 = st1;
          f1 = flags, st1 = st;
          ++tiles;
          step();
          take();
          continue;
        }
        if (open == 0) break;
        // O += P V of the oldest
        const int f = open == 2 ? f0 : f1, s = open == 2 ? st0 : st1;
        ok = f8_wait(b, &b->p_full[x][done % C::SBufs], (uint32_t)(done / C::SBufs) & 1u, a.err);
        if (ok && (f & kF8First)) {
          // the softmax warps have read the output of the segment before
          if (outs > 0) ok = f8_wait(b, &b->o_free[x], (uint32_t)(outs - 1) & 1u, a.err);
          ++outs;
        }
        if (!ok) break;
        tc_fence_after();
        const uint32_t vd = v_desc + (uint32_t)(s * (C::StageBytes / 16)), pc = s_col + done % C::SBufs * BN;
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          f8_mma_ts(o_col, pc + kk * 8, vd + kk * (2048 / 16), id_o, kk > 0 || !(f & kF8First));
        tc_commit(&b->kv_empty[s]);
        tc_commit(&b->o_done[x]);
        if (f & kF8Last) tc_commit(&b->o_full[x]);
        ++done;
      }
      tc_commit(&b->done);
      mbar_wait_bounded(&b->done, 0, kF8Wait);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------ softmax warps
    const int x = warp >> 2;                       // part
    const int t = (warp & 3) * 32 + lane;          // row of the part, TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_base = tbase + lane_off + x * (BN * C::SBufs), o_addr = tbase + lane_off + kF8OCol + x * HD;
    bool ok = true;
    int st = 0;             // stage of the key tile
    uint32_t kv_par = 0;    // and its phase parity
    int used = 0, segs = 0;
    // this thread's row of a segment's queries; zeros where there is none
    auto load_queries = [&]() {
      const int row = x * 128 + t, rows = seg.valid() ? seg.rows() : 0;
      if (rows <= x * 128) return;
      const int fr = seg.tile * C::Rows + row;
      const bool there = row < rows;
      const T* q = reinterpret_cast<const T*>(a.q);
      if (there) q += (int64_t)(seg.x.first + fr / a.group) * a.q_stride + (int64_t)(seg.h * a.group + fr % a.group) * HD;
      const uint32_t dst = smem_u32(sq) + x * C::PartBytes + t * 128;
#pragma unroll
      for (int c = 0; c < HD / 8; ++c)
        cp_async16(dst + (c >> 3) * (128 * 128) + (((c & 7) ^ (t & 7)) << 4), q + c * 8, there ? 16 : 0);
    };
    auto queries_there = [&]() {
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b->q_full[x]);
    };
    load_queries();
    if (seg.valid() && seg.rows() > x * 128) queries_there();
    while (ok && seg.valid()) {
      const int rows = seg.rows();
      const int tlo = seg.t_lo(), thi = seg.t_hi();
      if (rows <= x * 128) {  // the part has no rows
        for (int kt = tlo; kt < thi; ++kt)
          if (++st == C::Stages) {
            st = 0;
            kv_par ^= 1u;
          }
        seg.next(a, R);
        load_queries();
        if (seg.valid() && seg.rows() > x * 128) queries_there();
        continue;
      }
      const bool active = x * 128 + (warp & 3) * 32 < rows;  // this warp has rows
      const int fr = seg.tile * C::Rows + x * 128 + t;
      const int qpos = seg.x.ctx + fr / a.group;              // position of the row's token
      const int first_pos = seg.x.ctx + (fr - lane) / a.group;  // of the warp's first row
      const bool whole = tlo == 0 && thi == seg.n;
      T* op = reinterpret_cast<T*>(a.out) + (int64_t)(seg.x.first + fr / a.group) * a.out_stride +
              (int64_t)(seg.h * a.group + fr % a.group) * HD;
      if (tlo == 0 && !whole && threadIdx.x == 0)
        p.cuts[blockIdx.x] = F8Cut{(int64_t)seg.tile * C::Rows, seg.x.first, rows, seg.h,
                                   (int)((lo + seg.start + seg.n - 1) / W - blockIdx.x), 0};
      if (lane == 0) b->row_of[warp] = make_int4(seg.x.trow, seg.h, max(tlo, f8_masked_from(a, seg)) * BN, seg.x.n);
      float m_ref = -INFINITY, l = 0.f;
      // One key tile of the row; MASK: some row of the warp does not see all of it.
      auto softmax_tile = [&](int kt, auto masked) -> bool {
        constexpr bool MASK = decltype(masked)::value;
        const float4* info = b->info[st];
        const uint32_t s_addr = s_base + used % C::SBufs * BN;
        const int seen = min(BN, max(0, qpos - kt * BN + 1));  // keys of the tile that the row sees
        // Loops of 32 keys that stay loops: unrolled, the roles' code outgrows the instruction caches.
        uint32_t v[32];
        // largest y: per 16 keys the largest score, since their factor is not negative
        float mx = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          tmem_ld32(s_addr + 32 * c, v);
          const float4 f0 = info[2 * c], f1 = info[2 * c + 1];
          tmem_wait_ld();
          if constexpr (MASK) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * c + e >= seen) v[e] = 0xff800000u;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float* s = reinterpret_cast<const float*>(&v[16 * h]);
            const float s0 = f8_max3(f8_max3(s[0], s[1], s[2]), f8_max3(s[3], s[4], s[5]), f8_max3(s[6], s[7], s[8]));
            const float s1 = f8_max3(f8_max3(s[9], s[10], s[11]), f8_max3(s[12], s[13], s[14]), s[15]);
            mx = fmaxf(mx, fmaf(fmaxf(s0, s1), h ? f1.x : f0.x, h ? f1.y : f0.y));
          }
        }
        const bool raise = mx > m_ref + kF8Most;
        if (__any_sync(0xffffffffu, raise)) {
          const float to = mx - kF8Up;
          const float keep = raise ? (m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - to)) : 1.f;
          if (raise) {
            l *= keep;
            m_ref = to;
          }
          if (kt > tlo) {
            // O must hold the product of the tile before.  These scores were issued after the product of
            // the tile before that at least, so o_done has one phase to go at most: its parity is no riddle.
            if (!__all_sync(0xffffffffu, f8_wait(b, &b->o_done[x], (uint32_t)(used - 1) & 1u, a.err))) return false;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              tmem_ld32(o_addr + 32 * c, v);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * keep);
              tmem_st32(o_addr + 32 * c, v);
            }
          }
        }
        const float ref = m_ref == -INFINITY ? 0.f : m_ref;
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          tmem_ld32(s_addr + 32 * c, v);
          const float4 f0 = info[2 * c], f1 = info[2 * c + 1];
          tmem_wait_ld();
          uint32_t pk[16];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float fc = h ? f1.x : f0.x, fb = (h ? f1.y : f0.y) - ref;
            float r0 = 0.f, r1 = 0.f;
#pragma unroll
            for (int e = 16 * h; e < 16 * h + 16; e += 2) {
              float y0, y1;
              f8_fma2(y0, y1, __uint_as_float(v[e]), __uint_as_float(v[e + 1]), fc, fb);
              if constexpr (MASK) {
                if (32 * c + e >= seen) y0 = -INFINITY;
                if (32 * c + e + 1 >= seen) y1 = -INFINITY;
              }
              const float p0 = fast_exp2(y0), p1 = fast_exp2(y1);
              f8_add2(r0, r1, p0, p1);
              pk[e / 2] = pack_f16x2(p0, p1);
            }
            l = fmaf(r0 + r1, h ? f1.z : f0.z, l);
          }
          tmem_st16(s_addr + 16 * c, pk);  // over scores that were taken
        }
        tmem_wait_st();
        return true;
      };
      // Before a segment's first tile, its scores.  A part without rows passes tiles over without a wait, and its warps
      // may be two of a stage's phases ahead here, where kv_full's parity would take the older phase for theirs.
      // Behind s_full the tile's phase is over, and the next one waits for this warp's weights; the stages after it
      // are one phase behind at most, since the loaders fill them in turn.
      if (!f8_wait_call(b, &b->s_full[x][used % C::SBufs], (uint32_t)(used / C::SBufs) & 1u, a.err)) break;
      for (int kt = tlo; kt < thi; ++kt, ++used) {
        // the loaders' factors are there before the scores: waited for while there is time
        if (!f8_wait(b, &b->kv_full[st], kv_par, a.err) ||
            !f8_wait(b, &b->s_full[x][used % C::SBufs], (uint32_t)(used / C::SBufs) & 1u, a.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (kt + 1 == thi) {  // the segment's queries are done with: the next one's, under this tile
          seg.next(a, R);
          load_queries();
        }
        if (active) {
          if (kt * BN + BN - 1 > first_pos) ok = softmax_tile(kt, std::true_type{});
          else ok = softmax_tile(kt, std::false_type{});
          if (!ok) break;  // of one mind: the warp voted
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b->p_full[x][used % C::SBufs]);
        if (++st == C::Stages) {
          st = 0;
          kv_par ^= 1u;
        }
      }
      if (!ok) break;
      if (seg.valid() && seg.rows() > x * 128) queries_there();
      if (!f8_wait(b, &b->o_full[x], (uint32_t)(segs & 1), a.err)) break;
      ++segs;
      tc_fence_after();
      const int row = x * 128 + t;
      float* ps = p.partials + (int64_t)(2 * blockIdx.x + (tlo == 0)) * (HD + 2) * C::Rows + row;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (active) {
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + 32 * c, o);
          tmem_wait_ld();
          if (row < rows) {
            if (whole) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                T w[8];
#pragma unroll
                for (int d = 0; d < 8; ++d) w[d] = Num<T>::from_f(__uint_as_float(o[e + d]) * inv);
                *reinterpret_cast<uint4*>(op + 32 * c + e) = *reinterpret_cast<const uint4*>(w);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) ps[(2 + 32 * c + e) * C::Rows] = __uint_as_float(o[e]);
            }
          }
        }
        if (!whole && row < rows) {
          ps[0] = m_ref;
          ps[C::Rows] = l;
        }
        if (row < rows && *reinterpret_cast<volatile int*>(&b->nan_codes)) {  // known since the tile's kv_full
          const int4 of = b->row_of[warp];
          const int to = min(min(qpos + 1, thi * BN), of.w);
          if (whole) f8_put_nan(a, of.x, of.y, of.z, to, op, 1);
          else f8_put_nan(a, of.x, of.y, of.z, to, ps + 2 * C::Rows, C::Rows);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b->o_free[x]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::IssueWarp) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// Segments cut by borders: CTA (c, y) merges 32 rows of the one that begins in
// the first kernel's CTA c, its parts in order.  A thread: one row, every 8th dim, as
// the partials lie; the rows are turned in shared memory and leave in 16-byte pieces
// (stored value by value from there, 148 cuts of 256 rows of 128 took 41 us).
template <int HD, typename T>
__global__ void __launch_bounds__(256) kv8_prefill_merge_kernel(const __grid_constant__ Kv8Args a,
                                                                 const __grid_constant__ F8Plan p) {
  __shared__ float so[32][HD + 1];
  pdl_wait();
  const F8Cut cut = p.cuts[blockIdx.x];
  const int row0 = blockIdx.y * 32, lane = threadIdx.x & 31, d0 = threadIdx.x >> 5;
  if (cut.parts == 0 || row0 >= cut.rows) return;
  using C = F8Cfg<HD>;
  const int64_t size = (int64_t)(HD + 2) * C::Rows;
  if (row0 + lane < cut.rows) {
    // part 0 is the CTA's last segment, the others the first one of the CTAs behind it
    auto part = [&](int k) { return p.partials + (2 * (int64_t)(blockIdx.x + k) + (k == 0)) * size + row0 + lane; };
    float M = -INFINITY;
    for (int k = 0; k <= cut.parts; ++k) M = fmaxf(M, part(k)[0]);
    float L = 0.f, O[HD / 8];
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) O[d] = 0.f;
    for (int k = 0; k <= cut.parts; ++k) {
      const float* ps = part(k);
      const float f = ps[0] == -INFINITY ? 0.f : fast_exp2(ps[0] - M);
      L += ps[C::Rows] * f;
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) O[d] = fmaf(ps[(2 + d0 + 8 * d) * C::Rows], f, O[d]);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) so[lane][d0 + 8 * d] = O[d] * inv;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < min(32, cut.rows - row0) * (HD / 8); x += 256) {
    const int r = x / (HD / 8), d = x % (HD / 8) * 8;
    T w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = Num<T>::from_f(so[r][d + e]);
    const int64_t fr = cut.row0 + row0 + r;
    T* op = reinterpret_cast<T*>(a.out) + (cut.first + fr / a.group) * a.out_stride +
            (int64_t)(cut.kvh * a.group + fr % a.group) * HD + d;
    *reinterpret_cast<uint4*>(op) = *reinterpret_cast<const uint4*>(w);
  }
}

static size_t f8_cut_bytes(int ctas) { return ((size_t)ctas * sizeof(F8Cut) + 255) & ~size_t(255); }

size_t kv8_prefill_workspace(int sms, int head_dim) {
  const int rows = head_dim == 64 ? F8Cfg<64>::Rows : F8Cfg<128>::Rows;
  return f8_cut_bytes(sms) + (size_t)2 * sms * (head_dim + 2) * rows * sizeof(float);
}

bool kv8_prefill_takes(int dtype, const Kv8Args& a) {
  auto aligned = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  return (dtype == NIE_DTYPE_BF16 || dtype == NIE_DTYPE_F16) && (a.hd == 64 || a.hd == 128) && a.bs % 16 == 0 &&
         aligned(a.kc, 16) && aligned(a.vc, 16) && aligned(a.q, 16) && aligned(a.out, 16) && a.q_stride % 8 == 0 &&
         a.out_stride % 8 == 0 && a.nb * a.bs < (int64_t(1) << 31) && a.num_q_rows * a.group < (int64_t(1) << 31);
}

template <int HD, typename T>
static int launch_prefill(const Kv8Args& a, const F8Plan& p, int sms, cudaStream_t s) {
  using C = F8Cfg<HD>;
  const size_t smem = 1024 + (size_t)C::Parts * C::PartBytes + (size_t)C::Stages * C::StageBytes + 2 * C::CodeBytes + sizeof(F8Bars);
  auto* kernel = kv8_prefill_kernel<HD, T>;
  const int rc = opt_in_smem(kSmemKv8Prefill + (HD == 128) * 2 + std::is_same<T, __half>::value, (const void*)kernel, smem);
  if (rc != NIE_OK) return rc;
  kv8_launches() += 2;
  kernel<<<sms, C::Threads, smem, s>>>(a, p);
  const int st = check_launch("kv8_prefill_kernel");
  if (st != NIE_OK) return st;
  pdl_launch(kv8_prefill_merge_kernel<HD, T>, dim3((unsigned)sms, C::Rows / 32), dim3(256), s, a, p);
  return check_launch("kv8_prefill_merge_kernel");
}

int launch_kv8_prefill(int dtype, const Kv8Args& args, int num_requests, int sms, void* workspace, cudaStream_t s) {
  Kv8Args a = args;
  for (int at = 0; at < num_requests; at += kF8MaxReq) {
    F8Plan p{};
    p.num_req = std::min(num_requests - at, kF8MaxReq);
    if (at > 0) {
      // the next requests: of the list, or of the arrays that a request indexes
      if (a.req_list) {
        a.req_list += kF8MaxReq;
      } else {
        a.seq_lens += kF8MaxReq;
        a.qsl += kF8MaxReq;
        a.num_seqs -= kF8MaxReq;
        if (a.table_rows) a.table_rows += kF8MaxReq;
        else a.tables += kF8MaxReq * a.tstride, a.num_table_rows -= kF8MaxReq;
      }
    }
    p.cuts = (F8Cut*)workspace;
    p.partials = (float*)((char*)workspace + f8_cut_bytes(sms));
    int rc;
    if (a.hd == 64) rc = dtype == NIE_DTYPE_F16 ? launch_prefill<64, __half>(a, p, sms, s) : launch_prefill<64, __nv_bfloat16>(a, p, sms, s);
    else rc = dtype == NIE_DTYPE_F16 ? launch_prefill<128, __half>(a, p, sms, s) : launch_prefill<128, __nv_bfloat16>(a, p, sms, s);
    if (rc != NIE_OK) return rc;
  }
  return NIE_OK;
}

}  // namespace nie
