// Ragged causal attention over the 8-bit paged cache on tcgen05 / TMEM, for
// bf16 / f16 queries, head_dim 64 or 128, blocks of a multiple of 16 tokens.
//
// What bounds it: exp2.  A score costs 4 head_dim flops and one exp2; at 16
// exp2 per clock and SM against 8192 flops of f16 MMA, head_dim 64 spends twice
// the MMA's time in exp2 and head_dim 128 the same.  So the MMAs run behind
// the softmax of 256 query rows, and all else (loads, 8 bit to f16) is done by
// warps of its own.
//
// Rows.  The query heads of a kv head share its codes, so the rows of a tile are
// (token, head of the group) pairs in that order: 256 rows of one kv head, two
// MMA tiles A and B of 128.  A "segment" is one such tile of a request and kv
// head against all keys that its last token sees.
//
// Split.  All segments lie end to end, each weighted as its key tiles plus a
// fixed part; every CTA (one per SM) takes an equal stretch.  A segment cut by
// a border leaves (max, sum, unnormalised output) of each part for a merging
// kernel; which parts and in which order follows from the lengths alone.
//
// Roles (13 warps, all walking the same segments and key tiles):
//   warps 0-3, 4-7  softmax of tile A, B: a thread owns a row
//   warps 8-11      loaders: q to f16 (bf16 rows scaled by a power of two so that
//                   8 bits fit f16's 11 whatever the row's size), codes to f16
//                   (exact), into 128-byte swizzled shared memory; codes come
//                   two tiles ahead by cp.async into a thread's own bytes
//   warp 12         issues S = Q K^T, then O += P V (P from TMEM), A and B in turn:
//                   one tile's MMAs run under the other's softmax
//
// Softmax with scales as in the single-token kernel: y = S c + log2 vs per block
// of 16 keys, p = 2^(y - m) in f16 for the product (its error of 2^-12 is below
// the output's step), O = sum p vcode, l = sum p / vs from the unrounded p.  m
// is raised (and O and l rescaled) only when exceeded by more than 2^8.
//
// TMEM columns: S of A 0-127, of B 128-255 (P takes its place), O of A from 256,
// of B from 384.  Waits are bounded; one that runs out raises
// NIE_DEV_ERR_TIMEOUT and ends the CTA.
#include <algorithm>
#include <type_traits>

#include "nie_kv8_attn.cuh"

namespace nie {

constexpr int kF8Rows = 256;
constexpr int kF8Threads = 13 * 32;
constexpr int kF8Stages = 3;       // f16 key tiles in shared memory
constexpr int kF8MaxReq = 512;     // requests of one launch
constexpr int kF8SegCost = 2;      // a segment's fixed part, in key tiles
constexpr uint32_t kF8Wait = 1u << 22;
constexpr float kF8Log2e = 1.4426950408889634f;
constexpr float kF8Lazy = 8.f;
constexpr uint32_t kF8OCol = 256;

// What the merging kernel needs about the segment that begins in a CTA's
// stretch and goes on behind it (parts: CTAs after it that hold some of it).
struct F8Cut {
  int64_t row0;   // first row of the tile: (token, head) pairs of the request
  int64_t first;  // the request's first query row
  int32_t rows, kvh, parts, pad;
};

struct F8Plan {
  int num_req;
  float* partials;  // [2 * ctas][2 + hd][256]: a CTA's first segment (cut in front), its last (cut behind)
  F8Cut* cuts;      // [ctas]
};

template <int HD>
struct F8Cfg {
  static constexpr int BN = HD == 64 ? 128 : 64;          // keys of a tile
  static constexpr int QBufs = HD == 64 ? 2 : 1;
  static constexpr int QBytes = kF8Rows * HD * 2;
  static constexpr int TileBytes = BN * HD * 2;           // K or V of a tile in f16
  static constexpr int StageBytes = 2 * TileBytes;
  static constexpr int CodeBytes = 2 * BN * HD;           // codes of a tile
  static constexpr int Subs = BN / 16;
};

struct F8Bars {
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[kF8Stages], kv_empty[kF8Stages];
  uint64_t s_full[2], p_full[2], o_full[2], o_free[2];
  uint64_t done;
  uint32_t tmem_base;
  int abort;
  int start_req, start_tile, start_head;
  int64_t start_pos;
  float q_undo[2][kF8Rows];              // what undoes a row's scaling
  float4 info[kF8Stages][8];             // of 16 keys: score factor, log2 vs, 1 / vs
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
__device__ __forceinline__ uint32_t f8_pack(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void f8_cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// kind::f16 with f16 A and B, f32 D.
constexpr uint32_t f8_idesc(int m, int n, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// A request of the call; none of its fields depend on the kv head.
struct F8Req {
  int64_t first;  // first query row
  int64_t rows;   // query tokens * heads of a group
  int64_t ctx;    // keys before its first token (negative: the first tokens see none)
  int n;          // keys
  int trow;
  int tiles;      // 256-row tiles
};

__device__ __forceinline__ F8Req f8_request(const Kv8Args& a, int i, bool flag) {
  F8Req x{};
  const int r = a.req_list ? a.req_list[i] : i;
  const int tr = r < 0 || r >= a.num_seqs ? -1 : a.table_rows ? a.table_rows[r] : r;
  if (tr < 0 || tr >= a.num_table_rows) {
    if (flag) raise_flag(a.err, NIE_DEV_ERR_CAPACITY);
    return x;
  }
  Kv8Args q = a;
  if (!flag) q.err = nullptr;
  const Kv8Rows rows = kv8_rows(q, r);
  if (rows.count <= 0) return x;
  x.first = rows.first;
  x.rows = rows.count * a.group;
  x.ctx = rows.keys;
  x.n = max(a.seq_lens[r], 0);
  x.trow = tr;
  x.tiles = (int)((x.rows + kF8Rows - 1) / kF8Rows);
  return x;
}

// Keys that the last token of a tile sees, and the tiles of BN keys they fill (at
// least one: rows that see no key still get their zeros from a masked tile).
__device__ __forceinline__ int f8_keys(const F8Req& x, int group, int tile) {
  const int64_t last = (min(x.rows, (int64_t)(tile + 1) * kF8Rows) - 1) / group;
  return (int)max((int64_t)0, x.ctx + last + 1);
}
template <int BN>
__device__ __forceinline__ int f8_key_tiles(int keys) {
  return max(1, (keys + BN - 1) / BN);
}

// Walks the segments of a CTA's stretch [lo, hi): requests, tiles, kv heads.
template <int BN>
struct F8Walk {
  const Kv8Args* a;
  int num_req;
  int64_t lo, hi, start;  // start: cost position of the segment's first key tile
  int i, tile, h, keys, n;
  F8Req x;

  __device__ void load() {
    keys = f8_keys(x, a->group, tile);
    n = f8_key_tiles<BN>(keys);
  }
  __device__ void init(const Kv8Args* args, int R, const F8Bars* b, int64_t l, int64_t h_) {
    a = args;
    num_req = R;
    lo = l;
    hi = h_;
    i = b->start_req;
    tile = b->start_tile;
    h = b->start_head;
    x = f8_request(*a, i, false);
    load();
    start = b->start_pos + kF8SegCost;
  }
  __device__ bool valid() const { return start < hi; }
  __device__ int t_lo() const { return (int)(max(lo, start) - start); }
  __device__ int t_hi() const { return (int)(min(hi, start + n) - start); }
  __device__ int rows() const { return (int)min((int64_t)kF8Rows, x.rows - (int64_t)tile * kF8Rows); }
  __device__ void next() {
    start += n;
    if (++h == a->hkv) {
      h = 0;
      if (++tile >= x.tiles) {
        tile = 0;
        do {
          if (++i >= num_req) {
            start = hi;
            return;
          }
          x = f8_request(*a, i, false);
        } while (x.tiles == 0);
      }
      load();
    }
    start += kF8SegCost;
  }
};

template <int HD, typename T>
__global__ void __launch_bounds__(kF8Threads, 1) kv8_prefill_kernel(const Kv8Args a, const F8Plan p) {
  using C = F8Cfg<HD>;
  constexpr int BN = C::BN;
  extern __shared__ uint8_t f8_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(f8_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = sm;
  uint8_t* skv = sq + C::QBufs * C::QBytes;
  uint8_t* scode = skv + kF8Stages * C::StageBytes;
  F8Bars* b = reinterpret_cast<F8Bars*>(scode + 2 * C::CodeBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = p.num_req;

  pdl_wait();
  pdl_trigger();
  // ---- cost of each request (a warp each), then of all before it
  for (int i = warp; i < R; i += kF8Threads / 32) {
    const F8Req x = f8_request(a, i, blockIdx.x == 0 && lane == 0);
    int64_t cost = 0;
    for (int tile = lane; tile < x.tiles; tile += 32) cost += f8_key_tiles<BN>(f8_keys(x, a.group, tile)) + kF8SegCost;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) cost += __shfl_xor_sync(0xffffffffu, cost, o);
    if (lane == 0) b->cum[i + 1] = cost * a.hkv;
  }
  if (threadIdx.x == 0) {
    b->cum[0] = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b->q_full[i], 128);
      mbar_init(&b->q_empty[i], 1 + 8);
      mbar_init(&b->s_full[i], 1);
      mbar_init(&b->p_full[i], 128);
      mbar_init(&b->o_full[i], 1);
      mbar_init(&b->o_free[i], 128);
    }
    for (int s = 0; s < kF8Stages; ++s) {
      mbar_init(&b->kv_full[s], 128);
      mbar_init(&b->kv_empty[s], 1);
    }
    mbar_init(&b->done, 1);
    b->abort = 0;
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
    const F8Req x = f8_request(a, l, false);
    int64_t pos = b->cum[l];
    for (int t0 = 0; t0 < x.tiles; t0 += 32) {
      const int64_t c = t0 + lane < x.tiles ? f8_key_tiles<BN>(f8_keys(x, a.group, t0 + lane)) + kF8SegCost : 0;
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
  if (warp == 12) {
    tmem_alloc(&b->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = b->tmem_base;
  F8Walk<BN> seg;
  seg.init(&a, R, b, lo, hi);

  if (warp >= 8 && warp < 12) {
    // ------------------------------------------------------------ loaders
    const int tid = threadIdx.x - 256;
    const int64_t row_bytes = (int64_t)a.hkv * HD;
    const float coef = fabsf(a.scale) * kF8Log2e;
    const bool negate = a.scale < 0.f;
    // tiles come two ahead: `ahead` walks in front of `seg`
    F8Walk<BN> ahead = seg;
    int a_kt = ahead.valid() ? ahead.t_lo() : 0;
    while (ahead.valid() && a_kt >= ahead.t_hi()) {
      ahead.next();
      a_kt = ahead.valid() ? ahead.t_lo() : 0;
    }
    float pend_ks[2] = {0.f, 0.f}, pend_vs[2] = {1.f, 1.f};
    bool pend_ok[2] = {false, false};
    auto block_of = [&](const F8Walk<BN>& w, int key) -> int64_t {
      if (key >= w.keys || key >= w.x.n) return -1;
      const int lb = key / a.bs;
      const int64_t block = lb < a.tstride ? (int64_t)a.tables[(int64_t)w.x.trow * a.tstride + lb] : -1;
      if (block < 0 || block >= a.nb) {
        raise_flag(a.err, NIE_DEV_ERR_BLOCK_RANGE);
        return -1;
      }
      return block;
    };
    auto fetch = [&](int slot) {
      if (ahead.valid()) {
        const int key0 = a_kt * BN;
        const uint32_t base = smem_u32(scode + slot * C::CodeBytes) + tid * 16;
        int64_t block[BN / 32];
#pragma unroll
        for (int j = 0; j < BN / 32; ++j) block[j] = block_of(ahead, key0 + (tid >> 2) + 32 * j);
        const int64_t sb = tid < C::Subs ? block_of(ahead, key0 + 16 * tid) : -1;
        float ks = 0.f, vs = 1.f;
        if (sb >= 0) {
          ks = a.ks[sb * a.hkv + ahead.h];
          vs = a.vs[sb * a.hkv + ahead.h];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = (tid >> 2) + 32 * (j % (BN / 32)), half = j / (BN / 32);
          const int64_t blk = block[j % (BN / 32)];
          const int64_t off = blk < 0 ? 0
                                      : (blk * a.bs + (key0 + row) % a.bs) * row_bytes + (int64_t)ahead.h * HD + half * 64 +
                                            (tid & 3) * 16;
          f8_cp16(base + j * 2048, a.kc + off, blk < 0 ? 0 : 16);
          f8_cp16(base + (4 + j) * 2048, a.vc + off, blk < 0 ? 0 : 16);
        }
        pend_ks[slot] = fminf(fmaxf(ks, 0.f), kScaleMax);
        pend_vs[slot] = fminf(fmaxf(vs, kScaleMin), kScaleMax);
        pend_ok[slot] = sb >= 0;
        if (++a_kt >= ahead.t_hi()) {
          do {
            ahead.next();
            a_kt = ahead.valid() ? ahead.t_lo() : 0;
          } while (ahead.valid() && a_kt >= ahead.t_hi());
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(0);
    fetch(1);
    bool ok = true;
    int64_t g = 0;
    for (int k = 0; ok && seg.valid(); seg.next(), ++k) {
      // the tile's queries
      const int qb = k % C::QBufs;
      if (k >= C::QBufs && !f8_wait(b, &b->q_empty[qb], (uint32_t)((k / C::QBufs) - 1) & 1u, a.err)) break;
      constexpr int LPR = HD / 8;  // lanes of a row, 8 elements each
      const int rows = seg.rows();
      const int c = tid % LPR;
      uint8_t* qdst = sq + qb * C::QBytes;
      for (int r0 = 0; r0 < kF8Rows; r0 += 4 * (128 / LPR)) {
        uint4 raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int row = r0 + u * (128 / LPR) + tid / LPR;
          raw[u] = make_uint4(0u, 0u, 0u, 0u);
          if (row < rows) {
            const int64_t fr = (int64_t)seg.tile * kF8Rows + row;
            raw[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (seg.x.first + fr / a.group) * a.q_stride +
                                                     (int64_t)(seg.h * a.group + fr % a.group) * HD + c * 8);
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int row = r0 + u * (128 / LPR) + tid / LPR;
          uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
          float undo = 1.f;
          if constexpr (std::is_same<T, __half>::value) {
            if (negate) {
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] ^= 0x80008000u;
            }
          } else {
            float mx = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xffff0000u))));
#pragma unroll
            for (int o = 1; o < LPR; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            // largest element to [2^14, 2^15)
            const int e2 = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 127);
            float up = __uint_as_float((uint32_t)(127 + 14 - e2) << 23);
            undo = __uint_as_float((uint32_t)max(127 + e2 - 14, 1) << 23);
            if (negate) up = -up;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = f8_pack(__uint_as_float(w[e] << 16) * up, __uint_as_float(w[e] & 0xffff0000u) * up);
          }
          if (c == 0) b->q_undo[qb][row] = undo;
          uint8_t* dst = qdst + (row >> 7) * (128 * HD * 2) + (c >> 3) * (128 * 128) + (row & 127) * 128 +
                         (((c & 7) ^ (row & 7)) << 4);
          *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&b->q_full[qb]);
      // its key tiles
      const int thi = seg.t_hi();
      for (int kt = seg.t_lo(); kt < thi; ++kt, ++g) {
        const int st = (int)(g % kF8Stages), slot = (int)(g & 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        if (g >= kF8Stages && !f8_wait(b, &b->kv_empty[st], (uint32_t)((g / kF8Stages) - 1) & 1u, a.err)) {
          ok = false;
          break;
        }
        uint8_t* dst = skv + st * C::StageBytes;
        const uint8_t* src = scode + slot * C::CodeBytes + tid * 16;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int jj = j & 3;
          const int row = (tid >> 2) + 32 * (jj % (BN / 32)), half = jj / (BN / 32);
          const uint4 x = *reinterpret_cast<const uint4*>(src + j * 2048);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            h[2 * e] = e4m3x2_to_f16x2((uint16_t)(w[e] & 0xffffu));
            h[2 * e + 1] = e4m3x2_to_f16x2((uint16_t)(w[e] >> 16));
          }
          uint8_t* at = dst + (j >> 2) * C::TileBytes + half * (BN * 128) + row * 128;
          const int ch = 2 * (tid & 3);
          *reinterpret_cast<uint4*>(at + ((ch ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(at + (((ch + 1) ^ (row & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
        }
        if (tid < C::Subs)  // keys without a block have no weight
          b->info[st][tid] = pend_ok[slot] ? make_float4(pend_ks[slot] * coef, __log2f(pend_vs[slot]), 1.f / pend_vs[slot], 0.f)
                                           : make_float4(0.f, -INFINITY, 0.f, 0.f);
        fence_proxy_async_smem();
        mbar_arrive(&b->kv_full[st]);
        fetch(slot);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 12) {
    // --------------------------------------------------------- MMA issuer
    constexpr uint32_t id_s = f8_idesc(128, BN, false), id_o = f8_idesc(128, HD, true);
    // `nx` is the key tile whose scores are issued next, `cur` the one before it, whose P V follow
    struct Item {
      bool live = false, first = false, last = false, two = false;
      int k = 0, st = 0;
    } cur, nx;
    int k = 0, kt = 0;
    int64_t g = 0;
    bool fresh = true;
    int used[2] = {0, 0};       // scores issued per tile half
    int segs[2] = {0, 0};       // segments that wrote the half's output
    auto advance = [&]() {      // the next key tile of the stretch into nx
      nx.live = false;
      while (seg.valid()) {
        if (fresh) {
          kt = seg.t_lo();
          fresh = false;
        }
        if (kt < seg.t_hi()) {
          nx.live = true;
          nx.first = kt == seg.t_lo();
          nx.last = kt + 1 == seg.t_hi();
          nx.two = seg.rows() > 128;
          nx.k = k;
          nx.st = (int)(g % kF8Stages);
          ++kt;
          return;
        }
        seg.next();
        fresh = true;
        ++k;
      }
    };
    bool ok = true;
    auto scores = [&](int x) -> bool {  // S of half x for nx
      if (x == 0) {
        if (nx.first && !f8_wait(b, &b->q_full[nx.k % C::QBufs], (uint32_t)(nx.k / C::QBufs) & 1u, a.err)) return false;
        if (!f8_wait(b, &b->kv_full[nx.st], (uint32_t)(g / kF8Stages) & 1u, a.err)) return false;
      }
      tc_fence_after();
      if (lane == 0) {
        const uint32_t q = smem_u32(sq + (nx.k % C::QBufs) * C::QBytes + x * (128 * HD * 2));
        const uint32_t kk0 = smem_u32(skv + nx.st * C::StageBytes);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          tc_mma_ss(tbase + x * 128, smem_desc_sw128(q + (kk >> 2) * (128 * 128) + (kk & 3) * 32, 16, 1024),
                    smem_desc_sw128(kk0 + (kk >> 2) * (BN * 128) + (kk & 3) * 32, 16, 1024), id_s, kk > 0 ? 1u : 0u);
        tc_commit(&b->s_full[x]);
        // the queries are free once the segment's last scores are done
        if (nx.last && (x == 1 || !nx.two)) tc_commit(&b->q_empty[nx.k % C::QBufs]);
      }
      __syncwarp();
      return true;
    };
    auto product = [&](int x) -> bool {  // O of half x += P V for cur
      if (!f8_wait(b, &b->p_full[x], (uint32_t)(used[x] & 1), a.err)) return false;
      ++used[x];
      if (cur.first) {
        // the softmax warps have read the half's output of the segment before
        if (segs[x] > 0 && !f8_wait(b, &b->o_free[x], (uint32_t)(segs[x] - 1) & 1u, a.err)) return false;
        ++segs[x];
      }
      tc_fence_after();
      if (lane == 0) {
        const uint32_t v = smem_u32(skv + cur.st * C::StageBytes + C::TileBytes);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk) {
          // P of keys 64.. lies at the end of the S columns, see the softmax
          const uint32_t pcol = tbase + x * 128 + (kk < 4 ? kk * 8 : 96 + (kk - 4) * 8);
          tc_mma_ts(tbase + kF8OCol + x * 128, pcol, smem_desc_sw128(v + kk * 2048, BN * 128, 1024), id_o,
                    (!cur.first || kk > 0) ? 1u : 0u);
        }
        if (x == 1 || !cur.two) tc_commit(&b->kv_empty[cur.st]);
        if (cur.last) tc_commit(&b->o_full[x]);
      }
      __syncwarp();
      return true;
    };
    advance();
    if (nx.live) {
      ok = scores(0) && (!nx.two || scores(1));
      cur = nx;
      ++g;
      if (ok) advance();
      while (ok && cur.live) {
        ok = product(0);
        if (ok && nx.live) ok = scores(0);
        if (ok && cur.two) ok = product(1);
        if (ok && nx.live && nx.two) ok = scores(1);
        if (!ok) break;
        cur = nx;
        if (nx.live) {
          ++g;
          advance();
        }
      }
    }
    if (lane == 0) tc_commit(&b->done);
    __syncwarp();
    mbar_wait_bounded(&b->done, 0, kF8Wait);
  } else {
    // ------------------------------------------------------ softmax warps
    const int x = warp >> 2;                       // half
    const int t = (warp & 3) * 32 + lane;          // row of the half, TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tbase + lane_off + x * 128, o_addr = tbase + lane_off + kF8OCol + x * 128;
    bool ok = true;
    int64_t g = 0;
    int used = 0, segs = 0;
    for (int k = 0; ok && seg.valid(); seg.next(), ++k) {
      const int qb = k % C::QBufs;
      if (!f8_wait(b, &b->q_full[qb], (uint32_t)(k / C::QBufs) & 1u, a.err)) break;
      const int rows = seg.rows();
      const float undo = b->q_undo[qb][x * 128 + t];
      __syncwarp();
      if (lane == 0) mbar_arrive(&b->q_empty[qb]);
      const int tlo = seg.t_lo(), thi = seg.t_hi();
      if (x == 1 && rows <= 128) {  // the half has no rows
        g += thi - tlo;
        continue;
      }
      const bool active = x * 128 + (warp & 3) * 32 < rows;  // this warp has rows
      const int64_t fr = (int64_t)seg.tile * kF8Rows + x * 128 + t;
      const int64_t qpos = seg.x.ctx + fr / a.group;         // position of the row's token
      const int64_t first_pos = seg.x.ctx + (fr - lane) / a.group;  // of the warp's first row
      float m_ref = -INFINITY, l = 0.f;
      for (int kt = tlo; kt < thi; ++kt, ++g, ++used) {
        const int st = (int)(g % kF8Stages);
        if (!f8_wait(b, &b->s_full[x], (uint32_t)(used & 1), a.err) ||
            !f8_wait(b, &b->kv_full[st], (uint32_t)(g / kF8Stages) & 1u, a.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (active) {
          const float4* info = b->info[st];
          const int64_t key0 = (int64_t)kt * BN;
          const bool mask = key0 + BN - 1 > first_pos;
          const int seen = (int)min((int64_t)BN, max((int64_t)0, qpos - key0 + 1));  // keys of the tile that the row sees
          uint32_t v[64];
          float mx = -INFINITY;
          // largest y: per 16 keys the largest score, since their factor is not negative
#pragma unroll
          for (int h = 0; h < BN / 64; ++h) {
            tmem_ld32(s_addr + 64 * h, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
            tmem_ld32(s_addr + 64 * h + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
            tmem_wait_ld();
            if (mask) {
#pragma unroll
              for (int e = 0; e < 64; ++e)
                if (64 * h + e >= seen) v[e] = 0xff800000u;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              float s = __uint_as_float(v[16 * u]);
#pragma unroll
              for (int e = 1; e < 16; ++e) s = fmaxf(s, __uint_as_float(v[16 * u + e]));
              const float4 f = info[4 * h + u];
              mx = fmaxf(mx, fmaf(s, f.x * undo, f.y));
            }
          }
          const bool raise = mx > m_ref + kF8Lazy;
          if (__any_sync(0xffffffffu, raise)) {
            const float keep = raise ? (m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - mx)) : 1.f;
            if (raise) {
              l *= keep;
              m_ref = mx;
            }
            if (kt > tlo) {
              // O holds the products up to the last tile: these scores were issued after them, so their
              // arrival says that the products are done
              uint32_t o[32];
#pragma unroll
              for (int c = 0; c < HD / 32; ++c) {
                tmem_ld32(o_addr + 32 * c, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tmem_st32(o_addr + 32 * c, o);
              }
            }
          }
          const float ref = m_ref == -INFINITY ? 0.f : m_ref;
          // the half of the keys that is still in registers first: its P goes to the columns that it came from
#pragma unroll
          for (int h = BN / 64 - 1; h >= 0; --h) {
            if (h < BN / 64 - 1) {
              tmem_ld32(s_addr + 64 * h, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
              tmem_ld32(s_addr + 64 * h + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
              tmem_wait_ld();
            }
            uint32_t pk[32];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const float4 f = info[4 * h + u];
              const float fc = f.x * undo, fb = f.y - ref;
              float r0 = 0.f, r1 = 0.f;
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                float y0, y1;
                f8_fma2(y0, y1, __uint_as_float(v[16 * u + e]), __uint_as_float(v[16 * u + e + 1]), fc, fb);
                if (mask) {
                  if (64 * h + 16 * u + e >= seen) y0 = -INFINITY;
                  if (64 * h + 16 * u + e + 1 >= seen) y1 = -INFINITY;
                }
                const float p0 = fast_exp2(y0), p1 = fast_exp2(y1);
                f8_add2(r0, r1, p0, p1);
                pk[8 * u + e / 2] = f8_pack(p0, p1);
              }
              l = fmaf(r0 + r1, f.z, l);
            }
            tmem_st32(s_addr + 96 * h, pk);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(&b->p_full[x]);
      }
      if (!ok) break;
      if (!f8_wait(b, &b->o_full[x], (uint32_t)(segs & 1), a.err)) break;
      ++segs;
      tc_fence_after();
      const bool whole = tlo == 0 && thi == seg.n;
      const int row = x * 128 + t;
      float* ps = p.partials + (int64_t)(2 * blockIdx.x + (tlo == 0)) * (HD + 2) * kF8Rows + row;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* op = reinterpret_cast<T*>(a.out) + (seg.x.first + fr / a.group) * a.out_stride +
              (int64_t)(seg.h * a.group + fr % a.group) * HD;
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
              for (int e = 0; e < 32; ++e) ps[(2 + 32 * c + e) * kF8Rows] = __uint_as_float(o[e]);
            }
          }
        }
        if (!whole && row < rows) {
          ps[0] = m_ref;
          ps[kF8Rows] = l;
        }
      }
      tc_fence_before();
      mbar_arrive(&b->o_free[x]);
      if (tlo == 0 && thi < seg.n && threadIdx.x == 0)
        p.cuts[blockIdx.x] = F8Cut{(int64_t)seg.tile * kF8Rows, seg.x.first, rows, seg.h,
                                   (int)((seg.start + seg.n - 1) / W - blockIdx.x), 0};
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// Segments cut by borders: CTA (c, y) merges 32 rows of the one that begins in
// the first kernel's CTA c, its parts in order.  A thread: one row, every 8th dim.
template <int HD, typename T>
__global__ void __launch_bounds__(256) kv8_prefill_merge_kernel(const Kv8Args a, const F8Plan p) {
  pdl_wait();
  const F8Cut cut = p.cuts[blockIdx.x];
  const int row = blockIdx.y * 32 + (threadIdx.x & 31), d0 = threadIdx.x >> 5;
  if (cut.parts == 0 || row >= cut.rows) return;
  const int64_t size = (int64_t)(HD + 2) * kF8Rows;
  // part 0 is the CTA's last segment, the others the first one of the CTAs behind it
  auto part = [&](int k) { return p.partials + (2 * (int64_t)(blockIdx.x + k) + (k == 0)) * size + row; };
  float M = -INFINITY;
  for (int k = 0; k <= cut.parts; ++k) M = fmaxf(M, part(k)[0]);
  float L = 0.f, O[HD / 8];
#pragma unroll
  for (int d = 0; d < HD / 8; ++d) O[d] = 0.f;
  for (int k = 0; k <= cut.parts; ++k) {
    const float* ps = part(k);
    const float f = ps[0] == -INFINITY ? 0.f : fast_exp2(ps[0] - M);
    L += ps[kF8Rows] * f;
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) O[d] = fmaf(ps[(2 + d0 + 8 * d) * kF8Rows], f, O[d]);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int64_t fr = cut.row0 + row;
  T* op = reinterpret_cast<T*>(a.out) + (cut.first + fr / a.group) * a.out_stride +
          (int64_t)(cut.kvh * a.group + fr % a.group) * HD;
#pragma unroll
  for (int d = 0; d < HD / 8; ++d) op[d0 + 8 * d] = Num<T>::from_f(O[d] * inv);
}

static size_t f8_cut_bytes(int sms) { return ((size_t)sms * sizeof(F8Cut) + 255) & ~size_t(255); }

size_t kv8_prefill_workspace(int sms, int head_dim) {
  return f8_cut_bytes(sms) + (size_t)2 * sms * (head_dim + 2) * kF8Rows * sizeof(float);
}

bool kv8_prefill_takes(int dtype, const Kv8Args& a) {
  auto aligned = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  return (dtype == NIE_DTYPE_BF16 || dtype == NIE_DTYPE_F16) && (a.hd == 64 || a.hd == 128) && a.bs % 16 == 0 &&
         aligned(a.kc, 16) && aligned(a.vc, 16) && aligned(a.q, 16) && aligned(a.out, 16) && a.q_stride % 8 == 0 &&
         a.out_stride % 8 == 0;
}

template <int HD, typename T>
static int launch_prefill(const Kv8Args& a, const F8Plan& p, int sms, cudaStream_t s) {
  using C = F8Cfg<HD>;
  const size_t smem = 1024 + (size_t)C::QBufs * C::QBytes + (size_t)kF8Stages * C::StageBytes + 2 * C::CodeBytes + sizeof(F8Bars);
  auto* kernel = kv8_prefill_kernel<HD, T>;
  const int rc = opt_in_smem(kSmemKv8Prefill + (HD == 128) * 2 + std::is_same<T, __half>::value, (const void*)kernel, smem);
  if (rc != NIE_OK) return rc;
  kernel<<<sms, kF8Threads, smem, s>>>(a, p);
  const int st = check_launch("kv8_prefill_kernel");
  if (st != NIE_OK) return st;
  pdl_launch(kv8_prefill_merge_kernel<HD, T>, dim3((unsigned)sms, kF8Rows / 32), dim3(256), s, a, p);
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
