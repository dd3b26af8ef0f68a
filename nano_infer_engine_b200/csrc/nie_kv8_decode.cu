// Attention of one query token, or of a few, over the 8-bit paged cache for bf16 /
// f16 queries, head_dim 64 or 128, blocks of a multiple of 16 tokens.
//
// What bounds it: the codes, read once.  One query token gives each code two
// multiply-adds per query head of its group, far below the tensor rate, so the
// work is to keep the loads of all SMs in flight and the instructions per code
// few enough to hide behind them.  Measured: 64 requests of up to 29600 keys, 8 kv
// heads of 64, 171 us, 5.7 TB/s of codes; one of 131072 keys, 4 of 128, 35 us, 3.8
// TB/s (27 us of it without any arithmetic, 6 in the merging kernel); 16 of up to
// 4001 keys 17 us, which the longest one's share of a cluster decides.
//
// Split.  The keys of all requests form one list of tiles (TOK tokens each, 4
// KiB of codes per kv head); CTA c takes the c-th of equal stretches of it,
// whatever the lengths, for HC kv heads, and deals the tiles of the stretch to
// TS = 8 / HC warps in turn.  Warps merge per request through shared memory; a
// request that lies in one CTA's stretch is finished there, one cut by a border
// leaves (max, sum, unnormalised output) to a second kernel.  Where the tables are
// short, a cluster of CTAs shares one request instead and merges in distributed
// shared memory.  Every order of summation follows from the lengths and the
// tables' width alone.
//
// One warp and tile.  cp.async brings the tile's codes to the warp's own ring of
// two stages: no barrier between warps.  The products are transposed, so that
// the 16 tokens of a sub-block fill the 16 rows of an m16n8k16 f16 MMA and the
// query heads of the group its 8 columns (two MMAs for up to 16).  With several
// query tokens the columns are (token, head) pairs, each with its own last key:
//   S^T[token, head] = K Q^T      A = codes as f16 (exact), B = q in registers
//   O^T[dim, head]  += V^T P^T    A = codes as f16 (exact), B = P^T (movmatrix)
// q is f16 as it is, or bf16 scaled by a power of two per head so that its
// largest element is near 2^15: 8 bits fit f16's 11, elements down to 2^-29 of
// the largest keep them all.
//
// Softmax with scales.  With c = ks scale log2(e) of a block, each key's weight
// on the codes of V is 2^(S c + log2 vs): the running maximum is kept over
// y = S c + log2 vs, p = 2^(y - m), O = sum p vcode and l = sum p / vs, so that
// what a block adds to O does not depend on how its scale and its codes share it.
// p is rounded to f16 for the second product, an error of 2^-12 of it; l takes it
// unrounded.  Next to a bf16 output's half step of 2^-9 that is nothing (1.6e-3 of the
// output's size from 64 bits either way); next to f16's 2^-12 it is as much again (2.8e-4 from
// 64 bits where an fp32 p leaves 2.1e-4).  What the rounding leaves, taken along in a second
// product, costs 8 % of the time at 64 requests and 3 % at one of 131072 keys.
// m is raised, and O and l rescaled, only when a p would pass 2^15 (the largest
// is 2^9 then): f16 ends at 2^16, and so has the most room below.  Weights (times vs)
// under 2^-23 of the largest lose bits, those under 2^-34 are in l alone.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "nie_kv8_attn.cuh"

namespace cg = cooperative_groups;

namespace nie {

constexpr int kD8Warps = 8;
constexpr int kD8Stages = 2;
constexpr int kD8Stage = 4096;     // bytes of K and V codes of one tile
constexpr int kD8MaxReq = 512;     // requests of one launch (their lengths sit in shared memory)
// Columns x head_dim of a kv head up to which requests of several tokens come here; above it the tensor tiles of the
// ragged kernel are filled well enough.  8 requests of 8 tokens behind 2000 keys, 32 heads on 8 of 64: 23.5 us here
// and 49.2 there (of 16 tokens: 31.6 and 50.3); 16 on 4 of 128: 27.5 and 37.6 (38.3 and 38.9).
constexpr int kD8ShortCols = 4096;
constexpr int kD8MaxCluster = 8;
constexpr float kD8Log2e = 1.4426950408889634f;
constexpr float kD8Most = 15.f, kD8Up = 9.f;  // log2 of p: its most, and that of the key that raised m

struct D8Plan {
  int num_req;
  int hc, ts;          // kv heads and token splits of a CTA: hc * ts = 8
  int cols;            // columns per kv head: its query heads, or (token, query head) pairs of the longest request
  int rows, subs;      // columns of one MMA column set; column sets per kv head
  int min_tiles;       // a CTA takes at least this many tiles
  int whole, log2;     // a cluster of whole = 2^log2 CTAs takes one request, and no kernel has to merge (0: not so)
  float* partials;     // [ctas + num_req][hkv * cols][hd + 4]
  int32_t* cum_out;    // [num_req + 2]: tiles before each request, then tiles per CTA
};

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16_16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Both code pairs of a word as f16 pairs.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = e4m3x2_to_f16x2((uint16_t)(w & 0xffffu));
  hi = e4m3x2_to_f16x2((uint16_t)(w >> 16));
}

// MMA row i of a sub-block holds this token: the four tokens that a lane of the
// second product needs (rows 2t, 2t + 1, 2t + 8, 2t + 9) are then t, t + 4, t + 8,
// t + 12, whose V rows lie in different banks.
__device__ __forceinline__ int row_token(int i) { return (i & 8) + ((i & 7) >> 1) + 4 * (i & 1); }

// Column `col` of kv head kvh, of a request whose first row is `row`.
template <bool MULTI, typename P>
__device__ __forceinline__ P* d8_row(P* base, int64_t stride, const Kv8Args& a, int row, int kvh, int col) {
  const int64_t token = MULTI ? col / a.group : 0;
  return base + (row + token) * stride + (int64_t)(kvh * a.group + (MULTI ? col % a.group : col)) * (int64_t)a.hd;
}

// Merge factor of a partial with reference m against M: one that saw no key has
// nothing to add (and NaN, which leaves m alone, must reach the result).
__device__ __forceinline__ float merge_weight(float m, float M) { return m == -INFINITY ? 0.f : fast_exp2(m - M); }

// MULTI: requests of several query tokens.  A column is a (token, query head of the group) pair then, and sees
// the keys up to its token's.
template <int HD, int NT, bool MULTI, typename T>
__global__ void __launch_bounds__(kD8Warps * 32, 2) kv8_decode_kernel(const __grid_constant__ Kv8Args a,
                                                                           const __grid_constant__ D8Plan p) {
  constexpr int TOK = 2048 / HD, SUBS = TOK / 16, CPR = HD / 16;  // tokens, sub-blocks, 16-byte chunks per row
  constexpr int ITEMS = 32 / SUBS;                                // tiles whose rows a warp looks up at once
  constexpr int MS = HD + 4;                                      // floats between rows of the merge buffer
  extern __shared__ __align__(128) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int R = p.num_req;
  uint8_t* ring = sm + warp * kD8Stages * kD8Stage;
  float4* info = reinterpret_cast<float4*>(sm + kD8Warps * kD8Stages * kD8Stage) + warp * kD8Stages * SUBS;
  float* merge = reinterpret_cast<float*>(sm + kD8Warps * kD8Stages * (kD8Stage + SUBS * 16));
  float* merge_ml = merge + kD8Warps * NT * 8 * MS;  // [warps][NT * 8][m, l]
  int* cum = reinterpret_cast<int*>(merge_ml + kD8Warps * NT * 8 * 2);
  int* len = cum + R + 1;
  int* trow = len + R;
  int* qrow = trow + R;
  int* count = qrow + R;  // MULTI: query tokens,
  int* behind = count + R;  // and the keys that the first of them does not see
  __shared__ int warp_sum[kD8Warps];

  pdl_trigger();  // the merging kernel may be staged now (it waits for this grid)
  // ---- lengths, tables and query rows of the requests; tiles before each
  // Keys past the end of a table have no block.  (And no sum of tiles passes an int.)
  const int64_t most = min(a.twidth * a.bs, (int64_t)((1 << 30) / R) * TOK);
  for (int i = threadIdx.x; i < R; i += kD8Warps * 32) {
    const int r = a.req_list ? a.req_list[i] : i;
    int n = 0, tr = 0, qr = -1, c = 0, past = 0;
    if (r >= 0 && r < a.num_seqs) {
      tr = a.table_rows ? a.table_rows[r] : r;
      const Kv8Rows rows = kv8_rows(a, r, a.err);
      if (rows.count > 0 && tr >= 0 && tr < a.num_table_rows) {
        n = max(a.seq_lens[r], 0);
        if (n > most) {
          raise_flag(a.err, NIE_DEV_ERR_BLOCK_RANGE);
          past = n - (int)most;
          n = (int)most;
        }
        qr = (int)rows.first;
        c = (int)rows.count;
        if (MULTI && rows.count * a.group > p.cols) n = 0, qr = -1, c = 0;  // longer than the call said
      } else if (MULTI && rows.count <= 0 && tr >= 0 && tr < a.num_table_rows) {
        qr = 0;  // no query token: nothing to do, nothing wrong
      }
    }
    if (qr < 0) raise_flag(a.err, NIE_DEV_ERR_CAPACITY);
    if constexpr (MULTI) {
      count[i] = c;
      behind[i] = max(0, c - 1 - past);
    }
    len[i] = n;
    trow[i] = tr;
    qrow[i] = qr;
  }
  __syncthreads();
  {
    const int i0 = 2 * threadIdx.x, i1 = i0 + 1;
    const int v0 = i0 < R ? (len[i0] + TOK - 1) / TOK : 0, v1 = i1 < R ? (len[i1] + TOK - 1) / TOK : 0;
    int x = v0 + v1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    int before = x - v0 - v1;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    if (i0 <= R) cum[i0] = before;
    if (i1 <= R) cum[i1] = before + v0;
    if (threadIdx.x == kD8Warps * 32 - 1 && R == 2 * kD8Warps * 32) cum[R] = before + v0 + v1;
  }
  __syncthreads();
  const int total = cum[R];
  const int W = max((total + (int)gridDim.x - 1) / (int)gridDim.x, p.min_tiles);
  int lo = (int)min((int64_t)blockIdx.x * W, (int64_t)total), hi = min(total, lo + W);
  const int mine = blockIdx.x >> p.log2, rank = blockIdx.x & (p.whole - 1);  // of a cluster
  if (p.whole) {
    const int n = cum[mine + 1] - cum[mine];
    lo = cum[mine] + (n * rank >> p.log2);
    hi = cum[mine] + (n * (rank + 1) >> p.log2);
  }
  // Everything above reads the step's metadata; the codes, scales and queries
  // may come from the kernel before, and the workspace may be in use by it.
  pdl_wait();
  if (p.whole) {
    if (p.whole == 1 && lo == hi && qrow[blockIdx.x] >= 0) {  // a request without keys: zeros
      for (int c = 0; c < p.hc; ++c) {
        const int v = blockIdx.y * p.hc + c, first = v % p.subs * p.rows;
        const int n = min(p.rows, (MULTI ? count[blockIdx.x] * a.group : a.group) - first) * HD;
        for (int x = threadIdx.x; x < n; x += kD8Warps * 32)
          *(d8_row<MULTI>(reinterpret_cast<T*>(a.out), a.out_stride, a, qrow[blockIdx.x], v / p.subs, first + x / HD) + x % HD) =
              Num<T>::from_f(0.f);
      }
    }
  } else if (blockIdx.x == 0 && blockIdx.y == 0) {
    for (int i = threadIdx.x; i <= R; i += kD8Warps * 32) p.cum_out[i] = cum[i];
    if (threadIdx.x == 0) p.cum_out[R + 1] = W;
  }
  float* shared_part = reinterpret_cast<float*>(sm);  // [hc * rows][hd + 4] for the cluster, over the ring
  if (lo >= hi) {
    if (p.whole <= 1) return;
    for (int x = threadIdx.x; x < p.hc * p.rows; x += kD8Warps * 32)
      *reinterpret_cast<float2*>(shared_part + x * (HD + 4) + HD) = make_float2(-INFINITY, 0.f);
  }

  auto locate = [&](int x) {
    int l = 0, h = R;  // cum[l] <= x < cum[h]
    while (h - l > 1) {
      const int mid = (l + h) >> 1;
      if (cum[mid] <= x) l = mid; else h = mid;
    }
    return l;
  };

  // ---- this warp: kv head and column set, and its tiles lo + split, + ts, ...
  const int vh = blockIdx.y * p.hc + warp % p.hc, split = warp / p.hc;
  const int kvh = vh / p.subs, col0 = (vh % p.subs) * p.rows;
  int nrows = min(p.rows, p.cols - col0);  // columns of this warp
  const int first = lo + split;
  const int items = first < hi ? (hi - first - 1) / p.ts + 1 : 0;
  const int64_t row_bytes = (int64_t)a.hkv * HD;
  const uint8_t* kbase = a.kc + (int64_t)kvh * HD;
  const uint8_t* vbase = a.vc + (int64_t)kvh * HD;
  const float coef = a.scale * kD8Log2e;

  // window: lane holds sub-block lane % SUBS of tile base + lane / SUBS
  int win_base = 0, win_row = 0, win_n = 0;
  float win_ks = 0.f, win_vs = 1.f;
  auto refill = [&](int base) {
    win_base = base;
    win_row = 0;
    win_n = 0;
    win_ks = 0.f;
    win_vs = 1.f;
    const int item = base + lane / SUBS;
    if (item < items) {
      const int x = first + item * p.ts;
      const int i = locate(x);
      const int tok = ((x - cum[i]) * SUBS + lane % SUBS) * 16;
      const int n = min(16, len[i] - tok);
      if (n > 0) {
        const int lb = tok / a.bs;
        const int64_t block = a.tables[(int64_t)trow[i] * a.tstride + lb];  // lb is in the table: no length passes it
        if (block < 0 || block >= a.nb) {
          raise_flag(a.err, NIE_DEV_ERR_BLOCK_RANGE);
        } else {
          win_row = (int)(block * a.bs + tok % a.bs);
          win_n = MULTI ? len[i] - tok : n;  // MULTI: all keys from here on, for the columns' ends
          win_ks = a.ks[block * a.hkv + kvh];
          win_vs = fminf(fmaxf(a.vs[block * a.hkv + kvh], kScaleMin), kScaleMax);
        }
      }
    }
  };
  auto issue = [&](int j) {
    if (j < items) {
      if (j - win_base >= ITEMS) refill(j);
      const int st = j % kD8Stages;
      const uint32_t base = smem_u32(ring + st * kD8Stage);
      const int at = (j - win_base) * SUBS;
      if (lane / SUBS == j - win_base)
        info[st * SUBS + lane % SUBS] = make_float4(win_ks * coef, __log2f(win_vs), 1.f / win_vs, __int_as_float(win_n));
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int row = lane / CPR + q * (32 / CPR), c = lane % CPR;
        const int i = row & 15;
        const int from = __shfl_sync(0xffffffffu, win_row, at + (row >> 4));
        const int n = __shfl_sync(0xffffffffu, win_n, at + (row >> 4));
        const int kt = row_token(i);
        const int kc = HD == 64 ? c : c ^ (i & 1);
        const int vc = HD == 64 ? c ^ (i & 2) : c ^ ((i & 3) << 1);
        cp_async16(base + row * HD + kc * 16, kbase + (int64_t)(from + kt) * row_bytes + c * 16, kt < n ? 16 : 0);
        cp_async16(base + kD8Stage / 2 + row * HD + vc * 16, vbase + (int64_t)(from + i) * row_bytes + c * 16,
                   i < n ? 16 : 0);
      }
    }
    cp_commit();
  };

  uint32_t qf[HD / 16][NT][2];
  float qs[NT][2];  // what undoes the scaling of heads 2t, 2t + 1
  float o[HD / 16][NT][4];
  float m[NT][2], l[NT][2];
  int back[NT][2], back_max = 0;  // MULTI: keys at the end that columns 2t, 2t + 1 (that any column) do not see

  auto begin = [&](int i) {
    if constexpr (MULTI) {
      nrows = min(min(p.rows, p.cols - col0), count[i] * a.group - col0);
      back_max = behind[i];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) back[nt][e] = max(0, back_max - (col0 + nt * 8 + 2 * t + e) / a.group);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + g;  // this lane: dims [HD / 4 * t, + HD / 4) of column h
      uint32_t raw[HD / 8];
      if (h < nrows) {
        const T* qh = d8_row<MULTI>(reinterpret_cast<const T*>(a.q), a.q_stride, a, qrow[i], kvh, col0 + h) + HD / 4 * t;
#pragma unroll
        for (int u = 0; u < HD / 8; ++u) raw[u] = *reinterpret_cast<const uint32_t*>(qh + 2 * u);
      } else {
#pragma unroll
        for (int u = 0; u < HD / 8; ++u) raw[u] = 0u;
      }
      float undo = 1.f;
      if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
        float mx = 0.f;
#pragma unroll
        for (int u = 0; u < HD / 8; ++u)
          mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(raw[u] << 16)), fabsf(__uint_as_float(raw[u] & 0xffff0000u))));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // largest element to [2^14, 2^15); rows of denormals stay where f32 can scale them
        const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 127);
        const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        undo = __uint_as_float((uint32_t)max(127 + e - 14, 1) << 23);
#pragma unroll
        for (int u = 0; u < HD / 8; ++u)
          raw[u] = pack_f16x2(__uint_as_float(raw[u] << 16) * up, __uint_as_float(raw[u] & 0xffff0000u) * up);
      }
      qs[nt][0] = __shfl_sync(0xffffffffu, undo, 8 * t);      // head 2t is lane group g = 2t
      qs[nt][1] = __shfl_sync(0xffffffffu, undo, 8 * t + 4);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        qf[ks][nt][0] = raw[2 * ks];
        qf[ks][nt][1] = raw[2 * ks + 1];
      }
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < HD / 16; ++j) o[j][nt][0] = o[j][nt][1] = o[j][nt][2] = o[j][nt][3] = 0.f;
    }
  };

  auto tile = [&](int st) {
    const uint8_t* kt = ring + st * kD8Stage;
    const uint8_t* vt = kt + kD8Stage / 2;
    float s[SUBS][NT][4];
    float ivs[SUBS];
    float mx[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mx[nt][0] = mx[nt][1] = -INFINITY;
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      uint32_t w0[HD / 16], w1[HD / 16];  // rows g and g + 8, dims [HD / 4 * t, + HD / 4)
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const int chunk = HD == 64 ? t : (2 * t + c) ^ (g & 1);
        *reinterpret_cast<uint4*>(&w0[4 * c]) = *reinterpret_cast<const uint4*>(kt + (u * 16 + g) * HD + chunk * 16);
        *reinterpret_cast<uint4*>(&w1[4 * c]) = *reinterpret_cast<const uint4*>(kt + (u * 16 + g + 8) * HD + chunk * 16);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        uint32_t a0, a1, a2, a3;
        codes_to_f16(w0[ks], a0, a2);
        codes_to_f16(w1[ks], a1, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16_16816(s[u][nt], a0, a1, a2, a3, qf[ks][nt][0], qf[ks][nt][1]);
      }
      const float4 f = info[st * SUBS + u];
      const int n = __float_as_int(f.w);
      ivs[u] = f.z;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][nt][e] = fmaf(s[u][nt][e], f.x * qs[nt][e & 1], f.y);
      }
      if (n < 16 + (MULTI ? back_max : 0)) {  // the end of the sequence, or a block that does not exist
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (row_token(e < 2 ? g : g + 8) >= n - (MULTI ? back[nt][e & 1] : 0)) s[u][nt][e] = -INFINITY;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mx[nt][0] = fmaxf(mx[nt][0], fmaxf(s[u][nt][0], s[u][nt][2]));
        mx[nt][1] = fmaxf(mx[nt][1], fmaxf(s[u][nt][1], s[u][nt][3]));
      }
    }
    bool raise = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) raise |= mx[nt][0] > m[nt][0] + kD8Most || mx[nt][1] > m[nt][1] + kD8Most;
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = mx[nt][e];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = fmaxf(x - kD8Up, m[nt][e]);
          const float keep = x == m[nt][e] ? 1.f : fast_exp2(m[nt][e] - x);
          m[nt][e] = x;
          l[nt][e] *= keep;
#pragma unroll
          for (int j = 0; j < HD / 16; ++j) {
            o[j][nt][e] *= keep;
            o[j][nt][e + 2] *= keep;
          }
        }
      }
    }
    float ref[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      ref[nt][0] = m[nt][0] == -INFINITY ? 0.f : m[nt][0];
      ref[nt][1] = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
    }
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      uint32_t b[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float* x = s[u][nt];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fast_exp2(x[e] - ref[nt][e & 1]);
        l[nt][0] = fmaf(x[0] + x[2], ivs[u], l[nt][0]);
        l[nt][1] = fmaf(x[1] + x[3], ivs[u], l[nt][1]);
        b[nt][0] = movmatrix_trans(pack_f16x2(x[0], x[1]));
        b[nt][1] = movmatrix_trans(pack_f16x2(x[2], x[3]));
      }
      uint32_t w[4][HD / 32];  // tokens t, t + 4, t + 8, t + 12; dims [HD / 8 * g, + HD / 8)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int tok = t + 4 * k;
        if constexpr (HD == 64) {
          const int chunk = (g >> 1) ^ (t & 2);
          *reinterpret_cast<uint2*>(w[k]) =
              *reinterpret_cast<const uint2*>(vt + (u * 16 + tok) * HD + chunk * 16 + (g & 1) * 8);
        } else {
          *reinterpret_cast<uint4*>(w[k]) = *reinterpret_cast<const uint4*>(vt + (u * 16 + tok) * HD + ((g ^ (t << 1)) * 16));
        }
      }
      if constexpr (MULTI) {
        const int n = __float_as_int(info[st * SUBS + u].w);
        if (n < 16 + back_max) {
          // some columns do not see all of it: NaN codes stay out of the product and go to those that do
          uint32_t any = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
              const uint32_t nan = __vcmpeq4(w[k][c] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              w[k][c] &= ~nan;
              any |= nan;
            }
          }
          if (__any_sync(0xffffffffu, any != 0)) {
            for (int tok = 0; tok < min(n, 16); ++tok) {
              const uint8_t* row = vt + (u * 16 + tok) * HD +
                                   (HD == 64 ? ((g >> 1) ^ (tok & 2)) * 16 + (g & 1) * 8 : (g ^ ((tok & 3) << 1)) * 16);
#pragma unroll
              for (int d = 0; d < HD / 8; ++d) {
                if ((row[d] & 0x7f) != 0x7f) continue;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    if (tok < n - back[nt][e]) o[d >> 1][nt][e + 2 * (d & 1)] = __int_as_float(0x7fffffff);
                }
              }
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < HD / 16; ++j) {
        // rows g and g + 8 of M-tile j are dims HD / 8 * g + 2 j and the next
        const uint32_t sel = (j & 1) ? 0x7362u : 0x5140u;
        uint32_t a0, a1, a2, a3;
        codes_to_f16(__byte_perm(w[0][j >> 1], w[1][j >> 1], sel), a0, a1);
        codes_to_f16(__byte_perm(w[2][j >> 1], w[3][j >> 1], sel), a2, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16_16816(o[j][nt], a0, a1, a2, a3, b[nt][0], b[nt][1]);
      }
    }
  };

  // ---- warps to the CTA, the CTA to the output or the merging kernel
  auto finish = [&](int i, bool whole, bool last) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[nt][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int h = nt * 8 + 2 * t + e;
        float* row = merge + (warp * NT * 8 + h) * MS;
        if (g == 0) {
          merge_ml[(warp * NT * 8 + h) * 2] = m[nt][e];
          merge_ml[(warp * NT * 8 + h) * 2 + 1] = x;
        }
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) *reinterpret_cast<float2*>(row + HD / 8 * g + 2 * j) = make_float2(o[j][nt][e], o[j][nt][e + 2]);
      }
    }
    __syncthreads();
    // one thread: four dims of one query head
    const int per_head = p.rows * (HD / 4);
    for (int x = threadIdx.x; x < p.hc * per_head; x += kD8Warps * 32) {
      const int c = x / per_head, h = x % per_head / (HD / 4), d = x % (HD / 4) * 4;
      const int v = blockIdx.y * p.hc + c, sub = v % p.subs;
      const int col = sub * p.rows + h, kv = v / p.subs;
      if (col >= (MULTI ? count[i] * a.group : p.cols)) continue;
      float M = -INFINITY;
      for (int s = 0; s < p.ts; ++s) M = fmaxf(M, merge_ml[((s * p.hc + c) * NT * 8 + h) * 2]);
      float L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s = 0; s < p.ts; ++s) {
        const int w = (s * p.hc + c) * NT * 8 + h;
        const float f = merge_weight(merge_ml[w * 2], M);
        const float4 y = *reinterpret_cast<const float4*>(merge + w * MS + d);
        L += merge_ml[w * 2 + 1] * f;
        O.x += y.x * f, O.y += y.y * f, O.z += y.z * f, O.w += y.w * f;
      }
      if (whole && p.whole <= 1) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        T* out = d8_row<MULTI>(reinterpret_cast<T*>(a.out), a.out_stride, a, qrow[i], kv, col) + d;
        out[0] = Num<T>::from_f(O.x * inv);
        out[1] = Num<T>::from_f(O.y * inv);
        out[2] = Num<T>::from_f(O.z * inv);
        out[3] = Num<T>::from_f(O.w * inv);
      } else {
        float* ps = p.whole ? shared_part + (c * p.rows + h) * (HD + 4) :
                    p.partials + ((int64_t)(blockIdx.x + i) * a.hkv * p.cols + kv * p.cols + col) * (HD + 4);
        *reinterpret_cast<float4*>(ps + d) = O;
        if (d == 0) *reinterpret_cast<float2*>(ps + HD) = make_float2(M, L);
      }
    }
    if (!last) __syncthreads();
  };

  if (lo < hi) {
    refill(0);
#pragma unroll
    for (int j = 0; j < kD8Stages - 1; ++j) issue(j);
    int j = 0;
    for (int i = locate(lo), at = lo; at < hi; ++i) {
      if (cum[i + 1] == at) continue;  // a request without keys
      const int end = min(hi, cum[i + 1]);
      begin(i);
      for (; j < items && first + j * p.ts < end; ++j) {
        cp_wait<kD8Stages - 2>();
        __syncwarp();  // the tile is there for every lane, and every lane is done with the stage that comes next
        issue(j + kD8Stages - 1);
        tile(j % kD8Stages);
      }
      finish(i, cum[i] >= lo && cum[i + 1] <= hi, end == hi);
      at = end;
    }
  }
  cp_wait<0>();
  if (p.whole <= 1) return;
  // ---- the cluster's CTAs to the output, each a share of it, in the order of their ranks
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int per_head = p.rows * (HD / 4);
  for (int x = rank * (kD8Warps * 32) + threadIdx.x; x < p.hc * per_head; x += p.whole * (kD8Warps * 32)) {
    const int c = x / per_head, h = x % per_head / (HD / 4), d = x % (HD / 4) * 4;
    const int v = blockIdx.y * p.hc + c, col = v % p.subs * p.rows + h;
    if (qrow[mine] < 0 || col >= (MULTI ? count[mine] * a.group : p.cols)) continue;
    const float* at = shared_part + (c * p.rows + h) * (HD + 4);
    float2 ml[kD8MaxCluster];
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < kD8MaxCluster; ++k) {
      ml[k] = k < p.whole ? *reinterpret_cast<const float2*>(cluster.map_shared_rank(at, k) + HD) : make_float2(-INFINITY, 0.f);
      M = fmaxf(M, ml[k].x);
    }
    float L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kD8MaxCluster; ++k) {
      if (ml[k].x == -INFINITY && ml[k].y == 0.f) continue;  // no key; its output need not be there
      const float f = merge_weight(ml[k].x, M);
      const float4 y = *reinterpret_cast<const float4*>(cluster.map_shared_rank(at, k) + d);
      L += ml[k].y * f;
      O.x += y.x * f, O.y += y.y * f, O.z += y.z * f, O.w += y.w * f;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* out = d8_row<MULTI>(reinterpret_cast<T*>(a.out), a.out_stride, a, qrow[mine], v / p.subs, col) + d;
    out[0] = Num<T>::from_f(O.x * inv);
    out[1] = Num<T>::from_f(O.y * inv);
    out[2] = Num<T>::from_f(O.z * inv);
    out[3] = Num<T>::from_f(O.w * inv);
  }
  cluster.sync();  // until the others have read
}

// Requests cut by a border: merge the CTAs' partials in order.  One CTA per
// (request, column, 4 LANES dims); GROUPS groups of its threads take every
// GROUPS-th partial, all of a thread's loads go out together.  Requests without
// keys get zeros.
template <int HD, int GROUPS, int LANES, bool MULTI, typename T>
__global__ void __launch_bounds__(LANES * GROUPS) kv8_decode_merge_kernel(const __grid_constant__ Kv8Args a,
                                                                           const __grid_constant__ D8Plan p) {
  __shared__ float4 so[GROUPS][LANES];
  __shared__ float sm_m[GROUPS], sm_l[GROUPS];
  pdl_wait();
  const int i = blockIdx.x, h = blockIdx.y;
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES, d = blockIdx.z * LANES + lane;
  const int lo = p.cum_out[i], hi = p.cum_out[i + 1], W = p.cum_out[p.num_req + 1];
  const int r = a.req_list ? a.req_list[i] : i;
  if (r < 0 || r >= a.num_seqs) return;  // flagged by the first kernel
  if (a.table_rows && (a.table_rows[r] < 0 || a.table_rows[r] >= a.num_table_rows)) return;
  const Kv8Rows rows = kv8_rows(a, r, nullptr);
  const int col = h % p.cols;
  if (rows.count <= 0 || (MULTI && (rows.count * a.group > p.cols || col >= rows.count * a.group))) return;
  T* out = d8_row<MULTI>(reinterpret_cast<T*>(a.out), a.out_stride, a, (int)rows.first, h / p.cols, col);
  if (lo == hi) {
    if (group == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * d + e] = Num<T>::from_f(0.f);
    }
    return;
  }
  const int c0 = lo / W, n = (hi - 1) / W - c0 + 1;
  if (n == 1) return;
  const float* base = p.partials + ((int64_t)(c0 + i) * a.hkv * p.cols + h) * (HD + 4);
  const int64_t stride = (int64_t)a.hkv * p.cols * (HD + 4);
  constexpr int K = 5;
  float M = -INFINITY, L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c = group; c < n; c += GROUPS * K) {
    float2 ml[K];
    float4 x[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float* ps = base + (c + k * GROUPS) * stride;
      const bool ok = c + k * GROUPS < n;
      ml[k] = ok ? *reinterpret_cast<const float2*>(ps + HD) : make_float2(-INFINITY, 0.f);
      x[k] = ok ? *reinterpret_cast<const float4*>(ps + 4 * d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mn = M;
#pragma unroll
    for (int k = 0; k < K; ++k) mn = fmaxf(mn, ml[k].x);
    const float keep = merge_weight(M, mn);
    L *= keep;
    O.x *= keep, O.y *= keep, O.z *= keep, O.w *= keep;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float f = merge_weight(ml[k].x, mn);
      L += ml[k].y * f;
      O.x += x[k].x * f, O.y += x[k].y * f, O.z += x[k].z * f, O.w += x[k].w * f;
    }
    M = mn;
  }
  so[group][lane] = O;
  if (lane == 0) {
    sm_m[group] = M;
    sm_l[group] = L;
  }
  __syncthreads();
  if (group != 0) return;
  float mn = -INFINITY;
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) mn = fmaxf(mn, sm_m[k]);
  L = 0.f;
  O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) {
    const float f = merge_weight(sm_m[k], mn);
    const float4 y = so[k][lane];
    L += sm_l[k] * f;
    O.x += y.x * f, O.y += y.y * f, O.z += y.z * f, O.w += y.w * f;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  out[4 * d + 0] = Num<T>::from_f(O.x * inv);
  out[4 * d + 1] = Num<T>::from_f(O.y * inv);
  out[4 * d + 2] = Num<T>::from_f(O.z * inv);
  out[4 * d + 3] = Num<T>::from_f(O.w * inv);
}

static size_t d8_header(int R) { return (((size_t)(R + 2) * sizeof(int32_t)) + 255) & ~size_t(255); }

bool kv8_decode_takes(int dtype, const Kv8Args& a) {
  auto aligned = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  return (dtype == NIE_DTYPE_BF16 || dtype == NIE_DTYPE_F16) && (a.hd == 64 || a.hd == 128) && a.bs % 16 == 0 &&
         a.nb * a.bs < (int64_t(1) << 31) && a.num_q_rows < (int64_t(1) << 31) && aligned(a.kc, 16) && aligned(a.vc, 16) &&
         aligned(a.q, 4) && a.q_stride % 2 == 0 && a.hq <= 65535;
}

template <int HD, int NT, bool MULTI, typename T>
static int launch_decode(const Kv8Args& a, const D8Plan& p, dim3 grid, int sms, bool overlap, cudaStream_t s) {
  constexpr int SUBS = 2048 / HD / 16;
  const size_t smem = (size_t)kD8Warps * kD8Stages * (kD8Stage + SUBS * 16) +
                      (size_t)kD8Warps * NT * 8 * (HD + 4 + 2) * sizeof(float) + (size_t)((4 + 2 * MULTI) * p.num_req + 1) * sizeof(int);
  auto* kernel = kv8_decode_kernel<HD, NT, MULTI, T>;
  const int rc = opt_in_smem(kSmemKv8Decode + MULTI * 6 + (HD == 128 ? 4 : (NT == 2) * 2) + std::is_same<T, __half>::value,
                             (const void*)kernel, smem);
  if (rc != NIE_OK) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kD8Warps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (overlap) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.whole > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)p.whole;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  ++kv8_launches();
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, p);
  if (e != cudaSuccess) return fail(NIE_ERR_CUDA, "kv8_decode_kernel launch: %s", cudaGetErrorString(e));
  if (p.whole) return NIE_OK;
  ++kv8_launches();
  // A request is cut into 1 + grid.x / requests parts on average, so a large batch's requests into few: four groups
  // take them in one round of loads, and more of the small CTAs are on the GPU at once.  64 requests of up to 29600
  // keys x 32 heads take 171.1 us in all with 4 groups of a whole row and 175.9 with 16.  Few requests have many
  // parts.  With 4 groups, 16, and 32 of 32 dims each, on wide tables: one of 131072 keys x 32 heads 45.6, 36.4 and
  // 35.5 us, one of 29600 18.5, 14.1 and 14.3, 4 of 4001 12.3, 11.9 and 11.8, 8 14.4, 13.8 and 14.0, 16 of 1 to 4001
  // 17.7, 17.3 and 19.4, 18 of 1 to 2000 14.4, 13.9 and 16.4, 16 of 1 to 29600 55.2, 54.8 and 57.1.
  const dim3 merge_grid((unsigned)p.num_req, (unsigned)(a.hkv * p.cols));
  const int64_t rows = (int64_t)p.num_req * a.hkv * p.cols;
  if (rows > 4 * sms)
    pdl_launch(kv8_decode_merge_kernel<HD, 4, HD / 4, MULTI, T>, merge_grid, dim3(HD), s, a, p);
  else if (rows > sms)
    pdl_launch(kv8_decode_merge_kernel<HD, 16, HD / 4, MULTI, T>, merge_grid, dim3(4 * HD), s, a, p);
  else
    pdl_launch(kv8_decode_merge_kernel<HD, 32, 8, MULTI, T>, dim3(merge_grid.x, merge_grid.y, HD / 32), dim3(256), s, a, p);
  return check_launch("kv8_decode_merge_kernel");
}

// Columns to a kv head and how many of them a warp takes: up to 16 share a warp's pass over the codes at head_dim 64;
// 8 at 128, where 16 leave registers for one CTA to an SM.  8 requests of 16000 keys, 20 columns: 72.8 us with 8 to a
// warp and 85.4 with 16 at head_dim 128, 68.2 and 66.0 at 64; one of 2000 keys: 13.7 and 16.1, 11.6 and 13.2.
static void d8_columns(D8Plan& p, const Kv8Args& a, int max_query_len) {
  p.cols = a.group * max_query_len;
  const int most = a.hd == 64 ? 16 : 8;
  p.subs = (p.cols + most - 1) / most;
  p.rows = (p.cols + p.subs - 1) / p.subs;
  const int sets = a.hkv * p.subs;
  // Two column sets to a CTA halve the warps that are merged per set.  With one, two, four and eight: 64 requests of up
  // to 29600 keys, 8 sets, 175.2, 171.1, 171.9 and 174.0 us; 16 of 1 to 4001 on wide tables 18.1, 16.5, 16.5 and 17.5;
  // 8 x 5 drafts, 16 sets, 15.9, 16.3, 18.1 and 21.7; one of 131072 keys, 4 sets, 34.3, 35.8 and 39.5.
  p.hc = sets % 2 == 0 ? 2 : 1;
  p.ts = kD8Warps / p.hc;
  p.min_tiles = p.ts;
}

// Where the tables hold few keys, a cluster of CTAs takes a request and needs no second launch: one CTA, more while
// there are SMs for them and 256 keys to each.  With at most 1024 keys to a CTA one request of 100 keys takes 5.6 us
// against 7.2 in two launches, 8 of 2000 11.8 and 12.3, 32 of 2000 19.3 and 23.0, 8 x 5 drafts behind up to 2000 16.1
// and 19.1; requests of very uneven length lose by it (16 of 1 to 4001 keys 17.3 and 16.5, one launch less).
static int d8_cluster_log2(int64_t keys, int num_req, int sets, int sms) {
  const int64_t room = 2 * sms / ((int64_t)num_req * sets);
  int log2 = 0;
  while ((1 << log2) < kD8MaxCluster && (2 << log2) <= room && keys > (256 << log2)) ++log2;
  return keys > (1024 << log2) ? -1 : log2;
}

// The split of p.num_req requests; CTAs to a column set.
static int d8_split(D8Plan& p, const Kv8Args& a, int max_query_len, int sms) {
  d8_columns(p, a, max_query_len);
  const int sets = a.hkv * p.subs / p.hc;
  p.log2 = d8_cluster_log2(a.twidth * a.bs, p.num_req, sets, sms);
  p.whole = p.log2 < 0 ? 0 : 1 << p.log2;
  p.log2 = std::max(p.log2, 0);
  return p.whole ? p.num_req * p.whole : std::max(1, 2 * sms / sets);
}

template <bool MULTI>
static int run_decode(int dtype, const Kv8Args& args, int num_requests, int max_query_len, int sms, void* workspace,
                      bool overlap, cudaStream_t s) {
  Kv8Args a = args;
  for (int at = 0; at < num_requests; at += kD8MaxReq) {
    D8Plan p{};
    p.num_req = std::min(num_requests - at, kD8MaxReq);
    if (at > 0) {
      // the next requests: of the list, or of the arrays that a request indexes
      if (a.req_list) {
        a.req_list += kD8MaxReq;
      } else {
        a.seq_lens += kD8MaxReq;
        a.num_seqs -= kD8MaxReq;
        if (a.table_rows) a.table_rows += kD8MaxReq;
        else a.tables += kD8MaxReq * a.tstride, a.num_table_rows -= kD8MaxReq;
        if (MULTI) {
          a.qsl += kD8MaxReq;
        } else if (a.q_rows) {
          a.q_rows += kD8MaxReq;
        } else {
          a.q = (const char*)a.q + kD8MaxReq * a.q_stride * 2;
          a.out = (char*)a.out + kD8MaxReq * a.out_stride * 2;
          a.num_q_rows -= kD8MaxReq;
        }
      }
      overlap = false;  // the kernel before is this function's own, which reads the same workspace
    }
    const int ctas = d8_split(p, a, max_query_len, sms), sets = a.hkv * p.subs / p.hc;
    p.cum_out = (int32_t*)workspace;
    p.partials = (float*)((char*)workspace + d8_header(std::min(num_requests, kD8MaxReq)));
    const dim3 grid((unsigned)ctas, (unsigned)sets);
    const bool half = dtype == NIE_DTYPE_F16;
    auto launch = [&](auto type) {
      using T = decltype(type);
      if (a.hd == 128) return launch_decode<128, 1, MULTI, T>(a, p, grid, sms, overlap, s);
      return p.rows > 8 ? launch_decode<64, 2, MULTI, T>(a, p, grid, sms, overlap, s)
                        : launch_decode<64, 1, MULTI, T>(a, p, grid, sms, overlap, s);
    };
    const int rc = half ? launch(__half()) : launch(__nv_bfloat16());
    if (rc != NIE_OK) return rc;
  }
  return NIE_OK;
}

int launch_kv8_decode(int dtype, const Kv8Args& a, int num_requests, int sms, void* workspace, bool overlap,
                      cudaStream_t s) {
  return run_decode<false>(dtype, a, num_requests, 1, sms, workspace, overlap, s);
}

size_t kv8_decode_workspace(int sms, const Kv8Args& a, int num_requests, int max_query_len) {
  // of the first launch: the last one has fewer requests, and more CTAs to each
  D8Plan p{};
  p.num_req = std::min(num_requests, kD8MaxReq);
  const int ctas = d8_split(p, a, max_query_len, sms);
  if (p.whole) return 0;
  return d8_header(p.num_req) + (size_t)(ctas + p.num_req) * a.hkv * p.cols * (a.hd + 4) * sizeof(float);
}

bool kv8_short_takes(int sms, const Kv8Args& a, int num_requests, int max_query_len) {
  return (a.hd == 64 || a.hd == 128) && (int64_t)max_query_len * a.group * a.hd <= kD8ShortCols &&
         (int64_t)a.hq * max_query_len <= 65535 &&
         kv8_decode_workspace(sms, a, num_requests, max_query_len) <= kv8_prefill_workspace(sms, a.hd);
}

int launch_kv8_short(int dtype, const Kv8Args& a, int num_requests, int max_query_len, int sms, void* workspace,
                     cudaStream_t s) {
  return run_decode<true>(dtype, a, num_requests, max_query_len, sms, workspace, false, s);
}

}  // namespace nie
