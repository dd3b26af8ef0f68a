// Entry points of the attention over the 8-bit paged cache, and the kernel of
// the shapes that no other takes: any activation type / block size / head group,
// head_dim <= 256:
//   S = scale * q . (kc ks[block]),  P = softmax over the visible keys,
//   out = sum P (vc vs[block]),      everything in fp32, rounded once.
// One CTA per (request, query row, query head); its four warps walk the keys
// in turn with a running maximum and sum, and merge at the end.  A row that
// sees no key gives zeros.  Each query row and head reads the codes for itself, a byte a
// lane: 16 requests of up to 4001 keys, 32 heads on 8 of 64, take 1.6 ms in fp32 (17 us in
// bf16 by the fast kernel), 513 tokens behind 487 4.0 ms (37 us).
#include "nie_kv8_attn.cuh"

#include <algorithm>

namespace nie {

int& kv8_launches() {
  static thread_local int n = 0;
  return n;
}

constexpr int kG8Warps = 4;
constexpr int kG8MaxHd = 256;

template <typename T>
__global__ void __launch_bounds__(kG8Warps * 32) kv8_generic_kernel(Kv8Args a) {
  using N = Num<T>;
  constexpr int kPer = kG8MaxHd / 32;
  const int h = blockIdx.z, kvh = h / a.group;
  const int r = a.req_list ? a.req_list[blockIdx.x] : (int)blockIdx.x;
  const int trow = r < 0 || r >= a.num_seqs ? -1 : a.table_rows ? a.table_rows[r] : r;
  if (trow < 0 || trow >= a.num_table_rows) {
    raise_flag(a.err, NIE_DEV_ERR_CAPACITY);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t* table = a.tables + (int64_t)trow * a.tstride;
  const int64_t row_elems = (int64_t)a.hkv * a.hd;
  const Kv8Rows rows = kv8_rows(a, r, a.err);
  __shared__ float sm_m[kG8Warps], sm_l[kG8Warps], sm_o[kG8Warps][kG8MaxHd];

  for (int64_t j = blockIdx.y; j < rows.count; j += gridDim.y) {
    int64_t keys = rows.keys + j + 1;  // this row sees the keys [0, keys)
    if (keys > a.twidth * a.bs) {  // those past the end of the table have no block
      if (threadIdx.x == 0) raise_flag(a.err, NIE_DEV_ERR_BLOCK_RANGE);
      keys = a.twidth * a.bs;
    }
    const T* qp = reinterpret_cast<const T*>(a.q) + (rows.first + j) * a.q_stride + (int64_t)h * a.hd;
    float q[kPer], o[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int d = lane + 32 * u;
      q[u] = d < a.hd ? N::to_f(qp[d]) : 0.f;
      o[u] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int64_t p = warp; p < keys; p += kG8Warps) {
      const int64_t block = table[p / a.bs];
      if (block < 0 || block >= a.nb) {
        if (lane == 0) raise_flag(a.err, NIE_DEV_ERR_BLOCK_RANGE);
        continue;
      }
      const int64_t at = (block * a.bs + p % a.bs) * row_elems + (int64_t)kvh * a.hd;
      float dot = 0.f;
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int d = lane + 32 * u;
        if (d < a.hd) dot = fmaf(q[u], e4m3_to_float(a.kc[at + d]), dot);
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
      const float s = dot * a.ks[block * a.hkv + kvh] * a.scale;
      const float mn = fmaxf(m, s);
      const float keep = m == -INFINITY ? 0.f : expf(m - mn);  // no key so far: nothing to keep
      const float pr = s == -INFINITY ? 0.f : expf(s - mn);  // -inf - -inf where nothing finite came yet
      const float pv = pr * a.vs[block * a.hkv + kvh];
      l = l * keep + pr;
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int d = lane + 32 * u;
        if (d < a.hd) o[u] = fmaf(pv, e4m3_to_float(a.vc[at + d]), o[u] * keep);
      }
      m = mn;
    }
    if (lane == 0) {
      sm_m[warp] = m;
      sm_l[warp] = l;
    }
#pragma unroll
    for (int u = 0; u < kPer; ++u)
      if (lane + 32 * u < a.hd) sm_o[warp][lane + 32 * u] = o[u];
    __syncthreads();
    float gm = -INFINITY;
    for (int w = 0; w < kG8Warps; ++w) gm = fmaxf(gm, sm_m[w]);
    T* op = reinterpret_cast<T*>(a.out) + (rows.first + j) * a.out_stride + (int64_t)h * a.hd;
    for (int d = threadIdx.x; d < a.hd; d += kG8Warps * 32) {
      float num = 0.f, den = 0.f;
      for (int w = 0; w < kG8Warps; ++w) {
        // a warp without keys has nothing to add; NaN scores leave their mark in l
        const float f = sm_m[w] == -INFINITY ? (sm_l[w] == 0.f ? 0.f : 1.f) : expf(sm_m[w] - gm);
        num += f * sm_o[w][d];
        den += f * sm_l[w];
      }
      op[d] = N::from_f(den == 0.f ? 0.f : num / den);
    }
    __syncthreads();
  }
}

static int launch_kv8_generic(int dtype, const Kv8Args& a, int num_req, int max_q, cudaStream_t s) {
  if (a.hd > kG8MaxHd) return fail(NIE_ERR_UNSUPPORTED, "head_dim %d > %d", a.hd, kG8MaxHd);
  if (a.hq > 65535) return fail(NIE_ERR_UNSUPPORTED, "too many query heads: %d", a.hq);
  ++kv8_launches();
  const dim3 grid((unsigned)num_req, (unsigned)std::min(std::max(max_q, 1), 65535), (unsigned)a.hq);
  switch (dtype) {
    case NIE_DTYPE_F32: kv8_generic_kernel<float><<<grid, kG8Warps * 32, 0, s>>>(a); break;
    case NIE_DTYPE_BF16: kv8_generic_kernel<__nv_bfloat16><<<grid, kG8Warps * 32, 0, s>>>(a); break;
    default: kv8_generic_kernel<__half><<<grid, kG8Warps * 32, 0, s>>>(a); break;
  }
  return check_launch("kv8_generic_kernel");
}

static int check_args(const Kv8Args& a, int32_t dtype, int32_t layer, int64_t num_layers, int32_t num_requests) {
  NIE_REQUIRE(dtype_size(dtype) > 0, "unknown dtype %d", dtype);
  NIE_REQUIRE(a.q && a.out && a.kc && a.vc && a.ks && a.vs && a.tables && a.seq_lens, "null pointer argument");
  NIE_REQUIRE(layer >= 0 && layer < num_layers, "layer %d out of range", layer);
  NIE_REQUIRE(a.nb > 0 && a.bs > 0 && a.hkv > 0 && a.hd > 0 && a.hq > 0, "bad geometry");
  NIE_REQUIRE(a.hq % a.hkv == 0, "q_heads must be divisible by kv_heads");
  NIE_REQUIRE(num_requests >= 0, "num_requests must be non-negative");
  NIE_REQUIRE(a.twidth > 0 && a.tstride >= a.twidth, "table_width must be positive and at most table_stride");
  NIE_REQUIRE(a.num_q_rows >= 0 && a.num_table_rows >= 0 && a.num_seqs >= 0, "row counts must be non-negative");
  return NIE_OK;
}

static void to_layer(Kv8Args& a, int32_t layer) {
  const int64_t codes = (int64_t)layer * a.nb * a.bs * a.hkv * a.hd, scales = (int64_t)layer * a.nb * a.hkv;
  a.kc += codes;
  a.vc += codes;
  a.ks += scales;
  a.vs += scales;
  a.group = a.hq / a.hkv;
}

// What the choice of a kernel and its workspace depend on, into a.
static bool geometry(Kv8Args& a, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t block_size,
                     int64_t table_width) {
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0 || block_size <= 0 || table_width < 0)
    return false;
  a.hq = q_heads, a.hkv = kv_heads, a.hd = head_dim, a.bs = block_size, a.twidth = table_width;
  a.group = q_heads / kv_heads;
  return true;
}

static size_t varlen_workspace(int sms, const Kv8Args& a, int num_requests, int max_query_len) {
  return kv8_short_takes(sms, a, num_requests, max_query_len) ? kv8_decode_workspace(sms, a, num_requests, max_query_len)
                                                              : kv8_prefill_workspace(sms, a.hd);
}

static bool holds(const void* workspace, size_t bytes, size_t need) {
  return need == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && bytes >= need);
}

}  // namespace nie

using namespace nie;

extern "C" int nie_paged_decode_kv8(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride,
                                    int64_t num_q_rows, const void* key_cache, const void* value_cache,
                                    const float* key_scales, const float* value_scales, int32_t dtype, int32_t layer,
                                    int64_t num_layers, int64_t num_blocks, int32_t block_size, int32_t kv_heads,
                                    int32_t head_dim, int32_t q_heads, const int32_t* block_tables,
                                    int64_t table_stride, int64_t table_width, int64_t num_table_rows,
                                    const int32_t* table_rows, const int32_t* seq_lens, int32_t num_seqs,
                                    const int64_t* q_rows,
                                    const int32_t* req_list, int32_t num_requests, float scale,
                                    void* workspace, size_t workspace_bytes, int32_t overlap, int32_t* err_flag,
                                    void* stream) {
  kv8_launches() = 0;
  Kv8Args a{};
  a.q = q, a.out = out, a.q_stride = q_row_stride, a.out_stride = out_row_stride, a.num_q_rows = num_q_rows;
  a.kc = (const uint8_t*)key_cache, a.vc = (const uint8_t*)value_cache, a.ks = key_scales, a.vs = value_scales;
  a.nb = num_blocks, a.bs = block_size, a.hkv = kv_heads, a.hd = head_dim, a.hq = q_heads;
  a.tables = block_tables, a.tstride = table_stride, a.twidth = table_width, a.num_table_rows = num_table_rows, a.table_rows = table_rows;
  a.seq_lens = seq_lens, a.num_seqs = num_seqs, a.q_rows = q_rows, a.req_list = req_list;
  a.scale = scale, a.err = err_flag;
  const int rc = check_args(a, dtype, layer, num_layers, num_requests);
  if (rc != NIE_OK) return rc;
  if (num_requests == 0) return NIE_OK;
  to_layer(a, layer);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (kv8_decode_takes(dtype, a)) {
    const int sms = sm_count(stream_device(s));
    NIE_REQUIRE(sms > 0, "cannot query the SM count");
    NIE_REQUIRE(holds(workspace, workspace_bytes, kv8_decode_workspace(sms, a, num_requests, 1)),
                "workspace too small or not 256-byte aligned");
    return launch_kv8_decode(dtype, a, num_requests, sms, workspace, overlap != 0, s);
  }
  return launch_kv8_generic(dtype, a, num_requests, 1, s);
}

extern "C" int nie_kv8_launch_count(void) { return kv8_launches(); }

extern "C" size_t nie_paged_decode_kv8_workspace_size(int device, int32_t num_requests, int32_t q_heads,
                                                      int32_t kv_heads, int32_t head_dim, int32_t block_size,
                                                      int64_t table_width) {
  Kv8Args a{};
  const int sms = sm_count(device);
  if (sms <= 0 || num_requests <= 0 || !geometry(a, q_heads, kv_heads, head_dim, block_size, table_width)) return 0;
  return kv8_decode_workspace(sms, a, num_requests, 1);
}

extern "C" int nie_varlen_attention_kv8(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride,
                                        int64_t num_q_rows, const void* key_cache, const void* value_cache,
                                        const float* key_scales, const float* value_scales, int32_t dtype,
                                        int32_t layer, int64_t num_layers, int64_t num_blocks, int32_t block_size,
                                        int32_t kv_heads, int32_t head_dim, int32_t q_heads,
                                        const int32_t* block_tables, int64_t table_stride, int64_t table_width,
                                        int64_t num_table_rows, const int32_t* table_rows, const int32_t* seq_lens,
                                        int32_t num_seqs, const int64_t* query_start_loc,
                                        const int32_t* req_list, int32_t num_requests, int32_t max_query_len,
                                        float scale, void* workspace, size_t workspace_bytes, int32_t* err_flag,
                                        void* stream) {
  kv8_launches() = 0;
  Kv8Args a{};
  a.q = q, a.out = out, a.q_stride = q_row_stride, a.out_stride = out_row_stride, a.num_q_rows = num_q_rows;
  a.kc = (const uint8_t*)key_cache, a.vc = (const uint8_t*)value_cache, a.ks = key_scales, a.vs = value_scales;
  a.nb = num_blocks, a.bs = block_size, a.hkv = kv_heads, a.hd = head_dim, a.hq = q_heads;
  a.tables = block_tables, a.tstride = table_stride, a.twidth = table_width, a.num_table_rows = num_table_rows, a.table_rows = table_rows;
  a.seq_lens = seq_lens, a.num_seqs = num_seqs, a.qsl = query_start_loc, a.req_list = req_list;
  a.scale = scale, a.err = err_flag;
  const int rc = check_args(a, dtype, layer, num_layers, num_requests);
  if (rc != NIE_OK) return rc;
  NIE_REQUIRE(query_start_loc, "null pointer argument");
  NIE_REQUIRE(max_query_len > 0, "max_query_len must be positive");
  if (num_requests == 0) return NIE_OK;
  to_layer(a, layer);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (kv8_prefill_takes(dtype, a)) {
    const int sms = sm_count(stream_device(s));
    NIE_REQUIRE(sms > 0, "cannot query the SM count");
    NIE_REQUIRE(holds(workspace, workspace_bytes, varlen_workspace(sms, a, num_requests, max_query_len)),
                "workspace too small or not 256-byte aligned");
    if (kv8_short_takes(sms, a, num_requests, max_query_len))
      return launch_kv8_short(dtype, a, num_requests, max_query_len, sms, workspace, s);
    return launch_kv8_prefill(dtype, a, num_requests, sms, workspace, s);
  }
  return launch_kv8_generic(dtype, a, num_requests, max_query_len, s);
}

extern "C" size_t nie_varlen_kv8_workspace_size(int device, int32_t num_requests, int32_t q_heads, int32_t kv_heads,
                                                int32_t head_dim, int32_t block_size, int64_t table_width,
                                                int32_t max_query_len) {
  Kv8Args a{};
  const int sms = sm_count(device);
  if (sms <= 0 || num_requests <= 0 || max_query_len <= 0 ||
      !geometry(a, q_heads, kv_heads, head_dim, block_size, table_width))
    return 0;
  return varlen_workspace(sms, a, num_requests, max_query_len);
}
