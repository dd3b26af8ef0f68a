// Declarations shared by the attention kernels over the 8-bit paged cache.
#pragma once

#include "nie_kv8.cuh"

namespace nie {

struct Kv8Args {
  const void* q;
  void* out;
  int64_t q_stride, out_stride;  // elements between token rows
  int64_t num_q_rows;            // rows of q and out
  int64_t num_table_rows;        // rows of tables
  int num_seqs;                  // entries of seq_lens, q_rows and table_rows
  const uint8_t* kc;             // codes and scales of the layer
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  int64_t nb;
  int bs, hkv, hd, hq, group;
  const int32_t* tables;
  int64_t tstride, twidth;       // entries from one row to the next, entries of a row
  const int32_t* table_rows;
  const int32_t* seq_lens;
  const int64_t* q_rows;  // single-token calls: a request's query row (null: its index)
  const int64_t* qsl;     // ragged calls (non-null): a request's rows are [qsl[r], qsl[r + 1])
  const int32_t* req_list;
  float scale;
  int32_t* err;
};

// Query rows of request r: [first, first + count); row j sees the keys [0, keys + j].
struct Kv8Rows {
  int64_t first;
  int64_t count;
  int64_t keys;
};

// Rows outside [0, num_q_rows) do not exist: the request is flagged and has none.
__device__ __forceinline__ Kv8Rows kv8_rows(const Kv8Args& a, int r, int32_t* err) {
  Kv8Rows x;
  const int64_t n = a.seq_lens[r];
  if (a.qsl) {
    x.first = a.qsl[r];
    x.count = a.qsl[r + 1] - x.first;
  } else {
    x.first = a.q_rows ? a.q_rows[r] : (int64_t)r;
    x.count = 1;
  }
  x.keys = n - x.count;
  if (x.count > 0 && (x.first < 0 || x.first + x.count > a.num_q_rows)) {
    raise_flag(err, NIE_DEV_ERR_CAPACITY);
    x.count = 0;
  }
  return x;
}

// Kernels that the calling thread's last attention call launched; each launch adds itself.
int& kv8_launches();

// 16 bytes to shared memory, those past `bytes` zeros.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The kernel of single tokens (nie_kv8_decode.cu), where kv8_decode_takes() says
// so; workspace of kv8_decode_workspace() bytes, 256-byte aligned (none where it is 0).
bool kv8_decode_takes(int dtype, const Kv8Args& a);
size_t kv8_decode_workspace(int sms, const Kv8Args& a, int num_requests, int max_query_len);
int launch_kv8_decode(int dtype, const Kv8Args& a, int num_requests, int sms, void* workspace, bool overlap,
                      cudaStream_t s);

// The same for requests of a few query tokens each, max_query_len at most, where kv8_short_takes() them, too.
bool kv8_short_takes(int sms, const Kv8Args& a, int num_requests, int max_query_len);
int launch_kv8_short(int dtype, const Kv8Args& a, int num_requests, int max_query_len, int sms, void* workspace,
                     cudaStream_t s);

// The tcgen05 kernel of ragged queries (nie_kv8_prefill.cu), likewise.
bool kv8_prefill_takes(int dtype, const Kv8Args& a);
size_t kv8_prefill_workspace(int sms, int head_dim);
int launch_kv8_prefill(int dtype, const Kv8Args& a, int num_requests, int sms, void* workspace, cudaStream_t s);

}  // namespace nie
