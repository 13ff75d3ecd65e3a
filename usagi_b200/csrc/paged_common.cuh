// paged_common.cuh -- what the paged-cache kernels share: the view of the cache and the batch,
// the rule that turns a sequence's lengths into tiles, and thin wrappers of the warp-level
// instructions (cp.async, ldmatrix, mma.sync, programmatic launch).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/bsattn.h"

namespace bsattn {

unsigned long long launch_timeout_ns();  // bsattn_set_timeout_ns
int launch_test_wait();                  // bsattn_test_unsignalled_wait

namespace paged {

constexpr int kHeadDim = 128;
constexpr int kTileKeys = 128;  // the block size of the window rule, keys of a tensor-core tile

// The cache and the batch as the kernels see them.  Strides are in bytes; the last dimension of
// the pages is contiguous.
struct Cache {
  const char* k;
  const char* v;
  long long k_page, k_head, k_tok;
  long long v_page, v_head, v_tok;
  const int32_t* table;
  long long table_stride;
  const int32_t* seq_lens;
  const int32_t* q_lens;  // null: every sequence has Tq live rows
  int max_pages, n_pages, page_shift;
  int B, Hkv, Tq;
  int* err;
};

__device__ __forceinline__ void raise(int* err, int code) { atomicCAS(err, 0, code); }

// Length of sequence b and its live rows, both forced into what the table and the call can hold;
// a value outside is reported and never used to form an address.
struct SeqLen {
  int len, rows;
  bool ok;  // neither had to be forced
};
__device__ __forceinline__ SeqLen seq_len(const Cache& c, int b) {
  SeqLen s;
  const int cap = c.max_pages << c.page_shift;
  const int len = __ldg(c.seq_lens + b);
  const int rows = c.q_lens != nullptr ? __ldg(c.q_lens + b) : c.Tq;
  s.len = min(max(len, 0), cap);
  s.rows = min(max(rows, 0), c.Tq);
  s.ok = s.len == len && s.rows == rows;
  if (!s.ok) raise(c.err, BSATTN_E_PAGE);
  return s;
}

// Page of key position `pos` of sequence b, or -1 (reported) when the table entry is no page.
__device__ __forceinline__ int page_checked(const Cache& c, int page) {
  if (static_cast<unsigned>(page) < static_cast<unsigned>(c.n_pages)) return page;
  raise(c.err, BSATTN_E_PAGE);
  return -1;
}

// Which keys a call reads: those from k0 on (behind a shared prefix), or by the window rule
// (window > 0, k0 == 0): for a row in block i = position / 128 the blocks < glob and > i - window.
struct Rule {
  int k0, window, glob;
};

// The live rows of a sequence: row t is the token at position first + t.
struct Rows {
  int rows, first;
};

// The keys one row sees: j < limit, and j >= lo or j < glob_end.  limit == 0: none.
struct RowKeys {
  int limit, lo;
};
__device__ __forceinline__ RowKeys row_keys(const Rows& t, const Rule& r, int row_t) {
  RowKeys k;
  const int pos = t.first + row_t;
  k.limit = (row_t < t.rows && pos >= 0) ? pos + 1 : 0;
  k.lo = r.window == 0 ? 0 : max(0, pos / kTileKeys - r.window + 1) * kTileKeys;
  return k;
}

// ---------------------------------------------------------------- instructions
// Loads of what is read once: L2 gives it up before anything else.
__device__ __forceinline__ uint64_t evict_first_policy() {
  uint64_t x;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(x));
  return x;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes, uint64_t pol) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src),
               "r"(bytes), "l"(pol)
               : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint64_t pol) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(pol)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Transposes an 8x8 matrix of 16-bit values held two per lane (row = lane / 4).
__device__ __forceinline__ uint32_t movm_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, const uint32_t* b) {
  if constexpr (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  }
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}
__device__ __forceinline__ uint32_t pack_out(float lo, float hi, int bf16) {
  return bf16 ? pack16<true>(lo, hi) : pack16<false>(lo, hi);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t v) {
  if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
// Programmatic launch.  Every kernel here is launched so that it may begin while its predecessor on the
// stream still runs, and waits for that one's end and results (pdl_wait) before it touches memory: what
// is saved is the launch, a microsecond or two of a call that takes ten.  It lets its own successor
// begin (pdl_trigger) only after that wait, so whoever comes next finds everything before it complete.
__device__ __forceinline__ void pdl_trigger() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---------------------------------------------------------------- host
// Number of SMs of the current device (checked to be sm_100).
int device_sms(int* sms);

// Launches a kernel of one parameter record, to begin while its predecessor still runs.
template <class P>
inline int launch(void (*kernel)(P), dim3 grid, int threads, size_t smem, cudaStream_t stream, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess) return BSATTN_OK;
  cudaGetLastError();
  return BSATTN_E_CUDA;
}

// Checks a call and fills the kernels' view of its cache (paged_attn.cu).
int fill_cache(Cache* c, const bsattn_paged_call* call);

}  // namespace paged
}  // namespace bsattn
