// Shared by the paged-cache kernels: kernel parameters, the span of a
// sequence's new tokens, and the host-side launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/kda_paged_hip.h"

namespace kda {

// The cache and the new tokens of a call (kda_paged_hip.h); strides in
// elements unless named otherwise.
struct PagedParams {
    int N, T, HQ, HKV, G;  // G = HQ / HKV
    int P, page_shift, M;
    int causal, window;
    int fp16;
    int cu_i64;
    float scale;
    const void* cu_seqlens;
    const int32_t* page_table;
    int64_t table_stride;
    const int32_t* seq_lens;
    uint16_t* k;
    uint16_t* v;
    uint32_t k_page, v_page;    // below 2^31 (bytes in 32 bits)
    int32_t k_token, v_token;   // a page of one head spans less than 2^30
    int64_t k_head, v_head;
    const uint16_t* q;
    int64_t q_row, q_token, q_head;
    uint16_t* o;
    float* lse;
    const uint16_t* nk;
    const uint16_t* nv;
    int64_t nk_row, nk_token, nk_head;
    int64_t nv_row, nv_token, nv_head;
    float* ws;
};

// Offset i of the packed sequences, clamped into [0, T].
__device__ __forceinline__ int paged_cu(const PagedParams& p, int i) {
    typedef __attribute__((address_space(4))) const int64_t c_i64;
    typedef __attribute__((address_space(4))) const int32_t c_i32;
    const int64_t x = p.cu_i64 ? ((c_i64*)p.cu_seqlens)[i] : (int64_t)((c_i32*)p.cu_seqlens)[i];
    return (int)(x < 0 ? 0 : (x > p.T ? p.T : x));
}

// The new tokens of sequence n: `count` of them, the first at token index
// `first` of its batch row (packed: of the one row) and at position `pos` of
// the sequence; `len` cached tokens (no more than the table's row holds).
struct NewTokens {
    int first, count, len, pos;
};
__device__ __forceinline__ NewTokens new_tokens(const PagedParams& p, int n) {
    NewTokens s;
    const int64_t most = (int64_t)p.M << p.page_shift;
    const int len = p.seq_lens[n];
    s.len = len < 0 ? 0 : ((int64_t)len > most ? (int)most : len);
    s.first = 0;
    s.count = p.T;
    if (p.cu_seqlens) {
        s.first = paged_cu(p, n);
        s.count = max(0, paged_cu(p, n + 1) - s.first);
    }
    s.pos = s.len - s.count;
    return s;
}

// Entry i of sequence n's row of the page table: the last one for any i past
// it.  A page only if is_page().
__device__ __forceinline__ int table_entry(const PagedParams& p, int n, int i) {
    typedef __attribute__((address_space(4))) const int32_t c_i32;
    return ((c_i32*)(p.page_table + (int64_t)n * p.table_stride))[i < p.M ? i : p.M - 1];
}
__device__ __forceinline__ bool is_page(const PagedParams& p, int x) { return (unsigned)x < (unsigned)p.P; }

// Inclusive prefix sum over the wave's lanes: within each 16 by DPP row_shr,
// then the last lane of one row to the next row or half (row_bcast 15, 31).
__device__ __forceinline__ uint32_t wave_prefix(uint32_t x) {
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);
    return x;
}

// The same with sums above `most` (below 2^31, as is every x) taken as `most`.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t x, uint32_t most) {
    x = min(x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false), most);
    x = min(x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false), most);
    x = min(x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false), most);
    x = min(x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false), most);
    x = min(x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false), most);
    x = min(x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false), most);
    return x;
}

// Pools and counts of a call on the pages (kda_paged_hip.h).
struct PagesParams {
    int N, M, P, F, page_shift;
    int num_pools;
    KdaPagePool pools[KDA_PAGED_MAX_POOLS];
    int32_t* table;
    int64_t table_stride;
    int32_t* lens;
    int32_t* refs;
    const int32_t* src;
    const int32_t* dst;
    const int32_t* more;
    uint8_t* ok;
    int32_t* out_table;
    int32_t* out_refs;
    int32_t* out_live;
    int32_t* ws;
};

size_t paged_attn_workspace(const PagedParams& p, int D);
hipError_t launch_paged_attn(const PagedParams& p, int D, hipStream_t stream);
hipError_t launch_paged_append(const PagedParams& p, int D, hipStream_t stream);
hipError_t launch_pages_reserve(const PagesParams& p, hipStream_t stream);
hipError_t launch_pages_free(const PagesParams& p, hipStream_t stream);
hipError_t launch_pages_fork(const PagesParams& p, hipStream_t stream);
hipError_t launch_pages_copy(const PagesParams& p, hipStream_t stream);
hipError_t launch_pages_compact(const PagesParams& p, hipStream_t stream);

}  // namespace kda
