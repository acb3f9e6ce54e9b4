// C ABI of the paged cache (include/kda_paged_hip.h): argument checks and
// launches.  The checks guard the kernels' indexing (sizes, strides,
// alignment, pointers, 32-bit offsets and grids); user-facing validation with
// its messages lives in the Python layer.
#include "kda_paged.h"

namespace {

using kda::PagedParams;
using kda::PagesParams;
using kda::SharedParams;
using kda::SinkParams;

constexpr int64_t I32_MAX = 0x7fffffffLL;

bool misaligned(const void* p, uintptr_t align) {
    return (reinterpret_cast<uintptr_t>(p) & (align - 1)) != 0;
}

// log2 of a page size the kernels take (a power of two from 16 to 1024), else -1.
int page_shift_of(int32_t page_size) {
    for (int s = 4; s <= 10; ++s)
        if (page_size == 1 << s) return s;
    return -1;
}

// Strides that keep 16-byte accesses aligned and never step backwards.
bool strides_ok(int64_t a, int64_t b, int64_t c) {
    return a >= 0 && b >= 0 && c >= 0 && a % 8 == 0 && b % 8 == 0 && c % 8 == 0;
}

// A page of one head, read through a buffer descriptor of 32-bit size.
bool page_span_ok(const KdaPagedArgs* a, int64_t token) {
    return token >= a->D && ((int64_t)(a->page_size - 1) * token + a->D) * 2 <= I32_MAX;
}

int paged_params(const KdaPagedArgs* a, PagedParams& p) {
    if (a == nullptr) return KDA_BT16_EINVAL;
    if (a->abi_version != KDA_PAGED_ABI_VERSION) return KDA_BT16_EABI;
    if (a->N <= 0 || a->T <= 0 || a->HKV <= 0 || a->P <= 0 || a->M <= 0) return KDA_BT16_EINVAL;
    if (a->D != 64 && a->D != 128) return KDA_BT16_EUNSUPPORTED;
    const int shift = page_shift_of(a->page_size);
    if (shift < 0) return KDA_BT16_EUNSUPPORTED;
    if (a->dtype != KDA_PAGED_BF16 && a->dtype != KDA_PAGED_FP16) return KDA_BT16_EINVAL;
    if (a->cu_seqlens) {
        const bool i64 = a->cu_seqlens_dtype == KDA_BT16_DTYPE_I64;
        if (!i64 && a->cu_seqlens_dtype != KDA_BT16_DTYPE_I32) return KDA_BT16_EINVAL;
        if (misaligned(a->cu_seqlens, i64 ? 8 : 4)) return KDA_BT16_EINVAL;
    }
    if (!a->page_table || !a->seq_lens || !a->k || !a->v) return KDA_BT16_EINVAL;
    if (misaligned(a->page_table, 4) || misaligned(a->seq_lens, 4) || misaligned(a->k, 16) || misaligned(a->v, 16))
        return KDA_BT16_EINVAL;
    if (a->table_stride < a->M) return KDA_BT16_EINVAL;
    if (!strides_ok(a->k_page, a->k_token, a->k_head) || !strides_ok(a->v_page, a->v_token, a->v_head))
        return KDA_BT16_EINVAL;
    if (!page_span_ok(a, a->k_token) || !page_span_ok(a, a->v_token)) return KDA_BT16_EUNSUPPORTED;
    if (a->k_page > I32_MAX || a->v_page > I32_MAX) return KDA_BT16_EUNSUPPORTED;
    // Positions are 32-bit.
    if (((int64_t)a->M << shift) > I32_MAX / 2) return KDA_BT16_EUNSUPPORTED;

    p = PagedParams{};
    p.N = a->N;
    p.T = a->T;
    p.HQ = a->HQ;
    p.HKV = a->HKV;
    p.P = a->P;
    p.page_shift = shift;
    p.M = a->M;
    p.causal = (a->flags & KDA_PAGED_CAUSAL) != 0;
    p.window = a->window < I32_MAX / 2 ? a->window : (int32_t)(I32_MAX / 2);  // (more than any position)
    p.fp16 = a->dtype == KDA_PAGED_FP16;
    p.cu_i64 = a->cu_seqlens_dtype == KDA_BT16_DTYPE_I64;
    p.scale = a->scale;
    p.cu_seqlens = a->cu_seqlens;
    p.page_table = a->page_table;
    p.table_stride = a->table_stride;
    p.seq_lens = a->seq_lens;
    p.k = static_cast<uint16_t*>(a->k);
    p.v = static_cast<uint16_t*>(a->v);
    p.k_page = (uint32_t)a->k_page;
    p.k_token = (int32_t)a->k_token;
    p.k_head = a->k_head;
    p.v_page = (uint32_t)a->v_page;
    p.v_token = (int32_t)a->v_token;
    p.v_head = a->v_head;
    return KDA_BT16_OK;
}

int attn_params(const KdaPagedArgs* a, PagedParams& p) {
    const int rc = paged_params(a, p);
    if (rc != KDA_BT16_OK) return rc;
    if (a->HQ <= 0 || a->HQ % a->HKV != 0) return KDA_BT16_EINVAL;
    if (a->window < 0 || !(a->scale > 0.0f)) return KDA_BT16_EINVAL;
    if (a->window > 0 && !p.causal) return KDA_BT16_EUNSUPPORTED;
    // Tiles of 32 keys of all sequences and heads (with up to as many again to
    // fill pieces), rows (token, head of a group) and work-groups are counted in
    // 32 bits.
    const int64_t tiles = ((((int64_t)a->M * a->page_size) >> 5) + 2) * a->HKV;
    if (tiles > I32_MAX / a->N) return KDA_BT16_EUNSUPPORTED;
    const int64_t tokens = a->cu_seqlens ? a->T : (int64_t)a->N * a->T;
    if ((tokens + (int64_t)a->N * 128) * a->HQ > I32_MAX / 4) return KDA_BT16_EUNSUPPORTED;
    if (!a->q || !a->o) return KDA_BT16_EINVAL;
    if (misaligned(a->q, 16) || misaligned(a->o, 16) || misaligned(a->lse, 4)) return KDA_BT16_EINVAL;
    if (!strides_ok(a->q_row, a->q_token, a->q_head)) return KDA_BT16_EINVAL;
    p.G = a->HQ / a->HKV;
    p.q = static_cast<const uint16_t*>(a->q);
    p.q_row = a->q_row;
    p.q_token = a->q_token;
    p.q_head = a->q_head;
    p.o = static_cast<uint16_t*>(a->o);
    p.lse = a->lse;
    return KDA_BT16_OK;
}

int append_params(const KdaPagedArgs* a, PagedParams& p) {
    const int rc = paged_params(a, p);
    if (rc != KDA_BT16_OK) return rc;
    if (!a->new_k || !a->new_v || misaligned(a->new_k, 16) || misaligned(a->new_v, 16)) return KDA_BT16_EINVAL;
    if (!strides_ok(a->nk_row, a->nk_token, a->nk_head) || !strides_ok(a->nv_row, a->nv_token, a->nv_head))
        return KDA_BT16_EINVAL;
    const int64_t tokens = a->cu_seqlens ? a->T : (int64_t)a->N * a->T;
    // one thread for each 16 bytes of a token's keys
    if (tokens > I32_MAX / 16 / a->HKV) return KDA_BT16_EUNSUPPORTED;
    p.nk = static_cast<const uint16_t*>(a->new_k);
    p.nv = static_cast<const uint16_t*>(a->new_v);
    p.nk_row = a->nk_row;
    p.nk_token = a->nk_token;
    p.nk_head = a->nk_head;
    p.nv_row = a->nv_row;
    p.nv_token = a->nv_token;
    p.nv_head = a->nv_head;
    return KDA_BT16_OK;
}

enum Need { POOLS = 1, TABLE = 2, REFS = 4, SRC = 8, DST = 16, WS = 32 };

int pages_params(const KdaPagesArgs* a, PagesParams& p, unsigned need) {
    if (a == nullptr) return KDA_BT16_EINVAL;
    if (a->abi_version != KDA_PAGED_ABI_VERSION) return KDA_BT16_EABI;
    if (a->P <= 0 || a->F < 0) return KDA_BT16_EINVAL;
    p = PagesParams{};
    p.P = a->P;
    p.F = a->F;
    if (need & POOLS) {
        if (a->num_pools <= 0 || a->num_pools > KDA_PAGED_MAX_POOLS) return KDA_BT16_EINVAL;
        for (int i = 0; i < a->num_pools; ++i) {
            const KdaPagePool& x = a->pools[i];
            if (!x.data || misaligned(x.data, 16) || x.lead <= 0 || x.page_bytes <= 0 || x.page_bytes % 16 != 0)
                return KDA_BT16_EINVAL;
            p.pools[i] = x;
        }
        p.num_pools = a->num_pools;
    }
    if (need & TABLE) {
        if (a->N <= 0 || a->M <= 0 || !a->page_table || misaligned(a->page_table, 4) || a->table_stride < a->M)
            return KDA_BT16_EINVAL;
        p.N = a->N;
        p.M = a->M;
        p.table = a->page_table;
        p.table_stride = a->table_stride;
    }
    if (need & REFS) {
        if (!a->page_refs || misaligned(a->page_refs, 16)) return KDA_BT16_EINVAL;
        // (the steps over the counts form numbers up to 2^15 past the last page)
        if (a->P > I32_MAX - (1 << 16)) return KDA_BT16_EUNSUPPORTED;
        p.refs = a->page_refs;
    }
    if ((need & SRC) && a->F > 0 && (!a->src || misaligned(a->src, 4))) return KDA_BT16_EINVAL;
    if ((need & DST) && a->F > 0 && (!a->dst || misaligned(a->dst, 4))) return KDA_BT16_EINVAL;
    p.src = a->src;
    p.dst = a->dst;
    if (need & WS) {
        if (!a->workspace || misaligned(a->workspace, 256) || a->workspace_bytes < kda_pages_workspace_bytes(a))
            return KDA_BT16_EWORKSPACE;
        p.ws = static_cast<int32_t*>(a->workspace);
    }
    return KDA_BT16_OK;
}

// Lengths, for the calls that read or change them.
int pages_lens(const KdaPagesArgs* a, PagesParams& p) {
    if (!a->seq_lens || misaligned(a->seq_lens, 4)) return KDA_BT16_EINVAL;
    p.lens = a->seq_lens;
    p.page_shift = page_shift_of(a->page_size);
    if (p.page_shift < 0 || ((int64_t)a->M << p.page_shift) > I32_MAX / 2) return KDA_BT16_EUNSUPPORTED;
    return KDA_BT16_OK;
}

int sink_params(const KdaPagedSinksArgs* a, SinkParams& p) {
    if (a == nullptr) return KDA_BT16_EINVAL;
    const int rc = attn_params(&a->paged, p);
    if (rc != KDA_BT16_OK) return rc;
    if (a->sinks < 0) return KDA_BT16_EINVAL;
    if (p.window == 0) return KDA_BT16_EUNSUPPORTED;  // (without one every key is visible)
    p.sinks = a->sinks < I32_MAX / 2 ? a->sinks : (int32_t)(I32_MAX / 2);
    return KDA_BT16_OK;
}

int shared_params(const KdaPagedSharedArgs* a, SharedParams& p) {
    if (a == nullptr) return KDA_BT16_EINVAL;
    const int rc = attn_params(&a->paged, p);
    if (rc != KDA_BT16_OK) return rc;
    if (!p.causal || p.window != 0) return KDA_BT16_EUNSUPPORTED;
    if (a->num_groups <= 0 || !a->cu_groups || !a->shared_lens || misaligned(a->cu_groups, 4) ||
        misaligned(a->shared_lens, 4))
        return KDA_BT16_EINVAL;
    p.NG = a->num_groups;
    p.cu_groups = a->cu_groups;
    p.shared_lens = a->shared_lens;
    return KDA_BT16_OK;
}

int launched(hipError_t e) { return e == hipSuccess ? KDA_BT16_OK : KDA_BT16_ELAUNCH; }

template <class P>
int attn_launch(const KdaPagedArgs* a, P& p, void* stream) {
    const size_t need = kda::paged_attn_workspace(p, a->D);
    if (need > 0) {
        if (!a->workspace || misaligned(a->workspace, 256) || a->workspace_bytes < need) return KDA_BT16_EWORKSPACE;
        p.ws = static_cast<float*>(a->workspace);
    }
    return launched(kda::launch_paged_attn(p, a->D, static_cast<hipStream_t>(stream)));
}

}  // namespace

extern "C" {

size_t kda_paged_attn_workspace_bytes(const KdaPagedArgs* args) {
    PagedParams p;
    return attn_params(args, p) == KDA_BT16_OK ? kda::paged_attn_workspace(p, args->D) : 0;
}

int kda_paged_attn_hip(const KdaPagedArgs* args, void* stream) {
    PagedParams p;
    const int rc = attn_params(args, p);
    return rc == KDA_BT16_OK ? attn_launch(args, p, stream) : rc;
}

size_t kda_paged_attn_sinks_workspace_bytes(const KdaPagedSinksArgs* args) {
    SinkParams p{};
    return sink_params(args, p) == KDA_BT16_OK ? kda::paged_attn_workspace(p, args->paged.D) : 0;
}

int kda_paged_attn_sinks_hip(const KdaPagedSinksArgs* args, void* stream) {
    SinkParams p{};
    const int rc = sink_params(args, p);
    return rc == KDA_BT16_OK ? attn_launch(&args->paged, p, stream) : rc;
}

size_t kda_paged_attn_shared_workspace_bytes(const KdaPagedSharedArgs* args) {
    SharedParams p{};
    return shared_params(args, p) == KDA_BT16_OK ? kda::paged_attn_workspace(p, args->paged.D) : 0;
}

int kda_paged_attn_shared_hip(const KdaPagedSharedArgs* args, void* stream) {
    SharedParams p{};
    const int rc = shared_params(args, p);
    return rc == KDA_BT16_OK ? attn_launch(&args->paged, p, stream) : rc;
}

int kda_paged_append_hip(const KdaPagedArgs* args, void* stream) {
    PagedParams p;
    const int rc = append_params(args, p);
    if (rc != KDA_BT16_OK) return rc;
    return launched(kda::launch_paged_append(p, args->D, static_cast<hipStream_t>(stream)));
}

int kda_paged_append_rotary_hip(const KdaPagedRotaryArgs* args, void* stream) {
    if (args == nullptr) return KDA_BT16_EINVAL;
    const KdaPagedArgs* a = &args->paged;
    kda::RotaryParams p{};
    const int rc = append_params(a, p);
    if (rc != KDA_BT16_OK) return rc;
    if (a->HQ <= 0 || !a->q || !args->q_out || !args->inv_freq) return KDA_BT16_EINVAL;
    if (misaligned(a->q, 16) || misaligned(args->q_out, 16) || misaligned(args->inv_freq, 4)) return KDA_BT16_EINVAL;
    if (!strides_ok(a->q_row, a->q_token, a->q_head) ||
        !strides_ok(args->out_row, args->out_token, args->out_head))
        return KDA_BT16_EINVAL;
    if (args->rotary_dim < 16 || args->rotary_dim > a->D || args->rotary_dim % 16 != 0) return KDA_BT16_EUNSUPPORTED;
    const int64_t tokens = a->cu_seqlens ? a->T : (int64_t)a->N * a->T;
    // one thread for each 16 elements of a token
    if (((int64_t)a->HQ + 2 * (int64_t)a->HKV) > I32_MAX / 16 / tokens) return KDA_BT16_EUNSUPPORTED;
    p.q = static_cast<const uint16_t*>(a->q);
    p.q_row = a->q_row;
    p.q_token = a->q_token;
    p.q_head = a->q_head;
    p.inv_freq = args->inv_freq;
    p.units = args->rotary_dim / 16;
    p.interleaved = args->interleaved;
    p.q_out = static_cast<uint16_t*>(args->q_out);
    p.out_row = args->out_row;
    p.out_token = args->out_token;
    p.out_head = args->out_head;
    return launched(kda::launch_paged_append_rotary(p, a->D, static_cast<hipStream_t>(stream)));
}

size_t kda_pages_workspace_bytes(const KdaPagesArgs* args) {
    if (args == nullptr || args->abi_version != KDA_PAGED_ABI_VERSION || args->P <= 0) return 0;
    // three lists of pages and the counts of each 4096 (kda_pages.hip)
    const int64_t P = args->P, ints = 3 * P + P / 4096 + 2;
    return (size_t)((ints * 4 + 255) / 256 * 256);
}

int kda_pages_reserve_hip(const KdaPagesArgs* args, void* stream) {
    PagesParams p;
    int rc = pages_params(args, p, TABLE | REFS);
    if (rc == KDA_BT16_OK) rc = pages_lens(args, p);
    if (rc != KDA_BT16_OK) return rc;
    if (!args->new_tokens || misaligned(args->new_tokens, 4) || !args->ok) return KDA_BT16_EINVAL;
    p.more = args->new_tokens;
    p.ok = args->ok;
    return launched(kda::launch_pages_reserve(p, static_cast<hipStream_t>(stream)));
}

int kda_pages_free_hip(const KdaPagesArgs* args, void* stream) {
    PagesParams p;
    int rc = pages_params(args, p, TABLE | REFS | DST);
    if (rc == KDA_BT16_OK) rc = pages_lens(args, p);
    if (rc != KDA_BT16_OK) return rc;
    if (p.F == 0) return KDA_BT16_OK;
    return launched(kda::launch_pages_free(p, static_cast<hipStream_t>(stream)));
}

int kda_pages_fork_hip(const KdaPagesArgs* args, void* stream) {
    PagesParams p;
    int rc = pages_params(args, p, POOLS | TABLE | REFS | SRC | DST);
    if (rc == KDA_BT16_OK) rc = pages_lens(args, p);
    if (rc != KDA_BT16_OK) return rc;
    if (p.F == 0) return KDA_BT16_OK;
    if (!args->ok) return KDA_BT16_EINVAL;
    p.ok = args->ok;
    return launched(kda::launch_pages_fork(p, static_cast<hipStream_t>(stream)));
}

int kda_pages_copy_hip(const KdaPagesArgs* args, void* stream) {
    PagesParams p;
    const int rc = pages_params(args, p, POOLS | SRC | DST);
    if (rc != KDA_BT16_OK) return rc;
    if (p.F == 0) return KDA_BT16_OK;
    return launched(kda::launch_pages_copy(p, static_cast<hipStream_t>(stream)));
}

int kda_pages_compact_hip(const KdaPagesArgs* args, void* stream) {
    PagesParams p;
    const int rc = pages_params(args, p, POOLS | TABLE | REFS | WS);
    if (rc != KDA_BT16_OK) return rc;
    if (!args->out_table || !args->out_refs || !args->out_live || misaligned(args->out_table, 4) ||
        misaligned(args->out_refs, 4) || misaligned(args->out_live, 4))
        return KDA_BT16_EINVAL;
    if ((int64_t)p.N * p.M > I32_MAX) return KDA_BT16_EUNSUPPORTED;
    p.out_table = args->out_table;
    p.out_refs = args->out_refs;
    p.out_live = args->out_live;
    return launched(kda::launch_pages_compact(p, static_cast<hipStream_t>(stream)));
}

int kda_paged_abi_version(void) { return KDA_PAGED_ABI_VERSION; }

}  // extern "C"
