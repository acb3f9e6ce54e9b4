/*
 * kda_paged_hip.h -- C ABI of libkda_bt16_hip.so for a paged cache of keys
 * and values: attention of new tokens over it, the append of their keys and
 * values (with the position rotation), and the work on its pages (reserve,
 * free, fork, compact, copy).
 *
 * For models that alternate KDA layers with softmax-attention layers: the
 * KDA layers keep a state of fixed size, the attention layers this cache.
 * No counterpart in the reference, which has no attention cache.  Every
 * call is asynchronous on the caller's HIP stream, returns 0 or a negative
 * KDA_BT16_E* code (kda_bt16_strerror), allocates nothing and reads no
 * device memory on the host.
 *
 * The cache of a layer:
 *   k, v        [P, page_size, HKV, D]  bf16 or fp16, P pages of page_size
 *                                       tokens; page, token and head strides
 *                                       are given in elements, multiples of
 *                                       8, a token's stride at least D
 *   page_table  [N, M] int32            the pages of each sequence in order,
 *                                       from the first entry on (row stride
 *                                       given), -1: none
 *   seq_lens    [N] int32               cached tokens of each sequence, those
 *                                       of the call included
 *   page_refs   [P] int32               how many sequences hold each page; 0:
 *                                       free
 * The new tokens of a call are [N, T, heads, D], or with cu_seqlens ([N + 1]
 * int32 or int64, from 0 to T, non-decreasing) T tokens of N sequences packed
 * one after another.  Sequence n's new tokens are its last ones: token i of
 * T_n sits at position seq_lens[n] - T_n + i.  Lowering seq_lens[n] takes the
 * last tokens back, those of a rejected draft: the pages behind the new length
 * stay the row's until it grows into them or ends.  It must not become shorter
 * than what it shares with a fork, whose page its next tokens would go into.
 *
 * Table entries outside [0, P), lengths beyond M * page_size, offsets outside
 * [0, T] and row numbers outside [0, N), or offsets that decrease, give
 * unspecified results but never an access outside the tensors.
 */
#ifndef KDA_PAGED_HIP_H
#define KDA_PAGED_HIP_H

#include "kda_bt16_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KDA_PAGED_ABI_VERSION 1

/* Element types of the cache and of the new tokens. */
#define KDA_PAGED_BF16 0
#define KDA_PAGED_FP16 1

/* kda_paged_attn_hip: a query sees the keys up to its own position only. */
#define KDA_PAGED_CAUSAL (1u << 0)

typedef struct KdaPagedArgs {
    int32_t abi_version;  /* KDA_PAGED_ABI_VERSION */
    int32_t N;            /* sequences */
    int32_t T;            /* new tokens a sequence; with cu_seqlens all of them */
    int32_t HQ;           /* query heads, a multiple of HKV (attention) */
    int32_t HKV;          /* heads of the cache */
    int32_t D;            /* 64 or 128 */
    int32_t dtype;        /* KDA_PAGED_BF16 or KDA_PAGED_FP16 */
    int32_t P;            /* pages */
    int32_t page_size;    /* tokens a page: a power of two, 16 to 1024 */
    int32_t M;            /* entries a row of the page table */
    uint32_t flags;
    int32_t window;       /* a query at position p sees keys above p - window; 0: no window */
    float scale;          /* of the scores, above 0 */
    int32_t cu_seqlens_dtype; /* KDA_BT16_DTYPE_I32 or KDA_BT16_DTYPE_I64 */
    const void* cu_seqlens;   /* optional */
    const int32_t* page_table;
    int64_t table_stride;     /* elements between rows of page_table */
    const int32_t* seq_lens;
    void* k;                  /* the cache; 16-byte aligned */
    void* v;
    int64_t k_page, k_token, k_head; /* strides in elements */
    int64_t v_page, v_token, v_head;
    /* Attention: the queries and the outputs.  Append: new_k, new_v. */
    const void* q;            /* 16-byte aligned; strides multiples of 8 */
    int64_t q_row, q_token, q_head; /* q_row: between batch rows (unused with cu_seqlens) */
    void* o;                  /* [N, T, HQ, D] (packed: [T, HQ, D]), contiguous */
    float* lse;               /* optional [N, T, HQ] (packed: [T, HQ]): natural log */
    const void* new_k;        /* [N, T, HKV, D] by the strides below */
    const void* new_v;
    int64_t nk_row, nk_token, nk_head;
    int64_t nv_row, nv_token, nv_head;
    void* workspace;          /* attention: kda_paged_attn_workspace_bytes() bytes, 256-byte aligned */
    size_t workspace_bytes;
} KdaPagedArgs;

/* o = softmax(scale * q k^T) v over the cached keys each query sees, query
 * head h reading the cache's head h / (HQ / HKV); lse = log of the sum of
 * the exponentials.  A query that sees no key has o = 0 and lse = -inf; one
 * with a score of NaN or +inf has NaN in both, and the other queries' results
 * stay as they are.  What the pages hold at and beyond seq_lens is not read into the
 * result, whatever it is; the keys and values before it have to be finite. */
size_t kda_paged_attn_workspace_bytes(const KdaPagedArgs* args);
int kda_paged_attn_hip(const KdaPagedArgs* args, void* stream);

/* The same with a window (which has to be given, and the causal flag) and the
 * first `sinks` tokens of every sequence visible outside of it too: a query at
 * position p sees the keys j <= p with j > p - window or j < sinks. */
typedef struct KdaPagedSinksArgs {
    KdaPagedArgs paged;
    int32_t sinks;  /* 0 or more */
    int32_t reserved;
} KdaPagedSinksArgs;
size_t kda_paged_attn_sinks_workspace_bytes(const KdaPagedSinksArgs* args);
int kda_paged_attn_sinks_hip(const KdaPagedSinksArgs* args, void* stream);

/* kda_paged_attn_hip (causal, no window) for sequences in groups that share
 * their first tokens, which are read and worked on once for a group: rows
 * cu_groups[g] to cu_groups[g + 1] - 1 of the table hold the same keys and values
 * in their first shared_lens[g] tokens, in the same pages (as kda_pages_fork_hip
 * leaves them) or in copies; one row's are read.  Which one, and how sums are
 * rounded, depends on the groups, nothing else does.  A sequence whose new tokens
 * do not all come behind the shared ones (an ended one's) is worked on by itself,
 * and so are rows of no group, and sequences whose new tokens fill a row tile
 * (T_n * HQ / HKV at least 128), which have nothing to gain.  Beyond 2048 sequences
 * or 2048 groups, mostly where every sequence has more than 128 rows (without
 * cu_seqlens), and where the table's rows are short (paged_attention_shared() in
 * Python says how short), all are worked on one by one, as by kda_paged_attn_hip. */
typedef struct KdaPagedSharedArgs {
    KdaPagedArgs paged;
    const int32_t* cu_groups;   /* [num_groups + 1], from 0 to N, non-decreasing */
    const int32_t* shared_lens; /* [num_groups] */
    int32_t num_groups;
    int32_t reserved;
} KdaPagedSharedArgs;
size_t kda_paged_attn_shared_workspace_bytes(const KdaPagedSharedArgs* args);
int kda_paged_attn_shared_hip(const KdaPagedSharedArgs* args, void* stream);

/* The new tokens' keys and values into their places in the pages.  Tokens at
 * negative positions, beyond the table or on no page are left out. */
int kda_paged_append_hip(const KdaPagedArgs* args, void* stream);

/* The append with the position rotation on the way, and the queries' with it. */
typedef struct KdaPagedRotaryArgs {
    KdaPagedArgs paged;     /* as for the append; q and its strides: the queries, HQ heads (any number) */
    const float* inv_freq;  /* [rotary_dim / 2] fp32: angle per position of each pair */
    int32_t rotary_dim;     /* elements of a head that are turned, the first: a multiple of 16, 16 to D */
    int32_t interleaved;    /* 0: pairs (i, i + rotary_dim / 2); else (2 i, 2 i + 1) */
    void* q_out;            /* [N, T, HQ, D] by the strides below; q itself (with q's strides) or apart from it */
    int64_t out_row, out_token, out_head;
} KdaPagedRotaryArgs;

/* A pair (a, b) of the token at position p becomes (a cos x - b sin x,
 * b cos x + a sin x), x = p * inv_freq of the pair, in every head of the
 * queries (to q_out) and of the new keys (into their places in the pages); the
 * values go into theirs as they are.  Tokens that the append leaves out have
 * their queries turned all the same, by their positions; tokens of no sequence
 * (packed, before the first offset or behind the last) are left as they are. */
int kda_paged_append_rotary_hip(const KdaPagedRotaryArgs* args, void* stream);

#define KDA_PAGED_MAX_POOLS 8

/* A pool: [lead, P, ...] contiguous, `page_bytes` a page (a multiple of 16),
 * 16-byte aligned; `lead` counts layers, keys and values. */
typedef struct KdaPagePool {
    void* data;
    int64_t lead;
    int64_t page_bytes;
} KdaPagePool;

typedef struct KdaPagesArgs {
    int32_t abi_version;  /* KDA_PAGED_ABI_VERSION */
    int32_t N;            /* rows of the page table */
    int32_t M;            /* entries a row */
    int32_t P;            /* pages (rows of the pools); with page_refs below 2^31 - 2^16 */
    int32_t page_size;    /* tokens a page, a power of two, 16 to 1024 */
    int32_t F;            /* rows to free or fork, pages to copy */
    int32_t num_pools;
    int32_t reserved;
    KdaPagePool pools[KDA_PAGED_MAX_POOLS];
    int32_t* page_table;
    int64_t table_stride;
    int32_t* seq_lens;
    int32_t* page_refs;
    const int32_t* src;        /* fork: rows; copy: pages */
    const int32_t* dst;        /* fork and free: rows; copy: pages */
    const int32_t* new_tokens; /* reserve: [N] */
    uint8_t* ok;               /* reserve: [N], fork: [F]; 1 where it was done */
    int32_t* out_table;        /* compact: [N, M] contiguous */
    int32_t* out_refs;         /* compact: [P] */
    int32_t* out_live;         /* compact: [1] */
    void* workspace;           /* compact: kda_pages_workspace_bytes() bytes, 256-byte aligned */
    size_t workspace_bytes;
} KdaPagesArgs;

/* Workspace of kda_pages_compact_hip (P read). */
size_t kda_pages_workspace_bytes(const KdaPagesArgs* args);

/* Room for new_tokens[n] more tokens of every sequence n: first the held pages
 * that follow its tokens' in its row, then the lowest free pages, in the
 * sequences' order, until they run out; seq_lens grows by as many.  A sequence whose pages cannot all be had, or do not fit its row,
 * keeps what it has and its ok is 0.  Once pages could not all be had, so is
 * every later one's that needs a page. */
int kda_pages_reserve_hip(const KdaPagesArgs* args, void* stream);

/* Rows dst[0..F) become empty: their pages lose one holder each, their
 * entries become -1, their lengths 0.  A row named twice is freed once. */
int kda_pages_free_hip(const KdaPagesArgs* args, void* stream);

/* Row dst[i] (new or freed, named once) becomes a copy of row src[i]: whole pages
 * are shared, the tokens of a last partial page are copied, in every pool, to
 * the lowest free page not taken by an earlier fork.  Without a free page the
 * row stays empty and ok[i] is 0.  No row is in src and in dst. */
int kda_pages_fork_hip(const KdaPagesArgs* args, void* stream);

/* Pages dst[i] of every pool become copies of pages src[i]; pairs outside
 * [0, P) are left out.  No page is in src and in dst, or in dst twice. */
int kda_pages_copy_hip(const KdaPagesArgs* args, void* stream);

/* Moves the held pages into the first `live` places of every pool, live
 * being their number: the i-th held page at or above live goes to the i-th
 * free place below it.  out_table, out_refs and out_live are the new table,
 * counts and number.  page_table and page_refs stay as they are, and the
 * pages moved away from keep their contents: a launch that still reads by the
 * old table stays right until those pages are handed out again. */
int kda_pages_compact_hip(const KdaPagesArgs* args, void* stream);

/* KDA_PAGED_ABI_VERSION of the built library. */
int kda_paged_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* KDA_PAGED_HIP_H */
