// The pages of a cache (kda_paged_hip.h): append of new tokens, reserve, free,
// fork, copy and compact.
//
// Which pages are free is what page_refs says and nothing else: a page with
// no holder is free, and every call hands out the lowest free pages.  So no
// list has to be kept, and results do not depend on the order in which
// work-groups run.
#include "kda_common.h"
#include "kda_paged.h"

#include <algorithm>

namespace kda {
namespace {

// ---- append ----

// The sequence of packed token t: the largest n with cu[n] <= t.
__device__ __forceinline__ int sequence_of(const PagedParams& p, int t) {
    int lo = 0, hi = p.N - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (paged_cu(p, mid) <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// One thread moves 16 bytes of a token's keys and the same of its values: as
// many threads as there are pieces, since what bounds it is the chain of loads
// before them (sequence, length, table entry).  128 tokens of 8 heads 3.2 us on
// the GPU, 1024 packed in 16 sequences (9.5 MB each way) 6.1.
template <int D>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedParams p, int total) {
    constexpr int PIECES = D / 8;
    const int id = blockIdx.x * 256 + threadIdx.x;
    if (id >= total) return;
    const int piece = id % PIECES, x = id / PIECES;
    const int h = x % p.HKV, t = x / p.HKV;
    const int n = p.cu_seqlens ? sequence_of(p, t) : t / p.T;
    const NewTokens s = new_tokens(p, n);
    const int tok = p.cu_seqlens ? t - s.first : t - n * p.T;
    const int pos = s.pos + tok;
    if (tok < 0 || tok >= s.count || pos < 0) return;
    const int64_t page = table_entry(p, n, pos >> p.page_shift);
    if (!is_page(p, (int)page)) return;
    const int in = pos & ((1 << p.page_shift) - 1);
    const int64_t row = p.cu_seqlens ? 0 : n, at = p.cu_seqlens ? t : tok;
    const u32x4 k = *reinterpret_cast<const u32x4*>(p.nk + row * p.nk_row + at * p.nk_token + h * p.nk_head + 8 * piece);
    const u32x4 v = *reinterpret_cast<const u32x4*>(p.nv + row * p.nv_row + at * p.nv_token + h * p.nv_head + 8 * piece);
    *reinterpret_cast<u32x4*>(p.k + page * p.k_page + (int64_t)in * p.k_token + h * p.k_head + 8 * piece) = k;
    *reinterpret_cast<u32x4*>(p.v + page * p.v_page + (int64_t)in * p.v_token + h * p.v_head + 8 * piece) = v;
}

// ---- scans ----

// Exclusive prefix sum over the work-group's threads, and the total.
template <int THREADS>
__device__ __forceinline__ int block_scan(int x, int* lds, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int inc = wave_prefix(x);
    __syncthreads();
    if (lane == 63) lds[wave] = inc;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        const int y = lds[w];
        before += w < wave ? y : 0;
        total += y;
    }
    return before + inc - x;
}

// Exclusive prefix sum over the work-group's threads, and the total, of numbers
// up to `most` (below 2^31), sums above it taken as `most`.
template <int THREADS>
__device__ __forceinline__ uint32_t block_scan_upto(uint32_t x, uint32_t most, int* lds, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t inc = wave_prefix(x, most);
    __syncthreads();
    if (lane == 63) lds[wave] = (int)inc;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w == wave) before = total;
        total = min(total + (uint32_t)lds[w], most);
    }
    // (the lane before's: a sum that was cut off says nothing about its parts)
    const uint32_t last = __shfl_up(inc, 1);
    return min(before + (lane == 0 ? 0u : last), most);
}

__device__ __forceinline__ int pages_for(int tokens, int shift) {
    return tokens <= 0 ? 0 : (int)(((int64_t)tokens + (1 << shift) - 1) >> shift);
}

// Four counts from page `i` on (i a multiple of 4); beyond the last: held.
__device__ __forceinline__ void read_refs(const PagesParams& p, int i, int (&r)[4]) {
    if (i + 4 <= p.P) {
        const int4 x = *reinterpret_cast<const int4*>(p.refs + i);
        r[0] = x.x; r[1] = x.y; r[2] = x.z; r[3] = x.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = i + j < p.P ? p.refs[i + j] : 1;
    }
}

// Free pages from `from` on in rising order, by a whole work-group: calls
// take(rank, page) for the first `want` of them (rank from 0) and returns how
// many there are, at most `want`; `next`: where a later search goes on.
template <int THREADS, class Take>
__device__ __forceinline__ int find_free(const PagesParams& p, int from, int want, int* lds, int& next, Take take) {
    constexpr int EACH = 4, STEP = THREADS * 4 * EACH;  // pages a thread and turn: 16, read together
    int found = 0;
    next = from;
    for (int i0 = from; i0 < p.P && found < want; i0 += STEP) {
        const int first = i0 + 4 * EACH * (int)threadIdx.x;
        int r[EACH][4], cnt = 0, total;
#pragma unroll
        for (int e = 0; e < EACH; ++e) read_refs(p, first + 4 * e, r[e]);
#pragma unroll
        for (int j = 0; j < 4 * EACH; ++j) cnt += r[j >> 2][j & 3] == 0;
        int at = found + block_scan<THREADS>(cnt, lds, total);
#pragma unroll
        for (int j = 0; j < 4 * EACH; ++j)
            if (r[j >> 2][j & 3] == 0) {
                if (at < want) take(at, first + j);
                ++at;
            }
        found += total;
        next = i0;
    }
    return min(found, want);
}

// ---- reserve ----

// One work-group, SEQS sequences at a time: the first rank of each among the
// pages that are needed; then, RANKS at a time, the free pages in order, each
// to the entry that its rank falls to, a thread a rank.  One, because each
// sequence's pages follow from what the earlier ones take; bound by its chain of
// loads, sums and barriers: 5.4 us for 32 sequences, 6.2 for 64 (0.8 of it the
// look into the row and sums that stop in time).
// A row's entries past its tokens are looked at one by one, but only where
// tokens need more pages: one entry each unless its length was lowered.
// Once the pages have run out no later sequence gets any, not even those that
// the one they ran out in gives back: else it would depend on SEQS who does.
constexpr int SEQS = 4096, RANKS = 4096;
__global__ __launch_bounds__(1024) void pages_reserve_kernel(PagesParams p) {
    __shared__ int lds[16];
    __shared__ int start[SEQS], had[SEQS];
    __shared__ int list[RANKS];
    const int tid = threadIdx.x;
    const int64_t most = (int64_t)p.M << p.page_shift;
    // More than there are: what sums of needs stop at (they may pass 32 bits).
    const uint32_t beyond = (uint32_t)p.P + 1;
    // pages that sequence n holds in all once it has its tokens; -1: more than
    // a row holds
    auto pages_of = [&](int n, int& len) {
        len = max(0, p.lens[n]);
        const int64_t want = (int64_t)len + max(0, p.more[n]);
        return want > most ? -1 : pages_for((int)want, p.page_shift);
    };
    // pages that it has: those of its tokens, and any that follow them in its
    // row (its length was lowered: the tokens of a rejected draft)
    auto pages_had = [&](int n, int len, int want) {
        const int32_t* row = p.table + n * p.table_stride;
        int have = pages_for(len, p.page_shift);
        for (; have < want; ++have) {
            const uint32_t page = (uint32_t)row[have];
            if (page >= (uint32_t)p.P || p.refs[page] == 0) break;
        }
        return have;
    };
    int from = 0;
    bool out = false;  // the pages have run out
    for (int n0 = 0; n0 < p.N; n0 += SEQS) {
        const int count = min(SEQS, p.N - n0);
        uint32_t sum = 0;
        for (int i0 = 0; i0 < count; i0 += 1024) {
            int have = 0, want = 0;
            uint32_t total;
            if (i0 + tid < count) {
                int len;
                want = pages_of(n0 + i0 + tid, len);
                have = pages_had(n0 + i0 + tid, len, want);
            }
            const uint32_t need = max(0, want - have);
            const uint32_t before = block_scan_upto<1024>(min(need, beyond), beyond, lds, total);
            if (i0 + tid < count) {
                start[i0 + tid] = (int)min(sum + before, beyond);
                had[i0 + tid] = have;
            }
            sum = min(sum + total, beyond);
        }
        const int needed = (int)sum;
        int found = 0;
        for (int base = 0; !out && base < needed && found == base; base += RANKS) {
            int next;
            const int got = find_free<1024>(p, from, min(RANKS, needed - base), lds, next,
                                            [&](int rank, int page) { list[rank] = page; });
            from = next;
            __syncthreads();
            for (int k = tid; k < got; k += 1024) {
                // the last sequence that starts at or before the rank (those
                // without need start where the next one does)
                int lo = 0, hi = count - 1;
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (start[mid] <= base + k) lo = mid;
                    else hi = mid - 1;
                }
                p.table[(n0 + lo) * p.table_stride + had[lo] + base + k - start[lo]] = list[k];
                p.refs[list[k]] = 1;
            }
            found += got;
            __syncthreads();
        }
        out |= found < needed;
        for (int i = tid; i < count; i += 1024) {
            int len;
            const int n = n0 + i, want = pages_of(n, len), have = had[i];
            const bool fits = want >= 0, ok = fits && (want <= have || want - have <= found - start[i]);
            if (ok) {
                p.lens[n] = len + max(0, p.more[n]);
            } else if (fits) {
                // pages ran out inside it: what it got goes back
                for (int j = 0; j < found - start[i]; ++j) {
                    int32_t* entry = p.table + n * p.table_stride + have + j;
                    p.refs[*entry] = 0;
                    *entry = -1;
                }
            }
            p.ok[n] = ok;
        }
        __syncthreads();
    }
}

// ---- free ----

// A work-group a row, an atomic a page (counts are whole numbers: their order
// does not matter).  16 rows of 4000 tokens 2.9 us, 63 of 8191 5.2.
__global__ __launch_bounds__(512) void pages_free_kernel(PagesParams p) {
    const int n = p.dst[blockIdx.x];
    if ((unsigned)n >= (unsigned)p.N) return;
    int32_t* row = p.table + n * p.table_stride;
    // (the exchange: a row named twice gives its pages back once)
    for (int i = threadIdx.x; i < p.M; i += 512) {
        const int page = atomicExch(row + i, -1);
        if ((unsigned)page < (unsigned)p.P) atomicSub(p.refs + page, 1);
    }
    if (threadIdx.x == 0) p.lens[n] = 0;
}

// ---- copies ----

// Threads move 16 bytes each, COPY_UNROLL at a time: a work-group 8 KiB of a
// page at most (a compaction that moves 0.5 GB: 187 us, with 4 at a time 190,
// with 8 278).
constexpr int COPY_UNROLL = 2;
constexpr int COPY_BYTES = 256 * 16 * COPY_UNROLL;

// Piece `seg` of page `src` of one pool's part `lead` to page `dst`.  What is
// written is not read here again: stored past the caches, and with STREAM read
// past them too (not for a fork, whose source others fork as well).
template <bool STREAM>
__device__ __forceinline__ void copy_piece(const PagesParams& p, const KdaPagePool& x, int64_t lead, int src, int dst,
                                           int64_t seg) {
    char* base = static_cast<char*>(x.data) + lead * p.P * x.page_bytes;
    const char* from = base + src * x.page_bytes;
    char* to = base + dst * x.page_bytes;
    const int64_t off = seg * COPY_BYTES + threadIdx.x * 16;
    u32x4 w[COPY_UNROLL];
#pragma unroll
    for (int i = 0; i < COPY_UNROLL; ++i)
        if (off + i * 4096 < x.page_bytes) {
            const u32x4* at = reinterpret_cast<const u32x4*>(from + off + i * 4096);
            w[i] = STREAM ? __builtin_nontemporal_load(at) : *at;
        }
#pragma unroll
    for (int i = 0; i < COPY_UNROLL; ++i)
        if (off + i * 4096 < x.page_bytes)
            __builtin_nontemporal_store(w[i], reinterpret_cast<u32x4*>(to + off + i * 4096));
}

__host__ __device__ inline int64_t pieces_of(const KdaPagePool& x) { return (x.page_bytes + COPY_BYTES - 1) / COPY_BYTES; }

// Copies `count` pairs in all parts of all pools: (pool, part, pair, piece),
// pieces innermost, so that the work-groups that run together are in one part
// and finish whole pages (pair by pair, or a piece of every pair in turn, a
// compaction that moves 0.5 GB took 196 us, so 187).
template <class Pair>
__device__ __forceinline__ void copy_pairs(const PagesParams& p, int64_t count, Pair pair) {
    int64_t id = blockIdx.x;
    for (int i = 0; i < p.num_pools; ++i) {
        const KdaPagePool& x = p.pools[i];
        const int64_t seg = pieces_of(x), items = x.lead * count * seg;
        for (; id < items; id += gridDim.x) {
            const int64_t pr = id / seg, lead = pr / count;
            int src, dst;
            if (pair((int)(pr - lead * count), src, dst)) copy_piece<true>(p, x, lead, src, dst, id - pr * seg);
        }
        id -= items;
    }
}

int64_t copy_pieces(const PagesParams& p) {  // of a pair
    int64_t pieces = 0;
    for (int i = 0; i < p.num_pools; ++i) pieces += p.pools[i].lead * pieces_of(p.pools[i]);
    return pieces;
}
unsigned copy_grid(const PagesParams& p, int64_t pairs) {
    return (unsigned)std::min(std::max(copy_pieces(p) * pairs, (int64_t)1), (int64_t)256 * 64);
}

// (8 rows of 12 layers' states, 201 MB each way: 65 us, 6.2 TB/s.)
__global__ __launch_bounds__(256) void pages_copy_kernel(PagesParams p) {
    copy_pairs(p, p.F, [&](int i, int& src, int& dst) {
        src = p.src[i];
        dst = p.dst[i];
        return (unsigned)src < (unsigned)p.P && (unsigned)dst < (unsigned)p.P;
    });
}

// ---- fork ----

// A work-group a fork.  Shared pages gain a holder, which makes no free page
// of theirs, so that every work-group can look for its own free page while the
// others count; the pages found are marked by the copy that follows.  Bound by
// its chain: the earlier forks' lengths, the free pages up to its own, the row.
// 16 forks 5.8 us, 63 forks of 511 shared pages 8.1.
constexpr int FORK_THREADS = 512;
__global__ __launch_bounds__(FORK_THREADS) void pages_fork_kernel(PagesParams p) {
    __shared__ int lds[FORK_THREADS / 64];
    __shared__ int fresh;
    const int i = blockIdx.x, tid = threadIdx.x;
    auto len_of = [&](int j) {
        const int s = p.src[j];
        if ((unsigned)s >= (unsigned)p.N) return 0;
        const int64_t most = (int64_t)p.M << p.page_shift;
        return (int)min((int64_t)max(0, p.lens[s]), most);
    };
    const int mask = (1 << p.page_shift) - 1;
    const int s = p.src[i], d = p.dst[i];
    const bool rows_ok = (unsigned)s < (unsigned)p.N && (unsigned)d < (unsigned)p.N;
    const int len = len_of(i), full = len >> p.page_shift;
    const bool part = rows_ok && (len & mask) != 0;
    if (tid == 0) fresh = -1;
    if (part) {
        // the forks before it that need a page
        int before = 0, rank;
        for (int j = tid; j < i; j += FORK_THREADS) before += (unsigned)p.dst[j] < (unsigned)p.N && (len_of(j) & mask) != 0;
        block_scan<FORK_THREADS>(before, lds, rank);
        int next;
        find_free<FORK_THREADS>(p, 0, rank + 1, lds, next, [&](int at, int page) {
            if (at == rank) fresh = page;
        });
        __syncthreads();
    }
    const int page = part ? fresh : -1;
    const bool ok = rows_ok && (!part || page >= 0);
    if (ok) {
        const int32_t* from = p.table + s * p.table_stride;
        int32_t* to = p.table + d * p.table_stride;
        for (int j = tid; j < p.M; j += FORK_THREADS) {
            int x = -1;
            if (j < full) {
                x = from[j];
                if ((unsigned)x < (unsigned)p.P) atomicAdd(p.refs + x, 1);
            } else if (j == full && part) {
                x = page;
            }
            to[j] = x;
        }
    }
    if (tid == 0) {
        if (ok) p.lens[d] = len;
        p.ok[i] = ok;
    }
}

// Fork i's last page, if it has one of its own: from the rows that the fork
// left.
__device__ __forceinline__ bool forked_page(const PagesParams& p, int i, int& src, int& dst) {
    if (!p.ok[i]) return false;
    const int s = p.src[i], d = p.dst[i], len = p.lens[d], full = len >> p.page_shift;
    if (len - (full << p.page_shift) == 0) return false;
    src = p.table[s * p.table_stride + full];
    dst = p.table[d * p.table_stride + full];
    return (unsigned)dst < (unsigned)p.P;
}
// `share` work-groups a fork, which look its page up once and move every
// share-th piece of it in all parts of all pools.  63 forks in 32 parts (66 MB
// written) 14.2 us.
__global__ __launch_bounds__(256) void pages_fork_copy_kernel(PagesParams p, int share) {
    int src, dst;
    const int f = blockIdx.x % p.F;
    if (!forked_page(p, f, src, dst)) return;
    int64_t piece = blockIdx.x / p.F;
    if (piece == 0 && threadIdx.x == 0) p.refs[dst] = 1;
    if ((unsigned)src >= (unsigned)p.P) return;
    for (int i = 0; i < p.num_pools; ++i) {
        const KdaPagePool& x = p.pools[i];
        const int64_t seg = pieces_of(x), items = x.lead * seg;
        for (; piece < items; piece += share) copy_piece<false>(p, x, piece / seg, src, dst, piece % seg);
        piece -= items;
    }
}

// ---- compact ----

// The held pages of each 4096: counts for the lists of a large pool.
constexpr int LIST_PAGES = 4096;
// Up to here every work-group of the lists counts all pages itself, 16 at a
// time a thread: a launch less (a compaction of 256 pages 11.4 -> 9.1 us).
constexpr int COUNT_PAGES = 16 * LIST_PAGES;
__device__ __forceinline__ int held_of(const PagesParams& p, int i) {
    int r[4], cnt = 0;
    read_refs(p, i, r);
#pragma unroll
    for (int j = 0; j < 4; ++j) cnt += i + j < p.P && r[j] != 0;
    return cnt;
}
__global__ __launch_bounds__(1024) void pages_count_kernel(PagesParams p) {
    __shared__ int lds[16];
    int total;
    block_scan<1024>(held_of(p, blockIdx.x * LIST_PAGES + 4 * threadIdx.x), lds, total);
    if (threadIdx.x == 0) p.ws[3 * (int64_t)p.P + blockIdx.x] = total;
}

// Free places below `live` (the number of held pages), held pages at or above
// it, and the number of either.  A held page is ranked from the last one
// down, which needs no count of the places: the page with e held ones after
// it goes to the place of rank places - 1 - e.
struct CompactLists {
    int *holes, *movers, *rank, *counts;
    int blocks;
};
__host__ __device__ inline CompactLists compact_lists(const PagesParams& p) {
    CompactLists x;
    x.holes = p.ws;
    x.movers = p.ws + p.P;
    x.rank = p.ws + 2 * (int64_t)p.P;
    x.blocks = (p.P + LIST_PAGES - 1) / LIST_PAGES;
    x.counts = p.ws + 3 * (int64_t)p.P;  // then the number of places
    return x;
}

// Each work-group lists the holes, the movers and the movers' ranks among its
// LIST_PAGES pages, its place in the lists from the counts of all: 3 to 5 us.
__global__ __launch_bounds__(1024) void pages_list_kernel(PagesParams p) {
    __shared__ int lds[16];
    const CompactLists x = compact_lists(p);
    const int tid = threadIdx.x;
    // held pages of the work-groups before, and of all
    int mine = 0, all = 0;
    if (p.P <= COUNT_PAGES) {
#pragma unroll 4
        for (int b = 0; b < x.blocks; ++b) {
            const int c = held_of(p, b * LIST_PAGES + 4 * tid);
            all += c;
            mine += b < (int)blockIdx.x ? c : 0;
        }
    } else {
        for (int b = tid; b < x.blocks; b += 1024) {
            const int c = x.counts[b];
            all += c;
            mine += b < (int)blockIdx.x ? c : 0;
        }
    }
    int before, live;
    block_scan<1024>(mine, lds, before);
    block_scan<1024>(all, lds, live);
    int r[4], total, cnt = 0;
    const int i = blockIdx.x * LIST_PAGES + 4 * tid;
    read_refs(p, i, r);
#pragma unroll
    for (int j = 0; j < 4; ++j) cnt += i + j < p.P && r[j] != 0;
    int held = before + block_scan<1024>(cnt, lds, total);  // held pages below the one looked at
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int page = i + j;
        if (page >= p.P) break;
        if (page == live) x.counts[x.blocks] = live - held;
        if (r[j] == 0 && page < live) x.holes[page - held] = page;
        if (r[j] != 0) {
            ++held;
            if (page >= live) {
                x.movers[live - held] = page;
                x.rank[page] = live - held;
            }
        }
        p.out_refs[page] = r[j];
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.out_live[0] = live;
        if (live == p.P) x.counts[x.blocks] = 0;
    }
}

// The new table and counts, and the pages: bound by HBM (540 MB read and as
// many written in 182 us, 5.9 TB/s; a large device copy reaches 4.7).
__global__ __launch_bounds__(256) void pages_move_kernel(PagesParams p) {
    const CompactLists x = compact_lists(p);
    const int live = p.out_live[0], places = x.counts[x.blocks];
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
    for (int64_t e = id; e < (int64_t)p.N * p.M; e += step) {
        int page = p.table[e / p.M * p.table_stride + e % p.M];
        // (a page that no count holds stays where it is)
        if (page >= live && page < p.P && p.refs[page] != 0) page = x.holes[places - 1 - x.rank[page]];
        p.out_table[e] = page;
    }
    for (int64_t i = id; i < places; i += step) {
        const int from = x.movers[places - 1 - i];
        p.out_refs[x.holes[i]] = p.refs[from];
        p.out_refs[from] = 0;
    }
    copy_pairs(p, places, [&](int i, int& src, int& dst) {
        src = x.movers[places - 1 - i];
        dst = x.holes[i];
        return true;
    });
}

}  // namespace

hipError_t launch_paged_append(const PagedParams& p, int D, hipStream_t stream) {
    const int64_t tokens = p.cu_seqlens ? p.T : (int64_t)p.N * p.T;
    const int64_t total = tokens * p.HKV * (D / 8);
    const dim3 grid((unsigned)((total + 255) / 256));
    if (D == 128) paged_append_kernel<128><<<grid, 256, 0, stream>>>(p, (int)total);
    else paged_append_kernel<64><<<grid, 256, 0, stream>>>(p, (int)total);
    return hipGetLastError();
}

hipError_t launch_pages_reserve(const PagesParams& p, hipStream_t stream) {
    pages_reserve_kernel<<<1, 1024, 0, stream>>>(p);
    return hipGetLastError();
}

hipError_t launch_pages_free(const PagesParams& p, hipStream_t stream) {
    pages_free_kernel<<<p.F, 512, 0, stream>>>(p);
    return hipGetLastError();
}

hipError_t launch_pages_copy(const PagesParams& p, hipStream_t stream) {
    pages_copy_kernel<<<copy_grid(p, p.F), 256, 0, stream>>>(p);
    return hipGetLastError();
}

hipError_t launch_pages_fork(const PagesParams& p, hipStream_t stream) {
    pages_fork_kernel<<<p.F, FORK_THREADS, 0, stream>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // a piece each where there are few, up to 4 where there are many
    const int64_t pieces = copy_pieces(p), each = std::min(std::max(pieces * p.F / 2048, (int64_t)1), (int64_t)4);
    const int64_t share = std::min((pieces + each - 1) / each, std::max((int64_t)256 * 64 / p.F, (int64_t)1));
    pages_fork_copy_kernel<<<dim3((unsigned)(share * p.F)), 256, 0, stream>>>(p, (int)share);
    return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesParams& p, hipStream_t stream) {
    const int blocks = compact_lists(p).blocks;
    hipError_t e = hipSuccess;
    if (p.P > COUNT_PAGES) {
        pages_count_kernel<<<blocks, 1024, 0, stream>>>(p);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    pages_list_kernel<<<blocks, 1024, 0, stream>>>(p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    // at most half of the pages move
    pages_move_kernel<<<copy_grid(p, p.P / 2), 256, 0, stream>>>(p);
    return hipGetLastError();
}

}  // namespace kda
