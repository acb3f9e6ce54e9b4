// The pages of a cache (kda_paged_hip.h): append of new tokens, reserve, free,
// fork, copy and compact.
//
// Which pages are free is what page_refs says and nothing else: a page with
// no holder is free, and every call hands out the lowest free pages.  So no
// list has to be kept, and results do not depend on the order in which
// work-groups run.
#include "kda_common.h"
#include "kda_paged.h"

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

// One thread moves 16 bytes of a token's keys and the same of its values.
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

__device__ __forceinline__ int wave_scan(int x, int lane) {  // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}

// Exclusive prefix sum over the work-group's threads, and the total.
template <int THREADS>
__device__ __forceinline__ int block_scan(int x, int* lds, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int inc = wave_scan(x, lane);
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

// ---- reserve ----

// One work-group: the pages each sequence needs and their first rank among
// all that are needed, the list of as many free pages, and their entries.
__global__ __launch_bounds__(1024) void pages_reserve_kernel(PagesParams p) {
    __shared__ int lds[16];
    int* list = p.ws;
    int* rank = p.ws + p.P;
    const int tid = threadIdx.x;
    const int64_t most = (int64_t)p.M << p.page_shift;
    auto need_of = [&](int n, int& have) {
        const int len = max(0, p.lens[n]);
        have = pages_for(len, p.page_shift);
        const int64_t want = (int64_t)len + max(0, p.more[n]);
        if (want > most) return -1;
        return max(0, pages_for((int)want, p.page_shift) - have);
    };
    int needed = 0;
    for (int n0 = 0; n0 < p.N; n0 += 1024) {
        int have, total;
        const int need = n0 + tid < p.N ? max(0, need_of(n0 + tid, have)) : 0;
        const int before = block_scan<1024>(need, lds, total);
        if (n0 + tid < p.N) rank[n0 + tid] = needed + before;
        needed += total;
    }
    int found = 0;
    for (int i0 = 0; i0 < p.P && found < needed; i0 += 4096) {
        int r[4], total;
        read_refs(p, i0 + 4 * tid, r);
        int cnt = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) cnt += r[j] == 0;
        int at = found + block_scan<1024>(cnt, lds, total);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (r[j] == 0) {
                if (at < needed) list[at] = i0 + 4 * tid + j;
                ++at;
            }
        found += total;
    }
    __syncthreads();
    // a wave a sequence: its entries
    const int lane = tid & 63;
    for (int n = tid >> 6; n < p.N; n += 16) {
        int have;
        const int need = need_of(n, have), start = rank[n];
        const bool ok = need == 0 || (need > 0 && start + need <= found);
        for (int i = lane; ok && i < need; i += 64) {
            const int page = list[start + i];
            p.table[n * p.table_stride + have + i] = page;
            p.refs[page] = 1;
        }
        if (lane == 0) {
            if (ok) p.lens[n] = max(0, p.lens[n]) + max(0, p.more[n]);
            p.ok[n] = ok;
        }
    }
}

// ---- free ----

__global__ __launch_bounds__(256) void pages_free_kernel(PagesParams p) {
    const int n = p.dst[blockIdx.x];
    if ((unsigned)n >= (unsigned)p.N) return;
    int32_t* row = p.table + n * p.table_stride;
    // (the exchange: a row named twice gives its pages back once)
    for (int i = threadIdx.x; i < p.M; i += 256) {
        const int page = atomicExch(row + i, -1);
        if ((unsigned)page < (unsigned)p.P) atomicSub(p.refs + page, 1);
    }
    if (threadIdx.x == 0) p.lens[n] = 0;
}

// ---- copies ----

// Threads move 16 bytes each, COPY_UNROLL at a time: a work-group 8 KiB of a
// page at most (more in flight a thread was slower: a compaction that moves
// 0.5 GB @COPY@).
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

// Work items of all pools for `count` pairs: (pool, lead, pair, piece), pieces
// innermost.
__host__ __device__ inline int64_t pieces_of(const KdaPagePool& x) { return (x.page_bytes + COPY_BYTES - 1) / COPY_BYTES; }

template <bool STREAM, class Pair>
__device__ __forceinline__ void copy_items(const PagesParams& p, int64_t count, Pair pair) {
    int64_t first = 0;
    for (int i = 0; i < p.num_pools; ++i) {
        const KdaPagePool& x = p.pools[i];
        const int64_t seg = pieces_of(x), items = x.lead * count * seg;
        // the first of this work-group's items in this pool
        int64_t id = blockIdx.x - first % gridDim.x;
        if (id < 0) id += gridDim.x;
        for (; id < items; id += gridDim.x) {
            const int64_t pr = id / seg, lead = pr / count;
            int src, dst;
            if (pair((int)(pr - lead * count), src, dst)) copy_piece<STREAM>(p, x, lead, src, dst, id - pr * seg);
        }
        first += items;
    }
}

constexpr int COPY_GRID = 256 * 64;

int copy_grid(const PagesParams& p, int64_t count) {
    int64_t items = 0;
    for (int i = 0; i < p.num_pools; ++i) items += p.pools[i].lead * count * pieces_of(p.pools[i]);
    return (int)(items < 1 ? 1 : (items > COPY_GRID ? COPY_GRID : items));
}

__global__ __launch_bounds__(256) void pages_copy_kernel(PagesParams p) {
    copy_items<true>(p, p.F, [&](int i, int& src, int& dst) {
        src = p.src[i];
        dst = p.dst[i];
        return (unsigned)src < (unsigned)p.P && (unsigned)dst < (unsigned)p.P;
    });
}

// ---- fork ----

// A work-group a fork.  Shared pages gain a holder, which makes no free page
// of theirs, so that every work-group can look for its own free page while the
// others count; the pages found are marked by the copy that follows.
__global__ __launch_bounds__(256) void pages_fork_kernel(PagesParams p) {
    __shared__ int lds[4];
    __shared__ int found;
    const int i = blockIdx.x, tid = threadIdx.x;
    int* whence = p.ws;
    int* fresh = whence + p.F;
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
    // the forks before it that need a page
    int rank = 0;
    for (int j0 = 0; j0 < i; j0 += 256) {
        int total;
        const int j = j0 + tid;
        const bool need = j < i && (unsigned)p.dst[j] < (unsigned)p.N && (len_of(j) & mask) != 0;
        block_scan<256>(need, lds, total);
        rank += total;
    }
    if (tid == 0) found = -1;
    __syncthreads();
    if (part) {
        int seen = 0;
        for (int i0 = 0; i0 < p.P && seen <= rank; i0 += 1024) {
            int r[4], total;
            read_refs(p, i0 + 4 * tid, r);
            int cnt = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) cnt += r[j] == 0;
            int at = seen + block_scan<256>(cnt, lds, total);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r[j] == 0) {
                    if (at == rank) found = i0 + 4 * tid + j;
                    ++at;
                }
            seen += total;
        }
        __syncthreads();
    }
    const int page = found;
    const bool ok = rows_ok && (!part || page >= 0);
    if (ok) {
        const int32_t* from = p.table + s * p.table_stride;
        int32_t* to = p.table + d * p.table_stride;
        for (int j = tid; j < p.M; j += 256) {
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
        whence[i] = ok && part ? p.table[s * p.table_stride + full] : -1;
        fresh[i] = ok && part ? page : -1;
    }
}

__global__ __launch_bounds__(256) void pages_fork_copy_kernel(PagesParams p) {
    const int* whence = p.ws;
    const int* fresh = whence + p.F;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < p.F; i += gridDim.x * 256)
        if (fresh[i] >= 0) p.refs[fresh[i]] = 1;
    copy_items<false>(p, p.F, [&](int i, int& src, int& dst) {
        src = whence[i];
        dst = fresh[i];
        return (unsigned)src < (unsigned)p.P && dst >= 0;
    });
}

// ---- compact ----

// The held pages of each 4096: counts for the lists of a large pool.
constexpr int LIST_PAGES = 4096;
// Up to here every work-group of the lists counts all pages itself, 16 at a
// time a thread: a launch less (256 pages, a compaction @COUNT@ us).
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
    copy_items<true>(p, places, [&](int i, int& src, int& dst) {
        src = x.movers[places - 1 - i];
        dst = x.holes[i];
        return true;
    });
}

}  // namespace

hipError_t launch_paged_append(const PagedParams& p, int D, hipStream_t stream) {
    const int64_t tokens = p.cu_seqlens ? p.T : (int64_t)p.N * p.T;
    const int64_t total = tokens * p.HKV * (D / 8);
    if (total > 0x7fffffff) return hipErrorInvalidValue;
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
    pages_free_kernel<<<p.F, 256, 0, stream>>>(p);
    return hipGetLastError();
}

hipError_t launch_pages_copy(const PagesParams& p, hipStream_t stream) {
    pages_copy_kernel<<<copy_grid(p, p.F), 256, 0, stream>>>(p);
    return hipGetLastError();
}

hipError_t launch_pages_fork(const PagesParams& p, hipStream_t stream) {
    pages_fork_kernel<<<p.F, 256, 0, stream>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    pages_fork_copy_kernel<<<copy_grid(p, p.F), 256, 0, stream>>>(p);
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
