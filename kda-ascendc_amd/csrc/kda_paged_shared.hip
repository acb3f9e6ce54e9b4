// Attention of new tokens over a paged cache by sequences in groups that share
// their first tokens (kda_paged_hip.h), with the loops over rows and keys of
// kda_paged_attn.h.
//
// A softmax over two sets of keys is put together from the two: with m, l and O
// (the maximum, the sum of e^(s-m), that of e^(s-m) v) of each,
//   m = max(m1, m2),  l = l1 e^(m1-m) + l2 e^(m2-m),  O likewise.
// So the shared tokens of a group are worked on once, for the queries of all of
// its sequences together (64 sequences of 4 heads a kv head: a row tile of 256
// rows instead of 64 that are an eighth full, and the keys read once instead of
// 64 times), the tokens behind them for each sequence, and the results joined.
//
// Three launches.  A plan, by one work-group: what there is to work on (for each
// group its shared tokens, for each sequence what is its own), into how many
// parts its keys are cut, where the partial results go.  The parts, a work-group
// each.  The join.
#include "kda_paged_attn.h"

namespace kda {
namespace {

// Sequences and groups that a plan has room for.
constexpr int MOST = 2048;

// What is worked on together: the queries of a group over its shared tokens, or
// those of a sequence over its own.  Records of all groups, then of all
// sequences.
struct Work {
    int first, count, len, pos;  // as NewTokens, `first` a token of all
    int from, row;               // the first key, a row of the table
    int parts, mt;               // parts of a row tile's keys; row tiles
    int place;                   // of the partial results, in 4 rows; NONE, or OVER where there is no room
    int group;                   // a sequence's record of shared tokens, -1: none
    int few, tiles;              // of few rows; tiles of keys
};
constexpr int NONE = -1, OVER = -2;

// The plan in the workspace: a head, the ends of every record's units of few
// and of many rows, the records.
constexpr int HEAD = 16;
struct Plan {
    int32_t* head;  // units of few rows, of many
    int32_t* few_end;
    int32_t* many_end;
    Work* work;
};
__host__ __device__ inline int round16(int x) { return (x + 15) & ~15; }
__device__ __forceinline__ Plan plan_of(const SharedParams& p) {
    const int V = round16(p.NG + p.N);
    return {p.plan, p.plan + HEAD, p.plan + HEAD + V, reinterpret_cast<Work*>(p.plan + HEAD + 2 * V)};
}
int64_t plan_bytes(const SharedParams& p) {
    const int64_t V = round16(p.NG + p.N);
    return (HEAD + 2 * V + V * (int64_t)(sizeof(Work) / 4)) * 4;
}

// Rows of a tile of partial results: a multiple of 4.
__host__ __device__ inline int padded(int rows) { return (rows + 3) & ~3; }

// Inclusive prefix sums of three numbers over the work-group's threads.
struct Three {
    int a, b, c;
};
template <int THREADS>
__device__ __forceinline__ Three scan(Three x, int (&lds)[3][16]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Three s = {(int)wave_prefix(x.a), (int)wave_prefix(x.b), (int)wave_prefix(x.c)};
    __syncthreads();
    if (lane == 63) {
        lds[0][wave] = s.a;
        lds[1][wave] = s.b;
        lds[2][wave] = s.c;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w)
        if (w < wave) {
            s.a += lds[0][w];
            s.b += lds[1][w];
            s.c += lds[2][w];
        }
    return s;
}
// Sums over the work-group's threads.
template <int THREADS>
__device__ __forceinline__ int64_t sum(int64_t x, int64_t (&lds)[16]) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) all += lds[w];
    return all;
}

// One work-group.  `waves`: those of a work-group of few rows; `room`: of the
// partial results, in 4 rows.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void paged_shared_plan_kernel(SharedParams p, int waves, int room) {
    __shared__ int cu[MOST + 1], least[MOST], sharing[MOST], shared_of[MOST];
    __shared__ int lds3[3][16];
    __shared__ int64_t lds[16];
    constexpr int BIG = 1 << 20;
    const int tid = threadIdx.x, V = p.NG + p.N, each = (V + THREADS - 1) / THREADS;  // records a thread
    const int64_t most = (int64_t)p.M << p.page_shift;
    for (int g = tid; g <= p.NG; g += THREADS) {
        cu[g] = min(max(p.cu_groups[g], 0), p.N);
        if (g < p.NG) {
            const int len = p.shared_lens[g];
            shared_of[g] = len < 0 ? 0 : ((int64_t)len > most ? (int)most : len);
            least[g] = p.N;
            sharing[g] = 0;
        }
    }
    __syncthreads();
    // The group of sequence n, -1 for none.
    auto group_of = [&](int n) {
        int lo = 0, hi = p.NG - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (cu[mid] <= n) lo = mid;
            else hi = mid - 1;
        }
        return cu[lo] <= n && n < cu[lo + 1] ? lo : -1;
    };
    // A sequence shares if its new tokens all come behind the group's shared ones.
    auto shares = [&](const NewTokens& s, int g) { return g >= 0 && s.count > 0 && shared_of[g] > 0 && s.pos >= shared_of[g]; };
    for (int n = tid; n < p.N; n += THREADS) {
        const NewTokens s = new_tokens(p, n);
        const int g = group_of(n);
        if (shares(s, g)) {
            atomicMin(&least[g], n);
            atomicAdd(&sharing[g], 1);
        }
        // (a sequence that fills a row tile by itself: nothing to gain for it)
        if (g >= 0 && (int64_t)s.count * p.G >= Shape<MANY>::MT) atomicOr(&sharing[g], BIG);
    }
    __syncthreads();
    auto active = [&](int g) { return sharing[g] >= 2 && sharing[g] < BIG; };

    // What there is to work on, and how much of each kind.
    const Plan plan = plan_of(p);
    int64_t few_all = 0, many_all = 0, many_tiles = 0;
    for (int v = tid * each; v < min(V, (tid + 1) * each); ++v) {
        Work w = {};
        w.group = -1;
        if (v >= p.NG) {
            const int n = v - p.NG;
            const NewTokens s = new_tokens(p, n);
            w.first = p.cu_seqlens ? s.first : n * p.T;
            w.count = s.count;
            w.len = s.len;
            w.pos = s.pos;
            w.row = n;
            const int g = group_of(n);
            if (shares(s, g) && active(g)) {
                w.group = g;
                w.from = shared_of[g];
            }
        } else if (active(v)) {
            const int n0 = cu[v], n1 = max(n0, cu[v + 1]);
            w.first = p.cu_seqlens ? paged_cu(p, n0) : n0 * p.T;
            w.count = max(0, (p.cu_seqlens ? paged_cu(p, n1) : n1 * p.T) - w.first);
            w.len = w.pos = shared_of[v];
            w.row = least[v];
        }
        if (w.count > 0) {
            w.few = (int64_t)w.count * p.G <= ROWS;
            const int TK = w.few ? Shape<FEW>::TK : Shape<MANY>::TK, MT = w.few ? Shape<FEW>::MT : Shape<MANY>::MT;
            w.mt = (int)(((int64_t)w.count * p.G + MT - 1) / MT);
            w.tiles = max(1, (w.len + TK - 1) / TK - w.from / TK);
            if (w.few) {
                few_all += w.tiles;
            } else {
                many_all += w.mt;
                many_tiles += (int64_t)w.mt * w.tiles;
            }
        }
        plan.work[v] = w;
    }
    few_all = sum<THREADS>(few_all, lds) * p.HKV;
    many_all = sum<THREADS>(many_all, lds) * p.HKV;
    many_tiles = sum<THREADS>(many_tiles, lds) * p.HKV;
    const int slots = few_slots(waves);
    const int64_t size = max((int64_t)waves, (few_all + slots - 1) / slots);
    const bool cut = many_all <= Shape<MANY>::SLOTS / 2;
    // Units of few and of many rows, and the room that a record's results need.
    auto needs = [&](Work& w, int v) {
        Three x = {0, 0, 0};
        if (w.count == 0) return x;
        if (w.few) {
            w.parts = (int)((w.tiles + size - 1) / size);
            x.a = w.parts * p.HKV;
        } else {
            w.parts = 1;
            if (cut) {
                const int64_t parts = (int64_t)w.tiles * Shape<MANY>::SLOTS / many_tiles;
                w.parts = (int)max((int64_t)1, min((int64_t)w.tiles / Shape<MANY>::LEAST, parts));
            }
            x.b = w.mt * w.parts * p.HKV;
        }
        w.place = NONE;
        if (w.parts > 1 || v < p.NG || w.group >= 0) x.c = padded(w.count * p.G) / 4 * w.parts * p.HKV;
        return x;
    };
    Three mine = {0, 0, 0};
    for (int v = tid * each; v < min(V, (tid + 1) * each); ++v) {
        Work w = plan.work[v];
        const Three x = needs(w, v);
        mine = {mine.a + x.a, mine.b + x.b, mine.c + x.c};
    }
    const Three upto = scan<THREADS>(mine, lds3);
    Three at = {upto.a - mine.a, upto.b - mine.b, upto.c - mine.c};
    for (int v = tid * each; v < min(V, (tid + 1) * each); ++v) {
        Work w = plan.work[v];
        const Three x = needs(w, v);
        if (x.c > 0) w.place = at.c + x.c <= room ? at.c : OVER;
        at = {at.a + x.a, at.b + x.b, at.c + x.c};
        plan.few_end[v] = at.a;
        plan.many_end[v] = at.b;
        plan.work[v] = w;
    }
    if (tid == THREADS - 1) {
        plan.head[0] = upto.a;
        plan.head[1] = upto.b;
    }
}

// Four rows of partial results in floats: m and l, then O.
template <int D>
constexpr int64_t FOUR = 4 * (D + 2);

// Where the part-th part of row tile m of (w, kv head h) is, of `rows` rows.
template <int D, int MT>
__device__ __forceinline__ int64_t place_of(const SharedParams& p, const Work& w, int m, int h, int part, int rows) {
    return FOUR<D> * (w.place + (int64_t)m * (MT / 4) * p.HKV * w.parts + (h * w.parts + part) * (rows / 4));
}
template <int MT>
__device__ __forceinline__ int tile_rows(const SharedParams& p, const Work& w, int m) {
    return padded(min(MT, w.count * p.G - m * MT));
}

__device__ __forceinline__ Work load_work(const Plan& plan, int v) {
    typedef __attribute__((address_space(4))) const int32_t c_i32;
    c_i32* at = (c_i32*)(plan.work + v);
    Work w;
    w.first = at[0];
    w.count = at[1];
    w.len = at[2];
    w.pos = at[3];
    w.from = at[4];
    w.row = at[5];
    w.parts = at[6];
    w.mt = at[7];
    w.place = at[8];
    w.group = at[9];
    w.few = at[10];
    return w;
}

// Unit x of kind KIND; false where its results have no room.
template <int KIND, int D>
__device__ __forceinline__ bool unit_of(const SharedParams& p, const Plan& plan, int x, int lane, Unit& u) {
    constexpr int TK = Shape<KIND>::TK, MT = Shape<KIND>::MT;
    const int32_t* ends = KIND == FEW ? plan.few_end : plan.many_end;
    const int V = p.NG + p.N;
    int v = 0, before = 0;
    for (int v0 = 0; v0 < V; v0 += 64) {
        const int end = v0 + lane < V ? ends[v0 + lane] : 0x7fffffff;
        const uint64_t past = __ballot(end > x);
        if (past) {
            const int at = __builtin_ctzll(past);
            v = v0 + at;
            if (at > 0) before = __builtin_amdgcn_readlane(end, at - 1);
            break;
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    v = __builtin_amdgcn_readfirstlane(v);
    const Work w = load_work(plan, v);
    if (w.place == OVER || w.count == 0) return false;
    x -= before;
    // heads innermost, as the XCDs go round; row tiles that see the most keys first
    u.n = w.row;
    u.h = x % p.HKV;
    x /= p.HKV;
    const int part = x % w.parts;
    u.m = w.mt - 1 - x / w.parts;
    u.s = NewTokens{w.first, w.count, w.len, w.pos};
    const int last = (min(w.count * p.G, u.m * MT + MT) - 1) / p.G;
    u.lo = w.from;
    u.hi = max(w.from, min(w.pos + last + 1, w.len));
    const int t0 = u.lo / TK;
    const int64_t tiles = max(t0, (u.hi + TK - 1) / TK) - t0;
    u.begin = t0 + (int)(tiles * part / w.parts);
    u.end = t0 + (int)(tiles * (part + 1) / w.parts);
    u.rows = tile_rows<MT>(p, w, u.m);
    u.place = w.place == NONE ? -1 : place_of<D, MT>(p, w, u.m, u.h, part, u.rows);
    return true;
}

// A part a work-group, those of many rows first (the grid is what the host knows
// that there can be at most).
template <class E, int D, int KIND>
__global__ __launch_bounds__(KIND == FEW ? 256 : 512, 2) void paged_shared_kernel(SharedParams p) {
    constexpr int WAVES = Shape<KIND == FEW ? FEW : MANY>::WAVES;
    typedef FewLds<D, WAVES> Lds;
    constexpr int RING = KIND == FEW ? 16 : 3 * Shape<MANY>::TK * D * 2;
    __shared__ alignas(1024) uint8_t kt[KIND == FEW ? WAVES * Lds::EACH : RING];
    __shared__ alignas(1024) uint8_t vt[RING];
    __shared__ alignas(1024) uint8_t more[KIND == FEW ? 16 : 2 * Lds::EACH];
    __shared__ float joint[WAVES * 2 * ROWS];
    const int lane = threadIdx.x & 63, id = blockIdx.x;
    const Plan plan = plan_of(p);
    typedef __attribute__((address_space(4))) const int32_t c_i32;
    const int few = ((c_i32*)plan.head)[0], many = ((c_i32*)plan.head)[1];
    if (id >= few + many) return;
    Unit u;
    if (KIND == FEW || id >= many) {
        if (unit_of<FEW, D>(p, plan, id - many, lane, u))
            few_rows<E, D, WAVES>(p, u, KIND == FEW ? Lds{kt, kt, kt} : Lds{kt, vt, more}, joint);
    } else if constexpr (KIND != FEW) {
        if (unit_of<MANY, D>(p, plan, id, lane, u)) many_rows<E, D>(p, u, kt, vt);
    }
}

// Joins the parts of (sequence n, kv head h): its own and those of its group's
// shared tokens, four elements of a row a thread, SLICES threads' parts in turn.
template <class E, int D>
__global__ __launch_bounds__(256) void paged_shared_join_kernel(SharedParams p, int groups) {
    __shared__ float lds[6 * 256];
    const Plan plan = plan_of(p);
    const int id = blockIdx.x / groups, n = id / p.HKV, h = id - n * p.HKV;
    const Work w = load_work(plan, p.NG + n);
    if (w.count == 0 || w.place < 0) return;
    Work g = {};
    if (w.group >= 0) g = load_work(plan, w.group);
    if (g.place == OVER) return;
    const int rows = w.count * p.G, rows_g = g.count * p.G;
    const bool w_few = w.few, g_few = g.few;
    const int slice = threadIdx.x >> 6;
    for (int group = blockIdx.x % groups; group * 64 < rows * (D / 4); group += groups) {
        const int e = group * 64 + (threadIdx.x & 63), r = e / (D / 4), piece = e % (D / 4);
        const bool live = r < rows;
        // its place in the group's rows
        const int rg = (w.first - g.first) * p.G + r;
        const int shared_parts = w.group >= 0 && rg >= 0 && rg < rows_g ? g.parts : 0;
        float mx = -INFINITY, total = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        if (live) {
            const int m = w_few ? 0 : r / Shape<MANY>::MT, mg = g_few ? 0 : rg / Shape<MANY>::MT;
            const int R = w_few ? tile_rows<ROWS>(p, w, 0) : tile_rows<Shape<MANY>::MT>(p, w, m);
            const int RG = g_few ? tile_rows<ROWS>(p, g, 0) : tile_rows<Shape<MANY>::MT>(p, g, mg);
            const float* own = p.ws + (w_few ? place_of<D, ROWS>(p, w, 0, h, 0, R) : place_of<D, Shape<MANY>::MT>(p, w, m, h, 0, R));
            const float* theirs = p.ws + (g_few ? place_of<D, ROWS>(p, g, 0, h, 0, RG) : place_of<D, Shape<MANY>::MT>(p, g, mg, h, 0, RG));
            const int r_own = r - m * Shape<MANY>::MT, r_theirs = rg - mg * Shape<MANY>::MT;
#pragma unroll 4
            for (int j = slice; j < shared_parts + w.parts; j += SLICES) {
                const bool s = j < shared_parts;
                const float* part = s ? theirs + (int64_t)j * (RG / 4) * FOUR<D> : own + (int64_t)(j - shared_parts) * (R / 4) * FOUR<D>;
                const int rr = s ? r_theirs : r_own, RR = s ? RG : R;
                const float mj = part[rr], lj = part[RR + rr];
                const f32x4 v = *reinterpret_cast<const f32x4*>(part + 2 * RR + rr * D + piece * 4);
                const float top = fmaxf(mx, mj), sub = top == -INFINITY ? 0.f : top;
                const float f0 = fast_exp2(mx - sub), f = fast_exp2(mj - sub);
                mx = top;
                total = fmaf(f, lj, total * f0);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = fmaf(f, v[i], o[i] * f0);
            }
        }
        const int t = threadIdx.x;
        lds[t] = mx;
        lds[256 + t] = total;
#pragma unroll
        for (int i = 0; i < 4; ++i) lds[(2 + i) * 256 + t] = o[i];
        __syncthreads();
        if (slice == 0 && live) {
            float top = mx;
#pragma unroll
            for (int k = 1; k < SLICES; ++k) top = fmaxf(top, lds[k * 64 + t]);
            const float sub = top == -INFINITY ? 0.f : top;
            float f = fast_exp2(mx - sub);
            total *= f;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] *= f;
#pragma unroll
            for (int k = 1; k < SLICES; ++k) {
                f = fast_exp2(lds[k * 64 + t] - sub);
                total = fmaf(f, lds[256 + k * 64 + t], total);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = fmaf(f, lds[(2 + i) * 256 + k * 64 + t], o[i]);
            }
            const float inv = total > 0.f ? 1.f / total : 0.f;
            const int tok = r / p.G;
            const int64_t out = ((int64_t)w.first + tok) * p.HQ + h * p.G + (r - tok * p.G);
            store_o<E, D>(p, out, piece * 4, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            if (p.lse && piece == 0) p.lse[out] = log_sum(top, total);
        }
        __syncthreads();
    }
}

// ---- launches ----

// Whether sequences are worked on together at all: not where each fills row
// tiles by itself, nor where there are more than a plan has room for.
bool together(const SharedParams& p) {
    return p.N >= 2 && p.N <= MOST && p.NG <= MOST && (p.cu_seqlens || (int64_t)p.T * p.G < Shape<MANY>::MT);
}
int64_t tokens_of(const SharedParams& p) { return p.cu_seqlens ? p.T : (int64_t)p.N * p.T; }
bool few_only(const SharedParams& p) { return tokens_of(p) * p.G <= ROWS; }

// Room of the partial results, in 4 rows: twice the rows that may be worked on
// together (a group's and the sequences', each filled up to 4), and the parts
// that keys are cut into.
int64_t room_of(const SharedParams& p) {
    const int64_t sharing = std::min(tokens_of(p), (int64_t)p.N * (Shape<MANY>::MT / p.G + 1));
    const int64_t rows = (2 * sharing * p.G + 3 * (int64_t)(p.N + p.NG)) * p.HKV;
    const int64_t few = 2 * (int64_t)few_slots(Shape<FEW>::WAVES) * ROWS;
    const int64_t many = few_only(p) ? 0 : (int64_t)Shape<MANY>::SLOTS * Shape<MANY>::MT;
    return (rows + few + many + 3) / 4;
}

// Units at most: a record's heads and row tiles, and the parts more that keys
// are cut into.  Records of many rows have more than ROWS of them.
int64_t units_of(const SharedParams& p, int waves) {
    const int64_t rows = tokens_of(p) * p.G;
    const int64_t groups = std::min(p.NG, p.N / 2), all = p.N + groups;
    const int64_t few = all * p.HKV + few_slots(waves);
    if (few_only(p)) return few;
    const bool members = p.cu_seqlens || (int64_t)p.T * p.G > ROWS;
    const int64_t records = std::min(groups + (members ? p.N : 0), (members ? 2 : 1) * rows / ROWS);
    return few + (records + (members ? 2 : 1) * rows / Shape<MANY>::MT) * p.HKV + Shape<MANY>::SLOTS;
}

template <class E, int D>
hipError_t launch_shared(SharedParams p, hipStream_t stream) {
    p.plan = reinterpret_cast<int32_t*>(p.ws + 4 * (D + 2) * room_of(p));
    const int V = p.NG + p.N, room = (int)std::min(room_of(p), (int64_t)0x7fffffff);
    const bool only = few_only(p);
    const int waves = Shape<FEW>::WAVES * (only ? 1 : 2);
    if (V <= 256) paged_shared_plan_kernel<256><<<1, 256, 0, stream>>>(p, waves, room);
    else paged_shared_plan_kernel<1024><<<1, 1024, 0, stream>>>(p, waves, room);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)units_of(p, waves));
    if (only) paged_shared_kernel<E, D, FEW><<<grid, 256, 0, stream>>>(p);
    else paged_shared_kernel<E, D, MIXED><<<grid, 512, 0, stream>>>(p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t rows = p.cu_seqlens ? ROWS : std::min((int64_t)p.T * p.G, (int64_t)ROWS);
    const int groups = (int)std::min((rows * (D / 4) + 63) / 64, (int64_t)4);
    paged_shared_join_kernel<E, D><<<dim3((unsigned)(p.N * p.HKV * groups)), 256, 0, stream>>>(p, groups);
    return hipGetLastError();
}

}  // namespace

size_t paged_attn_workspace(const SharedParams& p, int D) {
    if (!together(p)) return paged_attn_workspace(static_cast<const PagedParams&>(p), D);
    return (size_t)(4 * (D + 2) * room_of(p) * 4 + plan_bytes(p));
}

hipError_t launch_paged_attn(const SharedParams& p, int D, hipStream_t stream) {
    if (!together(p)) return launch_paged_attn(static_cast<const PagedParams&>(p), D, stream);
    if (D == 128) return p.fp16 ? launch_shared<FP16, 128>(p, stream) : launch_shared<BF16, 128>(p, stream);
    return p.fp16 ? launch_shared<FP16, 64>(p, stream) : launch_shared<BF16, 64>(p, stream);
}

}  // namespace kda
