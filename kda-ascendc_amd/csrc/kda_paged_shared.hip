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
// each.  The join, which also works on the own keys of sequences that have few.
//
// 64 answers with 10 to 500 tokens of their own behind 16000, 32 / 8 heads: 47 us
// (390 to 400 one by one), where the keys read once at 5.2 TB/s are 19 and the products at
// 1.4 PFLOP/s 12.  The plan takes 4.5: its loads, three sums over the work-group.
// The parts 29: 1.8 until a work-group has its unit, 3 until its first keys, 16.5
// for 8 times two tiles (the matrix unit and the softmax in turn, as in
// many_rows()), 3 for the groups' join and the stores, the rest the kernel's
// beginning and end.  The join 14: 1 until it has its records, 11 for the longest
// own keys (4 tiles a wave one after the other; 5 in the middle), 2 for 16 parts.
#include "kda_paged_attn.h"

namespace kda {
namespace {

// Rows of a tile: fewer than a work-group's waves have, whose two groups of four
// have the same rows and go over keys of their own, every other tile.  Where a
// prefix is cut for the whole card the parts then leave half the partial results
// that they would with 256 rows (64 sequences of 4 heads a kv head behind 16000
// tokens: 17 MB instead of 34, 46 us instead of 50).
constexpr int MT = 128;
// Rows of a sequence's own tiles (but for a last one of up to MT) where there are
// enough of them for some rounds: as without groups, half as many beginnings and
// ends.  WIDE row tiles of MT rows, which 256 CUs work on in three rounds: 8 chunks
// of up to 2048 tokens behind 12000 771 -> 701 us (690 one by one), 2 of up to 4000
// behind 30000 1965 -> 1856 (1802).  With fewer the parts are coarser: 8 of up to
// 512 behind 12000 take 251 us so instead of 196, 4 of up to 300 158 instead of 137.
constexpr int WIDE_MT = Shape<MANY>::MT, WIDE = 3 * Shape<MANY>::SLOTS;

// Sequences, and groups, that a plan has room for (in LDS); more go one by one.
constexpr int MOST = 2048;

// What is worked on together: the queries of a group over its shared tokens, or
// those of a sequence over its own.  Records of all groups, then of all
// sequences.
struct alignas(16) Work {
    int first, count, len, pos;  // as NewTokens, `first` a token of all, or a group's of those that share
    int from, row;               // the first key, a row of the table
    int parts, mt;               // parts of a row tile's keys; row tiles
    int place;                   // of the partial results, in 4 rows; NONE, or OVER where there is no room or unit
    int group;                   // a sequence's record of shared tokens, -1: none
    int few, tiles;              // of few rows; tiles of keys
    int few_end, many_end;       // the units of few and of many rows up to this record's
    int sharer;                  // the first of its tokens among those that share
    int tile;                    // rows of a row tile
};
constexpr int NONE = -1, OVER = -2;

// The plan in the workspace: a head, the records, and the tokens that share (of
// each group one after the other: sequences that do not are left out).
constexpr int HEAD = 16;
struct Plan {
    int32_t* head;  // units of few rows, of many
    Work* work;
};
__device__ __forceinline__ Plan plan_of(const SharedParams& p) {
    return {p.plan, reinterpret_cast<Work*>(p.plan + HEAD)};
}
int64_t tokens_of(const SharedParams& p) { return p.cu_seqlens ? p.T : (int64_t)p.N * p.T; }
// Tokens that share at most: of each sequence fewer than fill a row tile.
int64_t sharing_tokens(const SharedParams& p) { return std::min(tokens_of(p), (int64_t)p.N * (MT / p.G + 1)); }
int64_t plan_bytes(const SharedParams& p) {
    return HEAD * 4 + ((int64_t)p.NG + p.N) * (int64_t)sizeof(Work) + 4 * sharing_tokens(p);
}

// Rows of a tile of partial results: a multiple of 4.
__host__ __device__ inline int padded(int rows) { return (rows + 3) & ~3; }

// Numbers of a thread, and their sums up to it (its own included) and over all of
// the work-group's; those from PLAIN on and their sums no more than LIMIT.
template <int K>
struct Numbers {
    uint32_t x[K] = {};
};
constexpr uint32_t LIMIT = 0x7fffffff;
template <int THREADS, int PLAIN, int K>
__device__ __forceinline__ Numbers<K> scan(const Numbers<K>& x, uint32_t (&lds)[K][16], Numbers<K>& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Numbers<K> s;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        s.x[k] = k < PLAIN ? wave_prefix(x.x[k]) : wave_prefix(x.x[k], LIMIT);
        if (lane == 63) lds[k][wave] = s.x[k];
    }
    __syncthreads();
    all = {};
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w)
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (w == wave) s.x[k] += all.x[k];
            all.x[k] += lds[k][w];
            if (k >= PLAIN) {
                s.x[k] = min(s.x[k], LIMIT);
                all.x[k] = min(all.x[k], LIMIT);
            }
        }
    return s;
}
__device__ __forceinline__ uint32_t limited(int64_t x) { return (uint32_t)min(x, (int64_t)LIMIT); }

// Of sequences that share, those with few rows and up to this many tiles of keys
// of their own have them worked on in the join: not in parts that would only
// begin when those of the prefixes are over.  With 8, 12, 16 and 24 tiles, single
// tokens of 32 / 8 heads, own tokens spread up to 500: 64 sequences behind 16000 62,
// 58, 54 and 54 us, 16 behind 8000 37, 38, 34 and 34, 8 behind 4000 20, 21, 22 and 22;
// up to 1000: 77, 76, 77 and 77, 44, 40, 41 and 43, 22, 22, 24 and 26; up to 2000: 102,
// 102, 103 and 106, 52, 52, 53 and 55, 22, 25, 25 and 27.  (40 drafts of 5, 24 / 4 heads
// of 64, behind 4000: up to 500 35, 35, 32 and 32, 1000 41, 41, 41 and 39, 2000 46, 46,
// 46 and 47; up to 200 own tokens all the same.)
constexpr int IN_JOIN = 16;
// Rounds of parts of many rows at most, on 256 CUs each.
constexpr int ROUNDS = 3;

// Parts that keys of few rows are cut into at most, two to four rounds of them: as
// many as run at once, or more that still have 4 tiles a wave (8 of head size 64, of
// half the bytes), as lengths are uneven and a round waits for its longest.  Decode,
// 32 / 8 heads: 32 pairs behind 8000 to 16000 tokens 335 -> 299 us, 16 fours behind 2000
// to 4000 72.5 -> 64.0, 4 groups of 16 behind 100 to 200 with up to 8000 of their own 165
// -> 146 (one by one 533, 145, 142); by 6 or 8 tiles a wave the fours take 72.5 again,
// with 1024 parts in any case 78.7.
constexpr int FEW_PARTS = 1024;

// One work-group.  `waves`: those of a work-group of few rows; `fine`: tiles of their
// parts where they are more than run at once; `rounds`: of parts of many rows, at
// most; `room`: of the partial results, in 4 rows; `grid`: units.  Both suffice
// whatever the lengths are; where offsets decrease, and sequences have more tokens
// than there are, what is past them is left out, and the join makes its rows NaN.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void paged_shared_plan_kernel(SharedParams p, int waves, int fine, int rounds, int room, uint32_t grid) {
    constexpr bool ONE = THREADS < 1024;  // a record a thread
    // (of the groups: their sequences' offsets, the first that shares, how many do,
    // with how many tokens; the shared ones.  Sharing tokens before each sequence.)
    __shared__ int cu[MOST + 1], least[MOST], sharing[MOST], tokens_of[MOST], shared_of[MOST], before[MOST + 1];
    __shared__ uint32_t lds5[5][16], lds3[3][16];
    const int tid = threadIdx.x, V = p.NG + p.N;
    const int each = ONE ? 1 : (V + THREADS - 1) / THREADS, v0 = tid * each, v1 = min(V, v0 + each);
    const int64_t most = (int64_t)p.M << p.page_shift;
    for (int g = tid; g <= p.NG; g += THREADS) {
        cu[g] = min(max(p.cu_groups[g], 0), p.N);
        if (g < p.NG) {
            const int len = p.shared_lens[g];
            shared_of[g] = len < 0 ? 0 : ((int64_t)len > most ? (int)most : len);
            least[g] = p.N;
            sharing[g] = tokens_of[g] = 0;
        }
    }
    NewTokens mine = {};  // (a record a thread: its sequence's)
    if (ONE && v0 >= p.NG && v0 < V) mine = new_tokens(p, v0 - p.NG);
    auto tokens = [&](int v) { return ONE ? mine : new_tokens(p, v - p.NG); };
    __syncthreads();
    // The group that sequence n shares with, -1 for none: if its new tokens all come
    // behind the group's shared ones, and do not fill a row tile by themselves (which
    // then has nothing to gain).
    auto group_of = [&](int n, const NewTokens& s) {
        int lo = 0, hi = p.NG - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (cu[mid] <= n) lo = mid;
            else hi = mid - 1;
        }
        const bool in = cu[lo] <= n && n < cu[lo + 1] && shared_of[lo] > 0 && s.pos >= shared_of[lo];
        return in && s.count > 0 && (int64_t)s.count * p.G < MT ? lo : -1;
    };
    for (int v = max(v0, p.NG); v < v1; ++v) {
        const NewTokens s = tokens(v);
        const int g = group_of(v - p.NG, s);
        if (g < 0) continue;
        atomicMin(&least[g], v - p.NG);
        atomicAdd(&sharing[g], 1);
        atomicAdd(&tokens_of[g], s.count);
    }
    __syncthreads();

    const Plan plan = plan_of(p);
    // Record v, but for its parts, their place and where its group's rows begin.
    auto record = [&](int v) {
        Work w = {};
        w.group = NONE;
        w.place = NONE;
        if (v >= p.NG) {
            const int n = v - p.NG;
            const NewTokens s = tokens(v);
            w.first = p.cu_seqlens ? s.first : n * p.T;
            w.count = s.count;
            w.len = s.len;
            w.pos = s.pos;
            w.row = n;
            const int g = group_of(n, s);
            if (g >= 0 && sharing[g] >= 2) {
                w.group = g;
                w.from = shared_of[g];
            }
        } else if (sharing[v] >= 2) {
            w.count = tokens_of[v];
            w.len = w.pos = shared_of[v];
            w.row = least[v];
        }
        w.few = (int64_t)w.count * p.G <= ROWS;
        const int shift = w.few ? 5 : 6;
        static_assert(Shape<FEW>::TK == 32 && Shape<MANY>::TK == 64, "keys a tile");
        w.tile = w.few ? ROWS : MT;
        w.mt = (int)(((int64_t)w.count * p.G + w.tile - 1) / w.tile);
        w.tiles = max(1, (int)(((uint32_t)w.len + (1u << shift) - 1) >> shift) - (w.from >> shift));
        return w;
    };
    // Whether the join works on a record's keys.
    auto in_join = [&](const Work& w) { return w.few && w.group >= 0 && w.tiles <= IN_JOIN; };
    Work w;
    // records of few rows, tokens that share, row tiles of many; tiles of few, of many
    Numbers<5> x, all;
    for (int v = v0; v < v1; ++v) {
        w = record(v);
        if (w.group >= 0) x.x[1] += w.count;
        if (w.count > 0 && !in_join(w)) {
            if (w.few) {
                x.x[0] += p.HKV;
                x.x[3] = limited(x.x[3] + (int64_t)w.tiles * p.HKV);
            } else {
                x.x[2] += w.mt * p.HKV;
                x.x[4] = limited(x.x[4] + (int64_t)w.mt * p.HKV * w.tiles);
            }
        }
        if (!ONE) plan.work[v] = w;
    }
    const Numbers<5> upto5 = scan<THREADS, 3>(x, lds5, all);
    // Few rows: parts of `size` tiles, as many as run at once, or up to FEW_PARTS that
    // are still of `fine` tiles.  (Of LIMIT tiles, which are seconds of work, none
    // is cut.)
    const uint32_t slots = few_slots(waves), once = (all.x[3] + slots - 1) / slots;
    const uint32_t finer = max((all.x[3] + FEW_PARTS - 1) / FEW_PARTS, min(once, (uint32_t)fine));
    const uint32_t size = all.x[3] < LIMIT ? max((uint32_t)waves, finer) : LIMIT;
    // Many rows: with `units` row tiles of `tiles` tiles of keys together, `share`
    // parts of equal size if they can be had, in 1 to 3 rounds: the fewest tiles one
    // after the other, 7 more a round for its beginning and end (a tile of 128 rows
    // takes 1 us).  A few parts of few rows run in the first round too.  (Of LIMIT
    // tiles, which are hours of work, none is cut.)
    const bool wide = all.x[2] >= WIDE;
    const uint32_t units = wide ? all.x[2] / 2 : all.x[2], tiles = all.x[4], beside = all.x[3] / size + all.x[0];
    uint32_t share = 0;
    float best = 3.4e38f;
    for (int r = 1; r <= rounds && tiles < LIMIT; ++r) {
        const uint32_t most = r * Shape<MANY>::SLOTS - (beside <= Shape<MANY>::SLOTS / 4 ? beside : 0);
        const uint32_t k = units > 0 ? most / units : 0;
        const float cost = k > 0 ? r * ((float)tiles / (float)(units * k) + 7.f) : best;
        if (cost < best) {
            best = cost;
            share = most;
        }
    }
    // A record's parts; units of few and of many rows, and the room of its results.
    auto needs = [&](Work& w, int v) {
        Numbers<3> x;
        if (w.count == 0 || in_join(w)) return x;
        if (w.few) {
            w.parts = (int)((w.tiles + size - 1) / size);
            x.x[0] = w.parts * p.HKV;
        } else {
            w.parts = 1;
            uint32_t own = share;
            if (wide && v >= p.NG) {
                // (a row tile of twice the rows has twice the parts)
                const uint32_t narrow = (uint32_t)(((int64_t)w.count * p.G + MT - 1) / MT), mt = (narrow + 1) / 2;
                own = 2 * share - (narrow & 1 ? (share + mt - 1) / mt : 0);
                w.tile = WIDE_MT;
                w.mt = mt;
            }
            if (share > 0) {
                // (exact: the quotient of 32 bits by 32 is no nearer to a whole number than 2^-32)
                const uint32_t parts = (uint32_t)((double)w.tiles * (double)own / (double)tiles);
                w.parts = (int)max(1u, min((uint32_t)w.tiles / Shape<MANY>::LEAST, parts));
            }
            x.x[1] = w.mt * w.parts * p.HKV;
        }
        if (w.parts > 1 || v < p.NG || w.group >= 0) x.x[2] = limited((int64_t)(padded(w.count * p.G) / 4) * w.parts * p.HKV);
        return x;
    };
    Numbers<3> mine3, x3, all3;
    int sharers = upto5.x[1] - x.x[1];
    for (int v = v0; v < v1; ++v) {
        if (!ONE) w = plan.work[v];
        x3 = needs(w, v);
        mine3.x[0] += x3.x[0];
        mine3.x[1] += x3.x[1];
        mine3.x[2] = limited((int64_t)mine3.x[2] + x3.x[2]);
        if (v >= p.NG) {
            before[v - p.NG] = sharers;
            if (w.group >= 0) sharers += w.count;
        }
    }
    if (tid == 0) before[p.N] = all.x[1];
    const Numbers<3> upto = scan<THREADS, 2>(mine3, lds3, all3);  // (which waits for all of `before`)
    Numbers<3> at;
#pragma unroll
    for (int k = 0; k < 3; ++k) at.x[k] = upto.x[k] - mine3.x[k];
    for (int v = v0; v < v1; ++v) {
        if (!ONE) {
            w = plan.work[v];
            x3 = needs(w, v);
        }
        if (x3.x[2] > 0) w.place = upto.x[2] < LIMIT && at.x[2] + x3.x[2] <= (uint32_t)room ? (int)at.x[2] : OVER;
#pragma unroll
        for (int k = 0; k < 3; ++k) at.x[k] += x3.x[k];
        w.few_end = at.x[0];
        w.many_end = at.x[1];
        if (w.parts > 0 && (w.few ? all3.x[1] + at.x[0] : at.x[1]) > grid) w.place = OVER;
        if (v < p.NG) {
            w.first = w.sharer = before[cu[v]];
        } else {
            w.sharer = before[v - p.NG];
            if (w.group >= 0)
                for (int i = 0; i < w.count && w.sharer + i < p.map_size; ++i) p.map[w.sharer + i] = w.first + i;
        }
        plan.work[v] = w;
    }
    if (tid == THREADS - 1) {
        plan.head[0] = all3.x[0];
        plan.head[1] = all3.x[1];
    }
}

// Four rows of partial results in floats: m and l, then O.
template <int D>
constexpr int64_t FOUR = 4 * (D + 2);

// Where the part-th part of row tile m of (w, kv head h) is, of `rows` rows.
template <int D>
__device__ __forceinline__ int64_t place_of(const SharedParams& p, const Work& w, int m, int h, int part, int rows) {
    return FOUR<D> * (w.place + (int64_t)m * (w.tile / 4) * p.HKV * w.parts + (h * w.parts + part) * (rows / 4));
}
__device__ __forceinline__ int tile_rows(const SharedParams& p, const Work& w, int m) {
    return padded(min(w.tile, w.count * p.G - m * w.tile));
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
    w.sharer = at[14];
    w.tile = at[15];
    return w;
}

// ---- many rows ----

// The two groups' products and softmax alternate as in many_rows(), and so do
// their tiles: group g's are g, g + 2 and so on.
//   slot     t (even)                        t + 1
//   group 0  products: V(t - 2), K(t)        loads K(t + 3), V(t + 1); softmax(t)
//   group 1  loads K(t + 2), V(t); softmax(t - 1)   products: V(t - 1), K(t + 1)
// The group that does the softmax loads for the other: a tile is waited for by
// its loader at the end of the next slot and read in the one after that.  So a
// tile needs its place for three slots, and the tiles of either parity have two
// places each: 4 tiles of keys, 4 of values.
template <class E, int D>
__device__ __forceinline__ void split_rows(const SharedParams& p, const Unit& u, uint8_t* kt, uint8_t* vt, float* joint) {
    constexpr int STEPS = D / 16, DB = D / 32, TK = Shape<MANY>::TK;
    constexpr int TILE = TK * D * 2, SHARE = TK / 4;  // keys that a wave loads of a tile
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = wave >> 2, in = wave & 3;
    const int row = in * ROWS + (lane & 31);
    const Row x = row_of(p, u, u.m * MT + row);
    const int count = u.end - u.begin;
    // the keys that every row of this wave sees, and those that any does
    const int all_hi = __builtin_amdgcn_readlane(x.hi, 0);
    const int any_hi = u.m * MT + in * ROWS < u.s.count * p.G ? __builtin_amdgcn_readlane(x.hi, 31) : 0;
    const float c = p.scale * LOG2E;
    Running run;
    f32x16 acc[DB], st[2];
    u32x4 pt[4];
#pragma unroll
    for (int i = 0; i < DB; ++i) acc[i] = f32x16{};

    const Loader<D, SHARE, false> k0(p.k, p.k_page, p.k_token, u.h * p.k_head, 0, lane);
    const Loader<D, SHARE, false> v0(p.v, p.v_page, p.v_token, u.h * p.v_head, 0, lane);
    // Where this wave's keys lie of 64 tiles of the other group's, j on (the tile
    // 2 j + 1 - g is its j-th).  Past the last: nothing, zeros.
    Place k_of, v_of;
    auto places = [&](int j) {
        const int t = 2 * (j + lane) + 1 - g;
        const int key = (u.begin + min(t, count)) * TK + SHARE * in;
        const int at = min(key >> p.page_shift, p.M - 1);
        const int page = t < count ? p.page_table[u.n * p.table_stride + at] : -1;
        k_of = k0.place(p, u, page, key);
        v_of = v0.place(p, u, page, key);
    };
    // places of tile t: parity, then every other
    auto place = [&](uint8_t* ring, int t) { return lds_address(ring) + ((t & 1) * 2 + ((t >> 1) & 1)) * TILE + in * (SHARE * D * 2); };
    auto load = [&](const Loader<D, SHARE, false>& of, const Place& at, int j, uint8_t* ring, int t) {
        of.load(of_lane(at, j & 63), place(ring, t));
    };
    // The loads in slot t: keys of tile t + 2 and values of tile t, the other group's.
    auto begin_loads = [&](int t) {
        const int j = (t - 1 + g) >> 1;
        // (the values' places of 64 tiles are the keys' before the next ones are found)
        load(v0, v_of, j, vt, t);
        if (((j + 1) & 63) == 0) places(j + 1);
        load(k0, k_of, j + 1, kt, t + 2);
    };
    places(0);
    load(k0, k_of, 0, kt, 1 - g);
    u32x4 q[STEPS];
    load_q<D>(p, u, x, half, q);

    auto key_of = [&](int t) { return (u.begin + t) * TK; };
    auto sees = [&](int t) { return (unsigned)t < (unsigned)count && key_of(t) < any_hi; };
    auto softmax = [&](int t) {
        if (!sees(t)) return;
        float alpha;
        const int key = key_of(t);
        if (softmax_tile<E, false>(st, key + 4 * half, x.lo, x.hi, 0, key < u.lo || key + TK > all_hi, c, run, pt, alpha)) {
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[d] *= alpha;
        }
    };
    const uint8_t *kg = kt + g * 2 * TILE, *vg = vt + g * 2 * TILE;
    const int steps = (count + 1) / 2;
    // This group's s-th tile, in place I = s % 2.
    auto step = [&](int s, auto I) {
        const int t = 2 * s + g;
        __builtin_amdgcn_s_setprio(1);
        if (s > 0 && sees(t - 2)) tile_outputs<E, D>(vg + (1 - I) * TILE, pt, acc, lane);
        if (sees(t)) tile_scores<E, D>(kg + I * TILE, q, st, lane);
        __builtin_amdgcn_s_setprio(0);
        wait_loads<0>();
        meet();
        begin_loads(t + 1);
        softmax(t);
        if (g == 0 || s + 1 < steps) meet();
    };
    if (count > 0) {
        // (where the compiler sees it: else it waits for q in every turn)
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt 0
        meet();
        if (g == 1) {
            begin_loads(0);
            meet();
        }
        for (int s = 0; s < steps; s += 2) {
            step(s, std::integral_constant<int, 0>{});
            if (s + 1 < steps) step(s + 1, std::integral_constant<int, 1>{});
        }
        wait_loads<0>();
        meet();
        const int last = 2 * (steps - 1) + g;
        if (sees(last)) tile_outputs<E, D>(vg + ((steps - 1) & 1) * TILE, pt, acc, lane);
    }
    // Join: the second group's sums through LDS, each lane's to the lane with the
    // same row and elements.
    run.l = sum_halves(run.l);
    __syncthreads();  // (all have read their values)
    f32x4* o = reinterpret_cast<f32x4*>(kt) + in * 64 + lane;
    if (g == 1) {
        if (half == 0) {
            joint[row] = run.log2_max();
            joint[MT + row] = run.l;
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[(4 * d + i) * 256] = f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
    }
    __syncthreads();
    if (g == 1 || !x.live) return;
    const float m0 = run.log2_max(), m1 = joint[row], top = fmaxf(m0, m1), sub = top == -INFINITY ? 0.f : top;
    const float f0 = fast_exp2(m0 - sub), f1 = fast_exp2(m1 - sub);
    const float l = fmaf(f1, joint[MT + row], run.l * f0);
    float* part = u.place >= 0 ? p.ws + u.place : nullptr;
    const float inv = part ? 1.f : (l > 0.f ? 1.f / l : 0.f);
    const int64_t out = out_row(p, u, x);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 theirs = o[(4 * d + i) * 256];
            f32x4 sum;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = fmaf(f1, theirs[e], acc[d][4 * i + e] * f0) * inv;
            const int at = 32 * d + 8 * i + 4 * half;
            if (part) *reinterpret_cast<f32x4*>(part + 2 * u.rows + row * D + at) = sum;
            else store_o<E, D>(p, out, at, sum[0], sum[1], sum[2], sum[3]);
        }
    if (half == 0) {
        if (part) {
            part[row] = top;
            part[u.rows + row] = l;
        } else if (p.lse) {
            p.lse[out] = log_sum(top, l);
        }
    }
}

// ---- parts ----

// Unit x of kind KIND; false where its results have no room.  Every lane has a
// record: no load waits for another (but for every 64 records more).
template <int KIND, int D>
__device__ __forceinline__ bool unit_of(const SharedParams& p, const Plan& plan, int x, int lane, Unit& u) {
    constexpr int TK = Shape<KIND>::TK;
    const int V = p.NG + p.N;
    Work w = {};
    int before = 0;
    for (int v0 = 0; v0 < V; v0 += 64) {
        const Work mine = plan.work[min(v0 + lane, V - 1)];
        const int end = KIND == FEW ? mine.few_end : mine.many_end;
        const uint64_t past = __ballot(end > x);
        if (past) {
            const int at = __builtin_ctzll(past);
            if (at > 0) before = __builtin_amdgcn_readlane(end, at - 1);
            auto take = [&](int y) { return __builtin_amdgcn_readlane(y, at); };
            w.first = take(mine.first);
            w.count = take(mine.count);
            w.len = take(mine.len);
            w.pos = take(mine.pos);
            w.from = take(mine.from);
            w.row = take(mine.row);
            w.parts = take(mine.parts);
            w.mt = take(mine.mt);
            w.place = take(mine.place);
            w.tile = take(mine.tile);
            u.mapped = v0 + at < p.NG;
            break;
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    if (w.place == OVER || w.count == 0) return false;
    x -= before;
    // heads innermost, as the XCDs go round; row tiles that see the most keys first
    u.n = w.row;
    u.h = x % p.HKV;
    x /= p.HKV;
    const int part = x % w.parts;
    u.m = w.mt - 1 - x / w.parts;
    u.s = NewTokens{w.first, w.count, w.len, w.pos};
    const int last = (min(w.count * p.G, u.m * w.tile + w.tile) - 1) / p.G;
    u.lo = w.from;
    u.hi = max(w.from, min(w.pos + last + 1, w.len));
    const int t0 = u.lo / TK;
    const int64_t tiles = max(t0, (u.hi + TK - 1) / TK) - t0;
    u.begin = t0 + (int)(tiles * part / w.parts);
    u.end = t0 + (int)(tiles * (part + 1) / w.parts);
    u.rows = tile_rows(p, w, u.m);
    u.place = w.place == NONE ? -1 : place_of<D>(p, w, u.m, u.h, part, u.rows);
    if (KIND == MANY && u.rows <= MT) u.m *= w.tile / MT;  // (as split_rows counts)
    return true;
}

// A part a work-group, those of many rows first (the grid is what the host knows
// that there can be at most).  LONG: where there may be WIDE row tiles (in the
// others' kernel their code costs 1 %: 8 packed questions behind 12000 196 -> 198
// us, 16 chunks of up to 16 tokens 97.7 -> 99.2).
template <class E, int D, int KIND, bool LONG>
__global__ __launch_bounds__(KIND == FEW ? 256 : 512, 2) void paged_shared_kernel(SharedParams p) {
    constexpr int WAVES = Shape<KIND == FEW ? FEW : MANY>::WAVES;
    typedef FewLds<D, WAVES> Lds;
    __shared__ alignas(1024) uint8_t lds[WAVES * Lds::EACH];
    static_assert(WAVES == 4 || sizeof(lds) == 8 * Shape<MANY>::TK * D * 2, "four tiles of keys, four of values");
    __shared__ float joint[WAVES * 2 * ROWS];
    const int lane = threadIdx.x & 63, id = blockIdx.x;
    const Plan plan = plan_of(p);
    typedef __attribute__((address_space(4))) const int32_t c_i32;
    const int few = ((c_i32*)plan.head)[0], many = ((c_i32*)plan.head)[1];
    if (id >= few + many) return;
    // (of few rows only there are no others, unless the offsets are none)
    if (KIND == FEW && id < many) return;
    Unit u;
    if (KIND == FEW || id >= many) {
        if (unit_of<FEW, D>(p, plan, id - many, lane, u))
            few_rows<E, D, WAVES>(p, u, Lds{lds, lds + 3 * Lds::EACH, lds + 6 * Lds::EACH}, joint);
    } else if constexpr (KIND != FEW) {
        if (!unit_of<MANY, D>(p, plan, id, lane, u)) return;
        if constexpr (LONG) {
            if (u.rows > MT) {
                many_rows<E, D>(p, u, lds, lds + sizeof(lds) / 2);
                return;
            }
        }
        split_rows<E, D>(p, u, lds, lds + sizeof(lds) / 2, joint);
    }
}

// Where the partial results of a row are: `parts` of them, `step` floats apart,
// each of R rows with this one the r-th.
struct Parts {
    const float* first;
    int64_t step;
    int parts, R, r;
    __device__ __forceinline__ const float* at(int j) const { return first + j * step; }
};
template <int D>
__device__ __forceinline__ Parts parts_of(const SharedParams& p, const Work& w, int h, int row) {
    Parts x;
    const int m = row / w.tile;
    x.r = row - m * w.tile;
    x.R = tile_rows(p, w, m);
    x.first = p.ws + place_of<D>(p, w, m, h, 0, x.R);
    x.step = (x.R / 4) * FOUR<D>;
    x.parts = w.parts;
    return x;
}
__device__ __forceinline__ void add(Sums& s, float mx, float sum, const f32x4& o) {
    const float top = fmaxf(s.mx, mx), sub = top == -INFINITY ? 0.f : top;
    const float f0 = fast_exp2(s.mx - sub), f = fast_exp2(mx - sub);
    s.mx = top;
    s.sum = fmaf(f, sum, s.sum * f0);
#pragma unroll
    for (int i = 0; i < 4; ++i) s.o[i] = fmaf(f, o[i], s.o[i] * f0);
}
// Parts from, from + by and so on of four elements of a row, in one pass, so that
// no load waits for another.
__device__ __forceinline__ void add_parts(Sums& s, const Parts& x, int piece, int D, int from, int by) {
#pragma unroll 8
    for (int j = from; j < x.parts; j += by) {
        const float* part = x.at(j);
        add(s, part[x.r], part[x.R + x.r], *reinterpret_cast<const f32x4*>(part + 2 * x.R + x.r * D + piece * 4));
    }
}

// Joins the parts of (sequence n, kv head h): those of its group's shared tokens
// and its own, or its own keys worked on here where they are few (by each of its
// up to `groups` work-groups, which divide the joining).  Four elements of a row a
// thread; where rows are few, several threads' parts in turn.
template <class E, int D>
__global__ __launch_bounds__(256, 2) void paged_shared_join_kernel(SharedParams p, int groups, int fours) {
    constexpr int WAVES = Shape<FEW>::WAVES;
    typedef FewLds<D, WAVES> Lds;
    __shared__ alignas(1024) uint8_t lds[WAVES * Lds::EACH];
    __shared__ float joint[WAVES * 2 * ROWS];
    __shared__ float sums[6 * 256];
    const Plan plan = plan_of(p);
    // (the first work-groups of all first, as of the others many have nothing to do:
    // 64 packed single tokens behind 16000 47.5 us, with each one's together 90.9)
    const int pairs = p.N * p.HKV, group0 = blockIdx.x / pairs, id = blockIdx.x - group0 * pairs;
    const int n = id / p.HKV, h = id - n * p.HKV;
    const Work w = load_work(plan, p.NG + n);
    const bool here = w.parts == 0;
    // work-groups that there is some use for: one for every `fours` fours, for 128 at
    // least where each works on the own keys (with one for every 64, 8 sequences of
    // 4 rows behind 2000 tokens took 18.2 us instead of 16.8)
    const int rows = w.count * p.G, items = rows * (D / 4);
    const int each = here ? max(128, fours) : fours, used = min(groups, (items + each - 1) / each);
    if (group0 >= used || (!here && w.place == NONE)) return;
    Work g = {};
    if (w.group >= 0) g = load_work(plan, w.group);
    if (w.place == OVER || g.place == OVER) {
        const float nan = __builtin_nanf("");
        for (int e = group0 * 256 + threadIdx.x; e < items; e += used * 256) {
            const int r = e / (D / 4), piece = e % (D / 4), tok = r / p.G;
            const int64_t out = ((int64_t)w.first + tok) * p.HQ + h * p.G + (r - tok * p.G);
            store_o<E, D>(p, out, piece * 4, nan, nan, nan, nan);
            if (p.lse && piece == 0) p.lse[out] = nan;
        }
        return;
    }
    const Lds tiles = {lds, lds, lds};
    if (here) {
        Unit u;
        u.n = w.row;
        u.h = h;
        u.m = 0;
        u.s = NewTokens{w.first, w.count, w.len, w.pos};
        u.mapped = false;
        u.lo = w.from;
        u.hi = w.len;
        u.begin = w.from / Shape<FEW>::TK;
        u.end = (w.len + Shape<FEW>::TK - 1) / Shape<FEW>::TK;
        few_sums<E, D, WAVES>(p, u, tiles, joint);
    }
    // threads an item: 1, 2 or 4
    const int shift = items > 128 * used ? 0 : (items > 64 * used ? 1 : 2), per = 256 >> shift;
    const int slice = threadIdx.x / per, item = threadIdx.x % per;
    for (int group = group0; group * per < items; group += used) {
        const int e = group * per + item, r = e / (D / 4), piece = e % (D / 4);
        const bool live = r < rows;
        Sums s = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
        if (live) {
            if (here && slice == 0) s = few_sum<D, WAVES>(tiles, joint, r, piece);
            const int rg = (w.sharer - g.sharer) * p.G + r;  // its place in the group's rows
            if (w.group >= 0 && rg >= 0 && rg < g.count * p.G) add_parts(s, parts_of<D>(p, g, h, rg), piece, D, slice, 1 << shift);
            if (!here) add_parts(s, parts_of<D>(p, w, h, r), piece, D, slice, 1 << shift);
        }
        if (shift > 0) {
            const int t = threadIdx.x;
            sums[t] = s.mx;
            sums[256 + t] = s.sum;
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[(2 + i) * 256 + t] = s.o[i];
            __syncthreads();
            if (slice == 0)
                for (int k = 1; k < 1 << shift; ++k) {
                    const int j = k * per + item;
                    add(s, sums[j], sums[256 + j], f32x4{sums[512 + j], sums[768 + j], sums[1024 + j], sums[1280 + j]});
                }
            __syncthreads();
        }
        if (live && slice == 0) {
            const float inv = s.sum > 0.f ? 1.f / s.sum : 0.f;
            const int tok = r / p.G;
            const int64_t out = ((int64_t)w.first + tok) * p.HQ + h * p.G + (r - tok * p.G);
            store_o<E, D>(p, out, piece * 4, s.o[0] * inv, s.o[1] * inv, s.o[2] * inv, s.o[3] * inv);
            if (p.lse && piece == 0) p.lse[out] = log_sum(s.mx, s.sum);
        }
    }
}

// ---- launches ----

// Rows of a sequence from which on a dense call is no different from one without
// groups: a row tile of the ordinary kernels'.
constexpr int WHOLE = Shape<MANY>::MT;

// Whether a plan has room for the sequences, and the table so many keys that one
// may pay.
//
// Where the table is so small that reading the shared keys again for each
// sequence costs less than the plan and the longer join, 15 us for 9, it does not:
// by the bytes that its rows have room for, whose second reading is from the caches.
// (The lengths are on the device: a wide table of short rows takes the three
// launches, 8 sequences behind 2000 tokens in rows of 8000 pages 17.4 us instead of
// 14.0, 2 16.8 instead of 10.3, 64 behind 100 22.8 instead of 15.8.)  Decode
// of 8 sequences, 32 / 8 heads: 67 MB 15.3 us one by one and 17.9 so, 131 MB 21.3
// and 19.4; 2 sequences: 66 MB 18.9 and 22.1, 131 MB 29.0 and 26.5.  Drafts of 5, 24
// / 4 heads of 64 (30 rows: their row tiles are full one by one too): 131 MB 24.4
// and 27.8, 262 MB 35.9 and 33.5.
//
// Nor where rows have room for no more keys than the ordinary kernel takes whole:
// one launch then instead of three, up to two rounds of its work-groups. Decode of
// sequences behind 400 to 700 shared tokens, 32 / 8 heads: 64 13.8 to 17.4 us one by
// one and 26.9 so, 128 24.2 to 32.7 and 33.4 to 33.9, but 256 (four rounds) 45 to 59
// and 48 to 49; 32 / 16 heads: 64 23.9 to 34.0 and 32.7 to 33.7, 128 44 to 63 and 44
// to 46; 800 keys, cut and joined: 64 36.5 and 26.1. (Packed single tokens are in
// the launch with many rows: 64 behind 100 to 700 26 to 38 and 26 to 30.)
bool planned(const SharedParams& p, int D) {
    if (p.N < 2 || p.N > MOST || p.NG > MOST || (!p.cu_seqlens && (int64_t)p.T * p.G >= WHOLE)) return false;
    const bool few = !p.cu_seqlens && (int64_t)p.T * p.G <= ROWS;
    if (few && !may_cut(static_cast<const PagedParams&>(p), FEW) && (int64_t)p.N * p.HKV <= 2 * Shape<FEW>::SLOTS) return false;
    const int64_t row = ((int64_t)p.M << p.page_shift) * p.HKV * D * 4;
    const int64_t least = tokens_of(p) * p.G <= (int64_t)p.N * (ROWS / 2) ? 112 << 20 : 224 << 20;
    return row >= least / p.N;
}
// Dense calls of more rows a sequence than fill a row tile, of which the plan lets
// none share.  In its row tiles of 128, the second one filled in part, they are
// slower than one by one in one of 256 (32 / 8 heads, 160 rows: 8 sequences behind
// 12000 tokens 98 us one by one and 150 so, 32 264 and 310, 64 behind 2000 114 and
// 123; 24 / 4 heads of 64, 162 rows: 64 behind 12000 212 and 253), but where row tiles
// are a quarter to a half of the CUs, which the ordinary kernel cuts in two or three
// and the plan in three to five (24 / 4 heads of 64: 32 behind 12000 216 and 130, behind
// 2000 52 and 37; 8 / 8 heads: 16 behind 7400 176 and 128).  Of 90 random calls the
// former took 0.93 of their time in groups one by one, the latter 1.22 of it.
// Of 128 rows, which share no more, one row tile is full and 256 rows are
// half empty: 8 behind 12000 88 and 75, 32 229 and 195, 64 behind 2000 102 and 93.
bool alone(const SharedParams& p) {
    const int64_t tiles = (int64_t)p.N * p.HKV;
    return !p.cu_seqlens && (int64_t)p.T * p.G > MT && (tiles <= Shape<MANY>::SLOTS / 4 || tiles > Shape<MANY>::SLOTS / 2);
}
// Whether sequences are worked on together at all.
bool together(const SharedParams& p, int D) { return planned(p, D) && !alone(p); }
bool few_only(const SharedParams& p) { return tokens_of(p) * p.G <= ROWS; }

// Row tiles of many rows at most.  Records of many rows have more than ROWS.
int64_t row_tiles(const SharedParams& p) {
    if (few_only(p)) return 0;
    const int64_t rows = tokens_of(p) * p.G;
    const bool members = p.cu_seqlens || (int64_t)p.T * p.G > ROWS;
    const int64_t records = std::min(std::min(p.NG, p.N / 2) + (members ? p.N : 0), (int)std::min((members ? 2 : 1) * rows / ROWS, (int64_t)MOST * 2));
    return (records + (members ? 2 : 1) * rows / MT) * p.HKV;
}
// Whether there may be WIDE row tiles.
bool may_be_wide(const SharedParams& p) { return row_tiles(p) >= WIDE; }
// Rounds of parts of many rows (two and more only with more than half as many row
// tiles as CUs: fewer are cut well in one).
int rounds_of(const SharedParams& p) {
    const int64_t tiles = row_tiles(p);
    return tiles == 0 ? 0 : tiles <= Shape<MANY>::SLOTS / 2 ? 1 : ROUNDS;
}

// Room of the partial results, in 4 rows: twice the rows that may be worked on
// together (a group's and the sequences', each filled up to 4), and the parts
// that keys are cut into.
int64_t room_of(const SharedParams& p) {
    const int64_t rows = (2 * sharing_tokens(p) * p.G + 3 * (int64_t)(p.N + p.NG)) * p.HKV;
    const int64_t few = (int64_t)FEW_PARTS * ROWS;
    const int64_t many = (int64_t)rounds_of(p) * Shape<MANY>::SLOTS * (may_be_wide(p) ? WIDE_MT : MT);
    return (rows + few + many + 3) / 4;
}

// Units at most: a record's heads and row tiles, and the parts more that keys
// are cut into.
int64_t units_of(const SharedParams& p) {
    const int64_t few = ((int64_t)p.N + std::min(p.NG, p.N / 2)) * p.HKV + FEW_PARTS;
    return few + row_tiles(p) + rounds_of(p) * Shape<MANY>::SLOTS;
}

template <class E, int D>
hipError_t launch_shared(SharedParams p, hipStream_t stream) {
    p.plan = reinterpret_cast<int32_t*>(p.ws + 4 * (D + 2) * room_of(p));
    p.map_size = (int)sharing_tokens(p);
    p.map = p.plan + HEAD + ((int64_t)p.NG + p.N) * (int64_t)(sizeof(Work) / 4);
    const int V = p.NG + p.N, room = (int)std::min(room_of(p), (int64_t)LIMIT - 1);
    const bool only = few_only(p);
    const int waves = Shape<FEW>::WAVES * (only ? 1 : 2), fine = 4 * waves * (128 / D);
    const dim3 grid((unsigned)units_of(p));
    if (V <= 256) paged_shared_plan_kernel<256><<<1, 256, 0, stream>>>(p, waves, fine, rounds_of(p), room, grid.x);
    else paged_shared_plan_kernel<1024><<<1, 1024, 0, stream>>>(p, waves, fine, rounds_of(p), room, grid.x);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (only) paged_shared_kernel<E, D, FEW, false><<<grid, 256, 0, stream>>>(p);
    else if (may_be_wide(p)) paged_shared_kernel<E, D, MIXED, true><<<grid, 512, 0, stream>>>(p);
    else paged_shared_kernel<E, D, MIXED, false><<<grid, 512, 0, stream>>>(p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    // Work-groups a (sequence, head): one for every 64 fours of its rows; where there
    // may be many rows, for so many fours that all rows together fill the card once
    // (8 tokens of each of 64 packed sequences behind 16000 tokens: 163 us, with one
    // for every 64 fours 276).  The grid has room for eight times as many, so that a
    // chunk among single tokens is divided too: 63 of them and a chunk of 300
    // tokens 175 us, with room for as many as run at once 412; the rest end at once.
    const int64_t pairs = (int64_t)p.N * p.HKV;
    const int64_t rows = std::min((int64_t)p.T * p.G, (int64_t)1 << 20);
    const bool many = rows > ROWS;
    const int64_t most = (many ? 8 : 1) * Shape<FEW>::SLOTS, all = tokens_of(p) * p.HQ * (D / 4);
    const int fours = (int)std::max((int64_t)64, many ? all / Shape<FEW>::SLOTS : 0);
    const int groups = (int)std::max((int64_t)1, std::min((rows * (D / 4) + fours - 1) / fours, most / pairs));
    paged_shared_join_kernel<E, D><<<dim3((unsigned)(pairs * groups)), 256, 0, stream>>>(p, groups, fours);
    return hipGetLastError();
}

}  // namespace

size_t paged_attn_workspace(const SharedParams& p, int D) {
    if (!together(p, D)) {
        // (the plan's few KB stay where there is room for one: callers that tell
        // the calls with one from paged_attention's do so by the size)
        const size_t one_by_one = paged_attn_workspace(static_cast<const PagedParams&>(p), D);
        return one_by_one + (planned(p, D) ? plan_bytes(p) : 0);
    }
    return (size_t)(4 * (D + 2) * room_of(p) * 4 + plan_bytes(p));
}

hipError_t launch_paged_attn(const SharedParams& p, int D, hipStream_t stream) {
    if (!together(p, D)) return launch_paged_attn(static_cast<const PagedParams&>(p), D, stream);
    if (D == 128) return p.fp16 ? launch_shared<FP16, 128>(p, stream) : launch_shared<BF16, 128>(p, stream);
    return p.fp16 ? launch_shared<FP16, 64>(p, stream) : launch_shared<BF16, 64>(p, stream);
}

}  // namespace kda
