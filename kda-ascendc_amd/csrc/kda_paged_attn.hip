// Attention of new tokens over a paged cache (kda_paged_hip.h).
//
// For each kv head the queries are rows: row r of sequence n is head r % G of
// its group and new token r / G, so that a key loaded once serves the whole
// group.  A work-group takes a tile of rows of one (sequence, kv head) and
// goes over the visible keys in tiles, one pass, with the running maximum m
// and sum l of the softmax:
//   s = scale * q.k,  m' = max(m, max s),  l' = l e^(m-m') + sum e^(s-m'),
//   o' = o e^(m-m') + sum e^(s-m') v;     o / l and m + ln l at the end.
//
// Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T, with
// 32x32x16 matrix ops.  A lane then holds one query (column lane & 31) and
// half of the keys of each block of 32: maximum and sum are sums within the
// lane and one exchange with lane ^ 32, and the rescaling of O^T is by a
// number of the lane's own.  The order of the keys inside a product is free,
// so P^T goes from the accumulators of the first product straight into the
// operand of the second, packed to 16 bits, and V^T's rows are read in the
// same order with transposing LDS reads.
#include "kda_common.h"
#include "kda_paged.h"

#include <algorithm>

namespace kda {
namespace {

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// Buffer descriptor word 3 for raw byte-addressed buffers.
constexpr int BUF_RAW = 0x00020000;

// Element types: the products and the packing of two floats (nearest even).
struct BF16 {
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack2(a, b); }
};
struct FP16 {
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
    }
};

constexpr int ROWS = 32;  // rows of a wave's products

// Two ways over the keys.  Few rows (a decode step, a draft): every wave of a
// work-group has the same 32 rows and keys of its own.  Many rows (a chunk):
// every wave has rows of its own, and the work-group's keys are shared.
constexpr int FEW = 0, MANY = 1, MIXED = 2;
template <int KIND>
struct Shape {
    static constexpr int WAVES = KIND == FEW ? 4 : 8;
    static constexpr int MT = KIND == FEW ? ROWS : WAVES * ROWS;  // rows a work-group
    static constexpr int TK = KIND == FEW ? 32 : 64;              // keys a tile
    // Tiles a work-group takes at least, where keys are split among several.
    static constexpr int LEAST = KIND == FEW ? 4 : 4;
    // Work-groups that run at once (LDS and registers: two of few rows on each
    // of 256 CUs, one of many): the parts that keys are split into.
    static constexpr int SLOTS = KIND == FEW ? 512 : 256;
    // Places for partial results in the workspace.
    static constexpr int PLACES = KIND == FEW ? 2 * SLOTS : SLOTS;
};

// A tile of keys (or values) in LDS: rows of D elements, in each the 16-byte
// piece c at place c ^ swizzle(row).  The swizzle keeps two reads free of bank
// conflicts: 16 rows at one piece (the first product's operand), and the
// transposing read's 4 rows at 4 consecutive pieces.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
    if constexpr (D == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// 16 bytes a lane from a buffer straight into LDS, lane l's to `lds` + 16 * l
// (a byte address, wave-uniform).  Written as an instruction: the compiler
// cannot tell the tiles of a ring apart and would wait, before any LDS read,
// for every such load under way.  So nothing but wait_loads() waits for it;
// it has no result in registers, and other loads' waits only become longer.
// The wait states: a buffer load may follow the lane read that wrote its
// descriptor's registers by 5, which the compiler sees to only for loads it
// knows.  Nothing else in these kernels uses m0.
// STREAM: for what is read once, past the caches' lines of other work (the
// decode step of 64 sequences of 3024 tokens, 32 / 8 heads: 141 us without,
// 124 us with, 6.4 TB/s; a long chunk's keys, read again by other work-groups,
// lose by it).
template <bool STREAM>
__device__ __forceinline__ void load_lds(u32x4 rsrc, int off, uint32_t lds) {
    if constexpr (STREAM)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen nt lds" ::"v"(off), "s"(rsrc),
                     "s"(lds)
                     : "memory");
    else
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc),
                     "s"(lds)
                     : "memory");
}
// One or two such loads at `AT` past `lds`, the second 1 KiB on.
template <int AT, int LOADS>
__device__ __forceinline__ void load_lds_at(u32x4 rsrc, const int (&off)[LOADS], uint32_t lds) {
    static_assert(LOADS <= 2, "one instruction each below");
    if constexpr (LOADS == 1)
        asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off[0]), "s"(rsrc),
                     "s"(lds), "i"(AT)
                     : "memory", "scc");
    else
        asm volatile("s_add_u32 m0, %3, %4\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %2, 0 offen lds\n\t"
                     "s_add_u32 m0, %3, %5\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"v"(off[0]),
                     "v"(off[LOADS - 1]), "s"(rsrc), "s"(lds), "i"(AT), "i"(AT + 1024)
                     : "memory", "scc");
}
// All but the last `n` of this wave's loads have arrived.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const uint8_t* p) {
    return (uint32_t)reinterpret_cast<uintptr_t>((lds_u8*)p);
}

// Operand of the first product: rows lane & 31, elements 16 * s + 8 * (lane >> 5) .. +7.
template <int D>
__device__ __forceinline__ const uint8_t* k_place(const uint8_t* lds, int row, int piece) {
    return lds + row * (D * 2) + ((piece ^ swizzle<D>(row)) << 4);
}
__device__ __forceinline__ u32x4 load_operand(uint32_t at) {
    typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
    return *reinterpret_cast<lds_u32x4*>(at);
}
template <int D>
__device__ __forceinline__ u32x4 read_k(const uint8_t* lds, int row, int piece) {
    return *reinterpret_cast<const u32x4*>(k_place<D>(lds, row, piece));
}

// Half an operand of the second product: lane's column d = 32 * db + (lane & 31)
// of rows key .. key + 3.  In each group of 16 lanes, lane n receives as item i
// element n % 4 of the 8 bytes that lane 4 * i + n / 4 points at.
template <int D>
__device__ __forceinline__ const uint8_t* v_place(const uint8_t* lds, int key, int db, int lane) {
    const int row = key + ((lane & 15) >> 2);
    const int d = 32 * db + (lane & 16) + 4 * (lane & 3);
    return lds + row * (D * 2) + (((d >> 3) ^ swizzle<D>(row)) << 4) + (d & 4) * 2;
}
__device__ __forceinline__ u32x2 load_transposed(uint32_t at) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4*>(at)));
}
template <int D>
__device__ __forceinline__ u32x2 read_v(const uint8_t* lds, int key, int db, int lane) {
    return load_transposed(lds_address(v_place<D>(lds, key, db, lane)));
}
// A number that the compiler takes as it is, where it stands: else it keeps, all
// along, whatever a kernel's addresses are made of, in more registers than there
// are.
__device__ __forceinline__ uint32_t hide(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Maximum and sum of x and the value of lane ^ 32: the swap exchanges the upper
// half of its first operand with the lower half of its second.  (The elements
// go through scalars: a bit cast of a vector's element takes the first one.)
struct Halves {
    float lower, upper;
};
__device__ __forceinline__ Halves halves(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ float max_halves(float x) {
    const Halves h = halves(x);
    return fmaxf(h.lower, h.upper);
}
__device__ __forceinline__ float sum_halves(float x) {
    const Halves h = halves(x);
    return h.lower + h.upper;
}

// The softmax over one tile's scores (16 * NB a lane, of keys key0 + 32 * b +
// 8 * (i / 4) + i % 4): its weights as operands of the second product, and the
// running m (in the scores' unit; c = scale * log2 e) and l.  Returns whether
// the sums so far have to shrink, by `alpha`.
// m follows the maximum only when a row's grows by more than a factor of 2^8
// (any m does as long as nothing overflows: weights stay at most 2^8, and fp32
// sums and 16-bit weights keep their relative precision), so that the rescaling
// of O, 64 multiplications a lane against the softmax's ~130 operations, is
// rare after the first tiles (a prompt of 8192 tokens: 557 us when m follows
// every growth, 522 so).
constexpr float GROWTH = 8.f;
struct Running {
    float m = -INFINITY;  // -inf: no key seen yet
    float mc = 0.f;       // m * c, or 0 with m = -inf: what the exponents subtract
    float l = 0.f;
    // (the two halves' sums joined) m * c for the join of several parts
    __device__ __forceinline__ float log2_max() const { return m == -INFINITY ? m : mc; }
};
template <class E, int NB>
__device__ __forceinline__ bool softmax_tile(f32x16 (&st)[NB], int key0, int lo, int hi, bool edge, float c,
                                             Running& run, u32x4 (&pt)[2 * NB], float& alpha) {
    if (edge) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = key0 + 32 * b + 8 * (i >> 2) + (i & 3);
                if (key < lo || key >= hi) st[b][i] = -INFINITY;
            }
    }
    float mx = st[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[b][i]);
    mx = max_halves(mx);
    const bool grow = __any((mx - run.m) * c > GROWTH);  // (-inf - -inf is no growth)
    if (grow) {
        const float m2 = fmaxf(run.m, mx), mc2 = m2 == -INFINITY ? 0.f : m2 * c;
        alpha = run.m == -INFINITY ? 0.f : fast_exp2(run.mc - mc2);
        run.m = m2;
        run.mc = mc2;
        run.l *= alpha;
    }
    const float sub = run.mc;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float e0 = fast_exp2(fmaf(st[b][i], c, -sub)), e1 = fast_exp2(fmaf(st[b][i + 1], c, -sub));
            sum += e0 + e1;
            pt[2 * b + (i >> 3)][(i & 7) >> 1] = E::pack(e0, e1);
        }
    run.l += sum;
    return grow;
}

// ---- the work and its split ----

// Row tile m of (sequence n, kv head h), the keys [lo, hi) that any of its rows
// sees, and which of their tiles [begin, end); `slot`: its place in the
// workspace, or -1 where these are all.
struct Unit {
    int n, h, m, lo, hi, begin, end, slot;
    NewTokens s;
};

// The keys that rows [m * MT, m * MT + MT) of a sequence see, and their tiles.
struct Tiles {
    int lo, hi, begin, end;
};
template <int KIND>
__device__ __forceinline__ Tiles tiles_of(const PagedParams& p, const NewTokens& s, int m) {
    constexpr int MT = Shape<KIND>::MT, TK = Shape<KIND>::TK;
    const int rows = s.count * p.G;
    const int first = m * MT / p.G, last = (min(rows, m * MT + MT) - 1) / p.G;
    const int hi = p.causal ? max(0, min(s.pos + last + 1, s.len)) : s.len;
    const int lo = p.window ? min(hi, max(0, s.pos + first + 1 - p.window)) : 0;
    return {lo, hi, lo / TK, max(lo / TK, (hi + TK - 1) / TK)};
}

// Lane `at`'s.
__device__ __forceinline__ NewTokens of_lane(const NewTokens& s, int at) {
    return {__builtin_amdgcn_readlane(s.first, at), __builtin_amdgcn_readlane(s.count, at),
            __builtin_amdgcn_readlane(s.len, at), __builtin_amdgcn_readlane(s.pos, at)};
}

// Whether a sequence is of the kind: packed ones are told apart by their rows.
template <int KIND>
__device__ __forceinline__ bool of_kind(const PagedParams& p, const NewTokens& s) {
    return s.count > 0 && (!p.cu_seqlens || (s.count * p.G <= ROWS) == (KIND == FEW));
}

// Few rows.  The tiles of all sequences and heads, one after the other (at
// least one a row tile, so that rows that see nothing are written too), are
// cut into pieces of `size`, one a work-group: the end of one row tile, whole
// ones, the start of another.  The two that a piece may not have whole go to
// places 2 b (its first) and 2 b + 1 of the workspace.  With many row tiles the
// pieces are the SLOTS that run at once, equal whatever the lengths (pieces of
// one row tile each left half of a second round empty).  With few each row
// tile is filled up to whole pieces, so that none has two, one after the other:
// SLOTS pieces hold what the tiles and the fillings come to.
// All work-groups come to the same cut, from the lengths on the device; every
// lane counts one sequence.
// !cut: row tiles whole, each filled up to a piece of FEW_WHOLE keys, which
// no row of the table exceeds.
constexpr int FEW_WHOLE = 24 * Shape<FEW>::TK;
struct Cut {
    uint32_t tiles, size;
    bool filled;
    NewTokens s0;  // of sequence `lane`, and its few_tiles
    int first;
    // Tiles of a row tile of c with its filling.
    __device__ __forceinline__ uint32_t span(uint32_t c) const { return filled ? (c + size - 1) / size * size : c; }
};
__device__ __forceinline__ int few_tiles(const PagedParams& p, int n, NewTokens& s) {
    if (n >= p.N) return 0;
    s = new_tokens(p, n);
    if (!of_kind<FEW>(p, s)) return 0;
    const Tiles t = tiles_of<FEW>(p, s, 0);
    return max(1, t.end - t.begin);
}
// Of work-groups with twice the waves half as many run at once.
constexpr uint32_t few_slots(int waves) { return Shape<FEW>::SLOTS * Shape<FEW>::WAVES / waves; }
__device__ __forceinline__ Cut few_cut(const PagedParams& p, bool cut, int waves, int lane) {
    const uint32_t slots = few_slots(waves);
    Cut c;
    uint32_t all = 0, units = 0;
    for (int n0 = 0; n0 < p.N; n0 += 64) {
        NewTokens s = {};
        const int x = few_tiles(p, n0 + lane, s);
        if (n0 == 0) {
            c.first = x;
            c.s0 = s;
        }
        all += (uint32_t)__builtin_amdgcn_readlane(wave_prefix(x), 63);
        units += __popcll(__ballot(x > 0));
    }
    c.tiles = all * p.HKV;
    units *= p.HKV;
    c.filled = !cut || units <= slots / 4;
    const uint32_t pieces = c.filled ? slots - units : slots;
    c.size = cut ? max((uint32_t)Shape<FEW>::LEAST, (c.tiles + pieces - 1) / pieces) : FEW_WHOLE / Shape<FEW>::TK;
    c.size = __builtin_amdgcn_readfirstlane(c.size);
    return c;
}
// Each lane's sequence n0 + lane: the tiles of one of its heads.
struct FewSpans {
    NewTokens s;
    int tiles;
    uint32_t span, upto;  // with its filling; the heads' sum up to its end
};
__device__ __forceinline__ FewSpans few_spans(const PagedParams& p, const Cut& cut, int n0, int lane) {
    FewSpans x;
    x.s = cut.s0;
    x.tiles = cut.first;
    if (n0 > 0) x.tiles = few_tiles(p, n0 + lane, x.s);
    x.span = cut.span(x.tiles);
    x.upto = wave_prefix(x.span * p.HKV);
    return x;
}

// Many rows.  Row tiles are taken whole where they are enough to fill the
// card, else the keys of one with t tiles are cut into t * SLOTS / all parts,
// all being the tiles of all (rounded down: the parts of all then number at
// most SLOTS and run at once), of LEAST tiles at least.
// Sequence by sequence, a sequence's row tiles last first (those of a causal
// chunk see the most keys), then its parts, heads innermost: work-groups go
// round the XCDs, so that with 8 heads each XCD's L2 has the keys of one.
struct ManyWork {
    int mt = 0, tiles = 0;  // row tiles, and tiles of keys that one sees at most
    NewTokens s;
};
__device__ __forceinline__ ManyWork many_work(const PagedParams& p, int n) {
    constexpr int MT = Shape<MANY>::MT, TK = Shape<MANY>::TK;
    ManyWork w = {};
    if (n >= p.N) return w;
    const NewTokens s = new_tokens(p, n);
    if (!of_kind<MANY>(p, s)) return w;
    w.s = s;
    w.mt = (s.count * p.G + MT - 1) / MT;
    w.tiles = (s.len + TK - 1) / TK;
    if (p.window) {
        // the tokens of a row tile and the window before the first
        const int64_t span = (int64_t)min(s.count, MT / p.G + 2) + p.window;
        w.tiles = (int)min((int64_t)w.tiles, (span + 2 * TK - 2) / TK);
    }
    return w;
}
// The lanes' sequences in the order of their tiles, most first, so that the
// longest row tiles do not start last (16 sequences of 512 new tokens after
// 1000 to 23000: 1027 us in their own order, 987 so): the lane's sequence then.
__device__ __forceinline__ int longest_first(const PagedParams& p, ManyWork& w, int lane) {
    int rank = 0;
    for (int j = 0; j < p.N; ++j) {
        const int t = __builtin_amdgcn_readlane(w.tiles, j);
        rank += t > w.tiles || (t == w.tiles && j < lane);
    }
    if (lane >= p.N) rank = lane;
    const int from = __builtin_amdgcn_ds_permute(rank << 2, lane);
    auto take = [&](int x) { return __builtin_amdgcn_ds_bpermute(from << 2, x); };
    w.mt = take(w.mt);
    w.tiles = take(w.tiles);
    w.s = {take(w.s.first), take(w.s.count), take(w.s.len), take(w.s.pos)};
    return from;
}
// Work-group (JOIN: row tile, its parts' first place and number) `id`'s part.
// `sort` (up to 64 sequences): the sequences that see the most keys first.
template <bool JOIN>
__device__ __forceinline__ bool many_unit(const PagedParams& p, int id, bool cut, bool sort, int lane, Unit& u, int& parts) {
    int64_t all = 0;
    if (cut) {
        for (int n0 = 0; n0 < p.N; n0 += 64) {
            const ManyWork w = many_work(p, n0 + lane);
            int64_t x = (int64_t)w.mt * w.tiles;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
            all += x;
        }
        all *= p.HKV;
    }
    int slots = 0;
    for (int n0 = 0; n0 < p.N; n0 += 64) {
        ManyWork w = many_work(p, n0 + lane);
        int seq = n0 + lane;
        if (sort) seq = longest_first(p, w, lane);
        const int np = cut && w.tiles >= 2 * Shape<MANY>::LEAST
                           ? max(1, min(w.tiles / Shape<MANY>::LEAST, (int)((int64_t)w.tiles * Shape<MANY>::SLOTS / all)))
                           : 1;
        const int end = wave_prefix(w.mt * p.HKV * (JOIN ? 1 : np));
        const int slot_end = wave_prefix(np > 1 ? w.mt * p.HKV * np : 0);
        const int total = __builtin_amdgcn_readlane(end, 63);
        if (id < total) {
            const int at = __builtin_ctzll(__ballot(end > id));
            const int before = at > 0 ? __builtin_amdgcn_readlane(end, at - 1) : 0;
            const int slot0 = slots + (at > 0 ? __builtin_amdgcn_readlane(slot_end, at - 1) : 0);
            const int mt = __builtin_amdgcn_readlane(w.mt, at);
            parts = __builtin_amdgcn_readlane(np, at);
            u.n = __builtin_amdgcn_readlane(seq, at);
            int x = id - before;
            u.h = x % p.HKV;
            x /= p.HKV;
            int part = 0;
            if (!JOIN) {
                part = x % parts;
                x /= parts;
            }
            u.m = mt - 1 - x;
            u.slot = parts > 1 ? slot0 + (x * p.HKV + u.h) * parts + part : -1;
            u.s = of_lane(w.s, at);
            const Tiles t = tiles_of<MANY>(p, u.s, u.m);
            const int64_t count = t.end - t.begin;
            u.lo = t.lo;
            u.hi = t.hi;
            u.begin = t.begin + (int)(count * part / parts);
            u.end = t.begin + (int)(count * (part + 1) / parts);
            return true;
        }
        id -= total;
        slots += __builtin_amdgcn_readlane(slot_end, 63);
    }
    return false;
}

// A part's rows in the workspace: m (times c), l, then the row tile's O.
template <int KIND, int D>
struct Partial {
    static constexpr int MT = Shape<KIND>::MT;
    static constexpr int64_t FLOATS = MT * (D + 2);
    static __device__ __forceinline__ float* at(float* ws, int slot) { return ws + slot * FLOATS; }
};
// Floats of the workspace before the parts of kind MANY.
template <int D>
constexpr int64_t few_floats() { return Shape<FEW>::PLACES * Partial<FEW, D>::FLOATS; }

// What a row sees: keys [lo, hi) of its sequence.
struct Row {
    int tok, head, lo, hi;
    bool live;
};
__device__ __forceinline__ Row row_of(const PagedParams& p, const Unit& u, int r) {
    Row x;
    const int rows = u.s.count * p.G;
    x.live = r < rows;
    const int rc = min(r, rows - 1);  // (rows past the last: its values again, unstored)
    x.tok = rc / p.G;
    x.head = u.h * p.G + (rc - x.tok * p.G);
    const int pos = u.s.pos + x.tok;
    x.hi = p.causal ? max(0, min(pos + 1, u.s.len)) : u.s.len;
    x.lo = p.window ? max(0, pos + 1 - p.window) : 0;
    return x;
}

__device__ __forceinline__ int64_t out_row(const PagedParams& p, const Unit& u, const Row& x) {
    return (p.cu_seqlens ? (int64_t)u.s.first + x.tok : (int64_t)u.n * p.T + x.tok) * p.HQ + x.head;
}

template <int D>
__device__ __forceinline__ void load_q(const PagedParams& p, const Unit& u, const Row& x, int half, u32x4 (&q)[D / 16]) {
    const uint16_t* at = p.q + (p.cu_seqlens ? u.s.first * p.q_token : u.n * p.q_row) + x.tok * p.q_token + x.head * p.q_head;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) q[s] = *reinterpret_cast<const u32x4*>(at + 16 * s + 8 * half);
}

// Keys (or values) in memory: the address of the first, and their bytes.
struct Place {
    uint32_t lo, hi, bytes;
};
__device__ __forceinline__ Place of_lane(const Place& x, int at) {
    return {(uint32_t)__builtin_amdgcn_readlane(x.lo, at), (uint32_t)__builtin_amdgcn_readlane(x.hi, at),
            (uint32_t)__builtin_amdgcn_readlane(x.bytes, at)};
}

// What a wave loads of a tile: NROWS keys (or values) of one head, all of one
// page, 1 KiB a load.
template <int D, int NROWS, bool STREAM>
struct Loader {
    static constexpr int PIECES = D / 8, R = 64 / PIECES, LOADS = NROWS / R;
    uint64_t head;            // byte address of the head in page 0
    uint32_t page_bytes, token_bytes;
    int off[LOADS];           // this lane's bytes of each load, within the rows
    // row0: the first row's place in its 16.
    __device__ __forceinline__ Loader(const uint16_t* cache, uint32_t page_stride, int token, int64_t h, int row0, int lane)
        : head(reinterpret_cast<uint64_t>(cache + h)), page_bytes(page_stride * 2), token_bytes(token * 2) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int row = j * R + lane / PIECES;
            off[j] = row * (int)token_bytes + (((lane & (PIECES - 1)) ^ swizzle<D>(row0 + row)) << 4);
        }
    }
    // Keys `key` on, of a page (an entry of the table).  In LDS, keys past the
    // last that the row tile sees become zeros (the descriptor ends with it),
    // and so do all where it sees none of them or there is no page: whatever
    // pages hold beyond a sequence, or had before its window, does not reach
    // the products.
    __device__ __forceinline__ Place place(const PagedParams& p, const Unit& u, int page, int key) const {
        const int n = is_page(p, page) && key + NROWS > u.lo ? min(u.hi - key, NROWS) : 0;
        const int in = key & ((1 << p.page_shift) - 1);
        const uint64_t at = head + (uint64_t)(n > 0 ? (uint32_t)page : 0u) * page_bytes + (uint32_t)in * token_bytes;
        return {(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, n > 0 ? (n - 1) * token_bytes + D * 2 : 0u};
    }
    // (the place the same in all lanes)
    __device__ __forceinline__ void load(const Place& x, uint32_t lds) const {
        const u32x4 rsrc = {x.lo, x.hi, x.bytes, BUF_RAW};
#pragma unroll
        for (int j = 0; j < LOADS; ++j) load_lds<STREAM>(rsrc, off[j], lds + j * 1024);
    }
    template <int AT>
    __device__ __forceinline__ void load_at(const Place& x, uint32_t lds) const {
        load_lds_at<AT, LOADS>(u32x4{x.lo, x.hi, x.bytes, BUF_RAW}, off, lds);
    }
};

// This wave's LDS reads have returned: what they read may be loaded over.
__device__ __forceinline__ void reads_done() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt 0
    __builtin_amdgcn_sched_barrier(0);
}

// Output or partial of one row's four elements from d on.
template <class E, int D>
__device__ __forceinline__ void store_o(const PagedParams& p, int64_t out, int d, float a, float b, float c, float e) {
    *reinterpret_cast<u32x2*>(p.o + out * D + d) = u32x2{E::pack(a, b), E::pack(c, e)};
}
// (l is 0 only where no key is seen; NaN, of scores that are not finite, stays)
__device__ __forceinline__ float log_sum(float mc, float l) {
    return l == 0.f ? -INFINITY : (mc + __builtin_amdgcn_logf(l)) * LN2;
}

// ---- few rows ----

// Each wave goes over every WAVES-th tile of 32 keys, through LDS of its own:
// while it multiplies keys the values arrive, and the other way round.  The
// waves' sums are joined at the end, in the same LDS (2 * TILE bytes a
// wave: a tile of keys, one of values; 32 rows of D floats).  Where there is
// much to read HBM bounds it (64 sequences of 100 to 16000 tokens, 32 / 8 heads,
// 765 MB in 130 us, 5.9 TB/s; a large read reaches 6.3), with little the chain
// of lengths, table entry, keys, values: 6 us, and 1.8 more for each further
// tile of a wave.
template <class E, int D, int WAVES>
__device__ __forceinline__ void few_loop(const PagedParams& p, const Unit& u, uint8_t* lds, int wave, Running& run,
                                         f32x16 (&acc)[D / 32]) {
    constexpr int STEPS = D / 16, DB = D / 32, TK = Shape<FEW>::TK;
    constexpr int TILE = TK * D * 2, LOADS = TILE / 1024;  // loads of a tile of keys, or of values
    const int lane = (int)hide(threadIdx.x & 63), half = lane >> 5;
    const Row x = row_of(p, u, u.m * ROWS + (lane & 31));
    // the keys that every row sees
    const int all_lo = __builtin_amdgcn_readlane(x.lo, 31), all_hi = __builtin_amdgcn_readlane(x.hi, 0);
    const float c = p.scale * LOG2E;
    u32x4 q[STEPS];
    load_q<D>(p, u, x, half, q);

    // The wave's tiles are first, first + WAVES and so on, `count` of them.  Where
    // 32 of them lie, 16 keys a lane: a tile's loads then need no more than lane
    // reads (found tile by tile with scalar operations, one sequence of 700 keys
    // took 10.4 us instead of 9.8, 64 sequences 132 instead of 130).
    const int first = u.begin + wave, count = (u.end - first + WAVES - 1) / WAVES;
    if (count <= 0) return;
    const Loader<D, 16, true> k0(p.k, p.k_page, p.k_token, u.h * p.k_head, 0, lane);
    const Loader<D, 16, true> v0(p.v, p.v_page, p.v_token, u.h * p.v_head, 0, lane);
    Place k_of, v_of;
    auto places = [&](int j) {
        const int mine = j + (lane >> 1);
        const int key = (first + min(mine, count - 1) * WAVES) * TK + 16 * (lane & 1);
        const int at = min(key >> p.page_shift, p.M - 1);
        const int page = mine < count ? p.page_table[u.n * p.table_stride + at] : -1;
        k_of = k0.place(p, u, page, key);
        v_of = v0.place(p, u, page, key);
    };
    auto load = [&](const Loader<D, 16, true>& from, const Place& at, int j, uint8_t* to) {
#pragma unroll
        for (int g = 0; g < 2; ++g) from.load(of_lane(at, 2 * (j & 31) + g), lds_address(to) + g * (TILE / 2));
    };
    uint32_t k_at[STEPS], v_at[DB][2];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) k_at[s] = lds_address(k_place<D>(lds, lane & 31, 2 * s + half));
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 2; ++i) v_at[d][i] = lds_address(v_place<D>(lds + TILE, 8 * i + 4 * half, d, lane));
    places(0);
    load(k0, k_of, 0, lds);
    load(v0, v_of, 0, lds + TILE);
    for (int j = 0; j < count; ++j) {
        const bool more = j + 1 < count;
        if (((j + 1) & 31) == 0) places(j + 1);
        // All operands of a product are read before it, so that its place is
        // loaded again while it runs.
        wait_loads<LOADS>();  // but for the values'
        u32x4 ka[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) ka[s] = load_operand(k_at[s]);
        reads_done();
        if (more) load(k0, k_of, j + 1, lds);
        f32x16 st[1] = {f32x16{}};
#pragma unroll
        for (int s = 0; s < STEPS; ++s) st[0] = E::mfma(ka[s], q[s], st[0]);
        if (more) wait_loads<LOADS>();  // but for the next keys'
        else wait_loads<0>();
        u32x4 va[2][DB];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const u32x2 a = load_transposed(v_at[d][0] + 16 * k * D * 2);
                const u32x2 b = load_transposed(v_at[d][1] + 16 * k * D * 2);
                va[k][d] = u32x4{a.x, a.y, b.x, b.y};
            }
        reads_done();
        if (more) load(v0, v_of, j + 1, lds + TILE);
        u32x4 pt[2];
        float alpha;
        const int key = (first + j * WAVES) * TK;
        if (softmax_tile<E, 1>(st, key + 4 * half, x.lo, x.hi, key < all_lo || key + TK > all_hi, c, run, pt, alpha)) {
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[d] *= alpha;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[d] = E::mfma(va[k][d], pt[k], acc[d]);
    }
    run.l = sum_halves(run.l);
}

// A wave's place in LDS: of four waves in one array; of eight, three in each of
// two and two in a third (the many rows' kernel: its rings, and an array more).
template <int D, int WAVES>
struct FewLds {
    static constexpr int EACH = 2 * Shape<FEW>::TK * D * 2;
    uint8_t *a, *b, *c;
    __device__ __forceinline__ uint8_t* of(int wave) const {
        if (WAVES == 4 || wave < 3) return a + wave * EACH;
        return wave < 6 ? b + (wave - 3) * EACH : c + (wave - 6) * EACH;
    }
};

template <class E, int D, int WAVES>
__device__ __forceinline__ void few_rows(const PagedParams& p, const Unit& u, const FewLds<D, WAVES>& lds, float* joint) {
    constexpr int DB = D / 32;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Running run;
    f32x16 acc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) acc[i] = f32x16{};
    uint8_t* mine = lds.of(wave);
    few_loop<E, D, WAVES>(p, u, mine, wave, run, acc);

    // Join: every wave's m and l, then its O over the tiles' LDS, row by row
    // in pieces of four (the rows' pieces turned by the row, so that the lanes
    // of a half, one row each, write different banks).
    const int row = lane & 31;
    if (half == 0) {
        joint[wave * 2 * ROWS + row] = run.log2_max();
        joint[wave * 2 * ROWS + ROWS + row] = run.l;
    }
    __syncthreads();
    float* own = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int piece = (32 * d + 2 * i + 4 * half) / 4;
            *reinterpret_cast<f32x4*>(own + row * D + ((piece + row) & (D / 4 - 1)) * 4) =
                f32x4{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
        }
    __syncthreads();
    float* part = u.slot >= 0 ? Partial<FEW, D>::at(p.ws, u.slot) : nullptr;
    for (int e = threadIdx.x; e < ROWS * (D / 4); e += WAVES * 64) {
        const int r = e / (D / 4), piece = e % (D / 4);
        const Row y = row_of(p, u, u.m * ROWS + r);
        if (!y.live) break;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mx = fmaxf(mx, joint[w * 2 * ROWS + r]);
        const float sub = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = fast_exp2(joint[w * 2 * ROWS + r] - sub);
            sum = fmaf(f, joint[w * 2 * ROWS + ROWS + r], sum);
            const float* src = reinterpret_cast<const float*>(lds.of(w));
            const f32x4 v = *reinterpret_cast<const f32x4*>(src + r * D + ((piece + r) & (D / 4 - 1)) * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = fmaf(f, v[i], o[i]);
        }
        if (part) {
            *reinterpret_cast<f32x4*>(part + 2 * ROWS + r * D + piece * 4) = o;
            if (piece == 0) {
                part[r] = mx;
                part[ROWS + r] = sum;
            }
        } else {
            const float inv = sum > 0.f ? 1.f / sum : 0.f;
            const int64_t out = out_row(p, u, y);
            store_o<E, D>(p, out, piece * 4, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            if (p.lse && piece == 0) p.lse[out] = log_sum(mx, sum);
        }
    }
}

// Work-group b's piece of the cut, row tile by row tile.
template <class E, int D, int WAVES>
__device__ __forceinline__ void few_piece(const PagedParams& p, int b, bool may_cut, const FewLds<D, WAVES>& lds,
                                          float* joint) {
    const int lane = threadIdx.x & 63;
    const Cut cut = few_cut(p, may_cut, WAVES, lane);
    const uint32_t first = b * cut.size, end = first + cut.size;
    uint32_t cur = first, base = 0;
    for (int n0 = 0; n0 < p.N && cur < end; n0 += 64) {
        const FewSpans x = few_spans(p, cut, n0, lane);
        const uint32_t total = __builtin_amdgcn_readlane(x.upto, 63);
        while (cur < end && cur < base + total) {
            const int at = __builtin_ctzll(__ballot(x.upto > cur - base));
            const uint32_t c = __builtin_amdgcn_readlane(x.tiles, at), span = __builtin_amdgcn_readlane(x.span, at);
            const uint32_t in = cur - base - (__builtin_amdgcn_readlane(x.upto, at) - span * p.HKV);
            Unit u;
            u.n = __builtin_amdgcn_readfirstlane(n0 + at);
            u.h = in / span;
            u.m = 0;
            u.s = of_lane(x.s, at);
            const uint32_t t = in - u.h * span, stop = min(span, t + (end - cur));
            const Tiles all = tiles_of<FEW>(p, u.s, 0);
            u.lo = all.lo;
            u.hi = all.hi;
            u.begin = all.begin + t;
            u.end = all.begin + min(c, stop);
            u.slot = t == 0 && stop >= c ? -1 : 2 * b + (cur == first ? 0 : 1);
            if (cur != first) __syncthreads();  // the last row tile's join is over
            few_rows<E, D, WAVES>(p, u, lds, joint);
            cur += stop - t;
        }
        base += total;
    }
}

// ---- many rows ----

// The work-group meets; the wave's LDS reads have returned.  The clobber keeps
// LDS accesses on their side.
__device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // (known to be zero: no waits for reads before)
}

// Eight waves, two on each SIMD, in two groups: while one group's waves form
// products (phase M: O += V^T P^T of the last tile, S of this one) the other
// group's do the softmax of theirs (phase S), and they meet after each phase.
// Left to themselves (two work-groups of four waves a CU) the two waves of a
// SIMD fell into step: a prompt of 8192 tokens, 32 / 8 heads, 558 us, so 521.
// S was then the longer phase (a lone wave issues a vector operation every 2.5 ns
// and an exponential every 6.8, and the loads' addresses took 80 scalar ones);
// with the places of 64 tiles found at once the prompt takes 970 kilocycles
// instead of 1137 and 489 to 516 us (1.1 PFLOP/s; a bf16 product of 8192^3
// reaches 1.15 to 1.2 on the same card), the matrix unit 54% busy.  15% fewer
// cycles were 6% less time: the clock (cycles over time) went from 2.08 to 1.90
// GHz, which looks like the card's power; no reading of it was taken.
// No gain from: two or three groups of operands ahead instead of one, both
// products in one straight block (540), the loads begun between matrix ops (540
// to 553), other orders of the softmax's operations.
//   slot     2t             2t + 1         2t + 2
//   group 0  M(t)           S(t)           M(t + 1)
//   group 1  S(t - 1)       M(t)           S(t)
// Keys and values go through three tiles of LDS each.  The softmax of tile t
// begins with this wave's loads (8 keys) of K(t + 2) and V(t + 1), over tiles
// last read in slot 2t - 1; slot 2t + 2 is the first to read K(t + 1) and V(t),
// which every wave has waited for by its end of slot 2t + 1.
template <class E, int D>
__device__ __forceinline__ void many_rows(const PagedParams& p, const Unit& u, uint8_t* kt, uint8_t* vt) {
    constexpr int STEPS = D / 16, DB = D / 32, TK = Shape<MANY>::TK, MT = Shape<MANY>::MT;
    constexpr int TILE = TK * D * 2;
    constexpr int SHARE = TK / Shape<MANY>::WAVES, LOADS = SHARE * D * 2 / 1024;  // keys and loads a wave and tile
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool second = wave >= 4;
    const int row = wave * ROWS + (lane & 31);
    const Row x = row_of(p, u, u.m * MT + row);
    const int count = u.end - u.begin;
    // the keys that every row of this wave sees, and those that any does; the
    // tiles of u.begin on that are among the first, and that have some of the others
    const int all_lo = __builtin_amdgcn_readlane(x.lo, 31), all_hi = __builtin_amdgcn_readlane(x.hi, 0);
    const int any_lo = __builtin_amdgcn_readlane(x.lo, 0);
    const int any_hi = u.m * MT + wave * ROWS < u.s.count * p.G ? __builtin_amdgcn_readlane(x.hi, 31) : 0;
    const int all0 = (int)(((unsigned)all_lo + TK - 1) / TK) - u.begin, any0 = max(any_lo / TK - u.begin, 0);
    const unsigned all_tiles = max(all_hi / TK - u.begin - all0, 0);
    const unsigned any_tiles = max((int)(((unsigned)any_hi + TK - 1) / TK) - u.begin - any0, 0);
    const float c = p.scale * LOG2E;
    Running run;
    f32x16 acc[DB], st[2];
    u32x4 pt[4];
#pragma unroll
    for (int i = 0; i < DB; ++i) acc[i] = f32x16{};

    const Loader<D, SHARE, false> k0(p.k, p.k_page, p.k_token, u.h * p.k_head, SHARE * wave & 15, lane);
    const Loader<D, SHARE, false> v0(p.v, p.v_page, p.v_token, u.h * p.v_head, SHARE * wave & 15, lane);
    const uint32_t k_lds = lds_address(kt) + wave * (SHARE * D * 2), v_lds = lds_address(vt) + wave * (SHARE * D * 2);
    // Where this wave's keys of 64 tiles lie, a tile a lane: a tile's loads then
    // need no more than lane reads (a table entry and an address for each, by
    // scalar operations, took a fifth of a slot).  Past the last tile: nothing,
    // zeros.
    auto places = [&](const Loader<D, SHARE, false>& of, int t) {
        const int key = (u.begin + max(min(t + lane, count - 1), 0)) * TK + SHARE * wave;
        const int at = min(key >> p.page_shift, p.M - 1);
        return of.place(p, u, t + lane < count ? p.page_table[u.n * p.table_stride + at] : -1, key);
    };
    Place k_of = places(k0, 0), v_of = places(v0, 0);
    k0.load(of_lane(k_of, 0), k_lds);
    k0.load(of_lane(k_of, 1), k_lds + TILE);
    v0.load(of_lane(v_of, 0), v_lds);
    u32x4 q[STEPS];
    load_q<D>(p, u, x, half, q);

    auto sees = [&](int t) { return (unsigned)(t - any0) < any_tiles; };
    auto begin_loads = [&](int t, auto I) {
        if (((t + 2) & 63) == 0) k_of = places(k0, t + 2);
        if (((t + 1) & 63) == 0) v_of = places(v0, t + 1);
        k0.template load_at<(I + 2) % 3 * TILE>(of_lane(k_of, (t + 2) & 63), k_lds);
        v0.template load_at<(I + 1) % 3 * TILE>(of_lane(v_of, (t + 1) & 63), v_lds);
    };
    // The products' operands are read one group of matrix ops ahead of their
    // use, a read between two matrix ops: an LDS read takes several of them.
    auto scores = [&](const uint8_t* ks) {
        u32x4 a[2][4];
        auto read = [&](int g, int i) {
            return read_k<D>(ks, 32 * (i & 1) + (lane & 31), 2 * (2 * g + (i >> 1)) + half);
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) a[0][i] = read(0, i);
        st[0] = st[1] = f32x16{};
#pragma unroll
        for (int g = 0; g < STEPS / 2; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (g + 1 < STEPS / 2) a[(g + 1) & 1][i] = read(g + 1, i);
                st[i & 1] = E::mfma(a[g & 1][i], q[2 * g + (i >> 1)], st[i & 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    auto outputs = [&](const uint8_t* vs) {
        u32x4 a[2][DB];
        auto read = [&](int k, int d) {
            const u32x2 v0 = read_v<D>(vs, 16 * k + 4 * half, d, lane);
            const u32x2 v1 = read_v<D>(vs, 16 * k + 8 + 4 * half, d, lane);
            return u32x4{v0.x, v0.y, v1.x, v1.y};
        };
#pragma unroll
        for (int d = 0; d < DB; ++d) a[0][d] = read(0, d);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                if (k + 1 < 4) a[(k + 1) & 1][d] = read(k + 1, d);
                acc[d] = E::mfma(a[k & 1][d], pt[k], acc[d]);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    auto products = [&](int t, const uint8_t* ks, const uint8_t* vs) {
        __builtin_amdgcn_s_setprio(1);
        if (sees(t - 1)) outputs(vs);
        if (sees(t)) scores(ks);
        __builtin_amdgcn_s_setprio(0);
    };
    auto softmax = [&](int t) {
        if (!sees(t)) return;
        float alpha;
        if (softmax_tile<E, 2>(st, (u.begin + t) * TK + 4 * half, x.lo, x.hi, (unsigned)(t - all0) >= all_tiles, c, run, pt,
                               alpha)) {
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[d] *= alpha;
        }
    };
    // Tile t, in place I = t % 3 of the rings.
    auto step = [&](int t, auto I) {
        products(t, kt + I * TILE, vt + (I + 2) % 3 * TILE);
        if (second) wait_loads<0>();
        meet();
        begin_loads(t, I);
        softmax(t);
        if (!second) wait_loads<2 * LOADS>();  // but for what was begun just now: K(t + 1) and V(t) have arrived
        meet();
    };
    if (count > 0) {
        // (where the compiler sees it: else it waits for q in every turn)
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt 0
        meet();
        if (second) meet();
        for (int t = 0; t < count; t += 3) {
            step(t, std::integral_constant<int, 0>{});
            if (t + 1 < count) step(t + 1, std::integral_constant<int, 1>{});
            if (t + 2 < count) step(t + 2, std::integral_constant<int, 2>{});
        }
        if (sees(count - 1)) outputs(vt + (count - 1) % 3 * TILE);
        if (!second) meet();
    }
    wait_loads<0>();  // (past the last tile)

    const float l = sum_halves(run.l);
    if (!x.live) return;
    if (u.slot >= 0) {
        float* part = Partial<MANY, D>::at(p.ws + few_floats<D>(), u.slot);
        if (half == 0) {
            part[row] = run.log2_max();
            part[MT + row] = l;
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4*>(part + 2 * MT + row * D + 32 * d + 2 * i + 4 * half) =
                    f32x4{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
        return;
    }
    const int64_t out = out_row(p, u, x);
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            store_o<E, D>(p, out, 32 * d + 2 * i + 4 * half, acc[d][i] * inv, acc[d][i + 1] * inv, acc[d][i + 2] * inv,
                          acc[d][i + 3] * inv);
    if (p.lse && half == 0) p.lse[out] = log_sum(run.mc, l);
}

// ---- kernels ----

template <class E, int D, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void paged_few_kernel(PagedParams p, bool cut) {
    typedef FewLds<D, WAVES> Lds;
    __shared__ alignas(1024) uint8_t lds[WAVES * Lds::EACH];
    __shared__ float joint[WAVES * 2 * ROWS];
    few_piece<E, D>(p, blockIdx.x, cut, Lds{lds, lds + 3 * Lds::EACH, lds + 6 * Lds::EACH}, joint);
}

// MIXED: the work-groups from `few_from` on take the sequences of few rows, with
// as many waves: packed batches of chunks and single tokens in one launch, the
// few rows on the CUs that the chunks' last row tiles leave (32 / 8 heads, 63
// sequences of a new token and 256 to 16384 keys and one of 512 after 5488: 316
// us in two launches, 240 to 247 so; 8 sequences of 1 to 1024 new tokens, a
// window of 4096: 144 and 140).
template <class E, int D, bool MIXED_KINDS>
__global__ __launch_bounds__(512, 2) void paged_many_kernel(PagedParams p, bool cut, bool sort, unsigned few_from, bool few_may_cut) {
    constexpr int WAVES = Shape<MANY>::WAVES, RING = 3 * Shape<MANY>::TK * D * 2;
    __shared__ alignas(1024) uint8_t kt[RING];
    __shared__ alignas(1024) uint8_t vt[RING];
    __shared__ alignas(1024) uint8_t more[MIXED_KINDS ? 2 * 2 * Shape<FEW>::TK * D * 2 : 16];
    __shared__ float joint[MIXED_KINDS ? WAVES * 2 * ROWS : 1];
    if (MIXED_KINDS && blockIdx.x >= few_from) {
        few_piece<E, D>(p, blockIdx.x - few_from, few_may_cut, FewLds<D, WAVES>{kt, vt, more}, joint);
        return;
    }
    Unit u;
    int parts;
    if (many_unit<false>(p, blockIdx.x, cut, sort, threadIdx.x & 63, u, parts)) many_rows<E, D>(p, u, kt, vt);
}

// Joins the partial results of one row tile: four elements of a row a thread,
// SLICES threads' parts in turn.  place(j): the j-th part's rows.
constexpr int SLICES = 4;  // few rows: the waves
template <class E, int D, int KIND, class Place>
__device__ __forceinline__ void join(const PagedParams& p, const Unit& u, int group, int parts, Place place, float* lds) {
    constexpr int MT = Shape<KIND>::MT, NS = KIND == FEW ? SLICES : 1;
    const int slice = KIND == FEW ? threadIdx.x >> 6 : 0;
    const int e = group * (256 / NS) + threadIdx.x % (256 / NS);
    const int r = e / (D / 4), piece = e % (D / 4);
    const Row y = row_of(p, u, u.m * MT + r);
    float mx = -INFINITY, sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (y.live) {
        // one pass, so that no load waits for another
#pragma unroll 4
        for (int j = slice; j < parts; j += NS) {
            const float* part = place(j);
            const float mj = part[r], lj = part[MT + r];
            const f32x4 v = *reinterpret_cast<const f32x4*>(part + 2 * MT + r * D + piece * 4);
            const float top = fmaxf(mx, mj), sub = top == -INFINITY ? 0.f : top;
            const float f0 = fast_exp2(mx - sub), f = fast_exp2(mj - sub);
            mx = top;
            sum = fmaf(f, lj, sum * f0);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = fmaf(f, v[i], o[i] * f0);
        }
    }
    if constexpr (NS > 1) {
        // the slices' sums, six numbers a thread
        const int t = threadIdx.x;
        lds[t] = mx;
        lds[256 + t] = sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) lds[(2 + i) * 256 + t] = o[i];
        __syncthreads();
        if (slice != 0) return;  // (no barrier follows in here)
        float top = mx;
#pragma unroll
        for (int w = 1; w < NS; ++w) top = fmaxf(top, lds[w * 64 + t]);
        const float sub = top == -INFINITY ? 0.f : top;
        float f = fast_exp2(mx - sub);
        sum *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= f;
#pragma unroll
        for (int w = 1; w < NS; ++w) {
            f = fast_exp2(lds[w * 64 + t] - sub);
            sum = fmaf(f, lds[256 + w * 64 + t], sum);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = fmaf(f, lds[(2 + i) * 256 + w * 64 + t], o[i]);
        }
        mx = top;
    }
    if (!y.live) return;
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    const int64_t out = out_row(p, u, y);
    store_o<E, D>(p, out, piece * 4, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    if (p.lse && piece == 0) p.lse[out] = log_sum(mx, sum);
}

// `few_groups` or `many_groups` work-groups a row tile.  Bound by the chain of
// lengths, cut and partial results: 5 us whatever there is to join.
template <class E, int D, int KIND>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p, int few, int few_groups, int many_groups, bool cut_many) {
    __shared__ float lds[KIND == MANY ? 1 : 6 * 256];
    const int lane = threadIdx.x & 63;
    Unit u;
    if (KIND == FEW || (KIND == MIXED && (int)blockIdx.x < few)) {
        const int id = blockIdx.x / few_groups;
        const Cut cut = few_cut(p, true, Shape<KIND == MIXED ? MANY : FEW>::WAVES, lane);
        u.n = id / p.HKV;
        u.h = id - u.n * p.HKV;
        u.m = 0;
        uint32_t first = 0, c = 0;  // its tiles [first, first + c) of all
        for (int n0 = 0; n0 <= u.n; n0 += 64) {
            const FewSpans x = few_spans(p, cut, n0, lane);
            if (u.n < n0 + 64) {
                c = __builtin_amdgcn_readlane(x.tiles, u.n - n0);
                u.s = of_lane(x.s, u.n - n0);
                const uint32_t span = __builtin_amdgcn_readlane(x.span, u.n - n0);
                first += __builtin_amdgcn_readlane(x.upto, u.n - n0) - (p.HKV - u.h) * span;
            } else {
                first += __builtin_amdgcn_readlane(x.upto, 63);
            }
        }
        if (c == 0) return;
        const uint32_t b0 = first / cut.size, b1 = (first + c - 1) / cut.size;
        if (b0 == b1) return;
        const int items = u.s.count * p.G * (D / 4);
        for (int group = blockIdx.x % few_groups; group * 64 < items; group += few_groups) {
            join<E, D, FEW>(p, u, group, b1 - b0 + 1, [&](int j) {
                const uint32_t b = b0 + j;
                return Partial<FEW, D>::at(p.ws, 2 * b + (b * cut.size >= first ? 0 : 1));
            }, lds);
            __syncthreads();
        }
    } else {
        int parts;
        const int x = (int)blockIdx.x - few;
        if (!many_unit<true>(p, x / many_groups, cut_many, false, lane, u, parts) || parts == 1) return;
        const int items = min(Shape<MANY>::MT, u.s.count * p.G - u.m * Shape<MANY>::MT) * (D / 4);
        for (int group = x % many_groups; group * 256 < items; group += many_groups)
            join<E, D, MANY>(p, u, group, parts, [&](int j) {
                return Partial<MANY, D>::at(p.ws + few_floats<D>(), u.slot + j);
            }, lds);
    }
}

// ---- launches ----

// What a call's kinds are from what the host knows: packed sequences may be of
// both, unless their tokens cannot be of many rows.
int kind_of(const PagedParams& p) {
    if ((int64_t)p.T * p.G <= ROWS) return FEW;
    return p.cu_seqlens ? MIXED : MANY;
}

// Row tiles of many rows at most (packed sequences each leave one unfilled).
int64_t many_units(const PagedParams& p) {
    constexpr int MT = Shape<MANY>::MT;
    const int64_t rows = (int64_t)p.T * p.G;
    return (p.cu_seqlens ? rows / MT + p.N : p.N * ((rows + MT - 1) / MT)) * p.HKV;
}

// Whether a row tile's keys may go to several work-groups.  Few rows: not where
// the table's rows hold so few keys that the join, a launch more, costs more:
// one sequence of 704 keys 9.5 us whole and 9.2 cut, but the host's part 10.1
// against 14.1; 64 of 700 keys 32.8 whole and 35.4 cut.  Many rows: row tiles
// that fill half of SLOTS are taken whole.
bool may_cut(const PagedParams& p, int kind) {
    const int64_t keys = (int64_t)p.M << p.page_shift;
    if (kind == FEW) return keys > FEW_WHOLE;
    return keys >= 2 * Shape<MANY>::LEAST * Shape<MANY>::TK && many_units(p) <= Shape<MANY>::SLOTS / 2;
}
// The waves of a work-group of few rows, in a call of their kind alone: twice as
// many where the row tiles are taken whole and all run at once so, and may be of
// more than two tiles a wave (one sequence of 700 keys, 8 heads, on the GPU
// 11.7 -> 10.5 us, 16 drafts of 5 over 700 10.3 -> 9.1; of up to 128 keys the
// join of more waves costs 0.4 to 0.7).
int few_waves(const PagedParams& p) {
    constexpr int ONCE = Shape<FEW>::WAVES;
    const int64_t keys = (int64_t)p.M << p.page_shift;
    const bool more = !may_cut(p, FEW) && keys > 2 * ONCE * Shape<FEW>::TK && (int64_t)p.N * p.HKV <= few_slots(2 * ONCE);
    return more ? 2 * ONCE : ONCE;
}

template <class E, int D, int KIND>
hipError_t launch(const PagedParams& p, hipStream_t stream) {
    const bool fc = KIND != MANY && may_cut(p, FEW), mc = KIND != FEW && may_cut(p, MANY);
    const int64_t units = KIND == FEW ? 0 : many_units(p);
    // (uncut: one piece a row tile)
    const int64_t whole = (int64_t)p.N * p.HKV;
    if constexpr (KIND == FEW) {
        constexpr int ONCE = Shape<FEW>::WAVES, TWICE = 2 * ONCE;
        if (few_waves(p) == TWICE)
            paged_few_kernel<E, D, TWICE><<<dim3((unsigned)whole), TWICE * 64, 0, stream>>>(p, false);
        else
            paged_few_kernel<E, D, ONCE><<<dim3((unsigned)(fc ? Shape<FEW>::SLOTS : whole)), ONCE * 64, 0, stream>>>(p, fc);
    } else {
        const int64_t many = units + (mc ? Shape<MANY>::SLOTS : 0);
        const int64_t few = KIND == MANY ? 0 : (fc ? Shape<MANY>::SLOTS : whole);
        const bool sort = p.N > 1 && p.N <= 64 && units > Shape<MANY>::SLOTS;
        paged_many_kernel<E, D, KIND == MIXED><<<dim3((unsigned)(many + few)), 512, 0, stream>>>(p, mc, sort, (unsigned)many, fc);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !(fc || mc)) return e;
    // work-groups a row tile: one for every 64 fours of what rows there can be, up to 4
    const int64_t rows = p.cu_seqlens || (int64_t)p.T * p.G > ROWS ? ROWS : p.T * p.G;
    const int groups = (int)std::min((rows * (D / 4) + 63) / 64, (int64_t)4);
    const int64_t few_joins = fc ? (int64_t)p.N * p.HKV * groups : 0;
    const int many_groups = (int)std::min(std::max((int64_t)1024 / std::max(units, (int64_t)1), (int64_t)1), (int64_t)Shape<MANY>::MT * (D / 4) / 256);
    const int64_t many_joins = mc ? units * many_groups : 0;
    paged_join_kernel<E, D, KIND><<<dim3((unsigned)(few_joins + many_joins)), 256, 0, stream>>>(p, (int)few_joins, groups, many_groups, mc);
    return hipGetLastError();
}

template <class E, int D>
hipError_t launch_kind(const PagedParams& p, hipStream_t stream) {
    switch (kind_of(p)) {
        case FEW: return launch<E, D, FEW>(p, stream);
        case MANY: return launch<E, D, MANY>(p, stream);
        default: return launch<E, D, MIXED>(p, stream);
    }
}

}  // namespace

size_t paged_attn_workspace(const PagedParams& p, int D) {
    const int kind = kind_of(p);
    const bool fc = kind != MANY && may_cut(p, FEW), mc = kind != FEW && may_cut(p, MANY);
    if (!fc && !mc) return 0;
    const int64_t few = (int64_t)Shape<FEW>::PLACES * Shape<FEW>::MT * (D + 2);
    const int64_t many = (int64_t)Shape<MANY>::PLACES * Shape<MANY>::MT * (D + 2);
    return (size_t)(few + (mc ? many : 0)) * 4;
}

hipError_t launch_paged_attn(const PagedParams& p, int D, hipStream_t stream) {
    if (D == 128) return p.fp16 ? launch_kind<FP16, 128>(p, stream) : launch_kind<BF16, 128>(p, stream);
    return p.fp16 ? launch_kind<FP16, 64>(p, stream) : launch_kind<BF16, 64>(p, stream);
}

}  // namespace kda
