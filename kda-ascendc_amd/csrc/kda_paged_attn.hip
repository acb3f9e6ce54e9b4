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

constexpr int WAVES = 4;
constexpr int ROWS = 32;            // rows a wave
constexpr int MT = WAVES * ROWS;    // rows a work-group
constexpr int TK = 64;              // keys a tile

// A tile of keys (or values) in LDS: rows of D elements, in each the 16-byte
// piece c at place c ^ swizzle(row).  The swizzle keeps two reads free of bank
// conflicts: 16 rows at one piece (the first product's operand), and the
// transposing read's 4 rows at 4 consecutive pieces.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
    if constexpr (D == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// 16 rows of a page into LDS (`rows` of them exist, the others become zeros:
// the descriptor ends with the last one).  Each load takes 1 KiB, lane l's 16
// bytes going to byte 16 * l of it.
template <int D>
__device__ __forceinline__ void load_rows(const uint16_t* head, int64_t token, int rows, int lane, uint8_t* lds) {
    constexpr int PIECES = D / 8, R = 64 / PIECES;
    const int bytes = rows > 0 ? (int)((rows - 1) * token + D) * 2 : 0;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)head, 0, bytes, BUF_RAW);
#pragma unroll
    for (int j = 0; j < 16 / R; ++j) {
        const int row = j * R + lane / PIECES;
        const int off = (int)(row * token) * 2 + (((lane & (PIECES - 1)) ^ swizzle<D>(row)) << 4);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_u8*)(lds + j * 1024), 16, off, 0, 0, 0);
    }
}

// Operand of the first product: rows lane & 31, elements 16 * s + 8 * (lane >> 5) .. +7.
template <int D>
__device__ __forceinline__ u32x4 read_k(const uint8_t* lds, int row, int piece) {
    return *reinterpret_cast<const u32x4*>(lds + row * (D * 2) + ((piece ^ swizzle<D>(row)) << 4));
}

// Half an operand of the second product: lane's column d = 32 * db + (lane & 31)
// of rows key .. key + 3.  In each group of 16 lanes, lane n receives as item i
// element n % 4 of the 8 bytes that lane 4 * i + n / 4 points at.
template <int D>
__device__ __forceinline__ u32x2 read_v(const uint8_t* lds, int key, int db, int lane) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const int row = key + ((lane & 15) >> 2);
    const int d = 32 * db + (lane & 16) + 4 * (lane & 3);
    const uint8_t* at = lds + row * (D * 2) + (((d >> 3) ^ swizzle<D>(row)) << 4) + (d & 4) * 2;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at));
}

__device__ __forceinline__ float other_half(float x) { return shfl(x, (threadIdx.x & 63) ^ 32); }

// Work-group -> (sequence, kv head, row tile): sequence by sequence, its row
// tiles last first (those of a causal chunk see the most keys), heads
// innermost.  Every lane counts one sequence's work-groups.
struct Unit {
    int n, h, m;
    NewTokens s;
};
__device__ __forceinline__ bool find_unit(const PagedParams& p, int id, int lane, Unit& u) {
    for (int n0 = 0; n0 < p.N; n0 += 64) {
        int tiles = 0;
        if (n0 + lane < p.N) {
            const NewTokens s = new_tokens(p, n0 + lane);
            tiles = (s.count * p.G + MT - 1) / MT;
        }
        int end = tiles * p.HKV;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(end, d);
            if (lane >= d) end += x;
        }
        const int total = __builtin_amdgcn_readlane(end, 63);
        if (id < total) {
            const int at = __builtin_ctzll(__ballot(end > id));
            const int before = at > 0 ? __builtin_amdgcn_readlane(end, at - 1) : 0;
            const int mt = __builtin_amdgcn_readlane(tiles, at);
            u.n = __builtin_amdgcn_readfirstlane(n0 + at);
            const int x = id - before;
            u.h = x % p.HKV;
            u.m = mt - 1 - x / p.HKV;
            u.s = new_tokens(p, u.n);
            return true;
        }
        id -= total;
    }
    return false;
}

template <class E, int D>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedParams p) {
    constexpr int STEPS = D / 16, DB = D / 32;
    __shared__ alignas(1024) uint8_t kt[TK * D * 2];
    __shared__ alignas(1024) uint8_t vt[TK * D * 2];
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Unit u;
    if (!find_unit(p, blockIdx.x, lane, u)) return;

    // This lane's query; rows past the last compute its values again, unstored.
    const int rows = u.s.count * p.G;
    const int r = u.m * MT + wave * ROWS + (lane & 31);
    const bool live = r < rows;
    const int rc = min(r, rows - 1);
    const int tok = rc / p.G, head = u.h * p.G + (rc - tok * p.G);
    const int64_t row0 = p.cu_seqlens ? u.s.first : 0;
    u32x4 q[STEPS];
    {
        const uint16_t* qp = p.q + (p.cu_seqlens ? 0 : u.n * p.q_row) + (row0 + tok) * p.q_token + head * p.q_head;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) q[s] = *reinterpret_cast<const u32x4*>(qp + 16 * s + 8 * half);
    }
    // The keys it sees, [lo, hi), and the tile's.
    const int pos = u.s.pos + tok;
    const int hi = p.causal ? max(0, min(pos + 1, u.s.len)) : u.s.len;
    const int lo = p.window ? max(0, pos + 1 - p.window) : 0;
    const int first_tok = u.m * MT / p.G, last_tok = min(rows - 1, u.m * MT + MT - 1) / p.G;
    const int tile_hi = p.causal ? max(0, min(u.s.pos + last_tok + 1, u.s.len)) : u.s.len;
    const int tile_lo = p.window ? max(0, u.s.pos + first_tok + 1 - p.window) : 0;

    const float c = p.scale * LOG2E;
    float m = -INFINITY, l = 0.f;
    f32x16 acc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) acc[i] = f32x16{};

    for (int t0 = tile_lo & -TK; t0 < tile_hi; t0 += TK) {
        __syncthreads();
        {
            // 16 rows a wave, all of one page
            const int key = t0 + 16 * wave;
            const int left = u.s.len - key;
            const int page = left > 0 ? page_of(p, u.n, key >> p.page_shift) : -1;
            const int in = key & ((1 << p.page_shift) - 1);
            const int n = page < 0 ? 0 : min(left, 16);
            const int64_t pg = page < 0 ? 0 : page;
            load_rows<D>(p.k + pg * p.k_page + in * p.k_token + u.h * p.k_head, p.k_token, n, lane,
                         kt + wave * (16 * D * 2));
            load_rows<D>(p.v + pg * p.v_page + in * p.v_token + u.h * p.v_head, p.v_token, n, lane,
                         vt + wave * (16 * D * 2));
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();

        f32x16 st[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            st[b] = f32x16{};
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
                st[b] = E::mfma(read_k<D>(kt, 32 * b + (lane & 31), 2 * s + half), q[s], st[b]);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = t0 + 32 * b + 8 * (i >> 2) + 4 * half + (i & 3);
                if (key < lo || key >= hi) st[b][i] = -INFINITY;
                mx = fmaxf(mx, st[b][i]);
            }
        mx = fmaxf(mx, other_half(mx));
        // (a row that has seen no key yet keeps m = -inf and subtracts 0)
        const float m2 = fmaxf(m, mx);
        const float sub = m2 == -INFINITY ? 0.f : m2 * c;
        const float alpha = fast_exp2(fmaf(m, c, -sub));
        m = m2;
        float sum = 0.f;
        u32x4 pt[4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float e0 = fast_exp2(fmaf(st[b][i], c, -sub)), e1 = fast_exp2(fmaf(st[b][i + 1], c, -sub));
                sum += e0 + e1;
                pt[2 * b + (i >> 3)][(i & 7) >> 1] = E::pack(e0, e1);
            }
        l = fmaf(l, alpha, sum);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            acc[d] *= alpha;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const u32x2 v0 = read_v<D>(vt, 16 * k + 4 * half, d, lane);
                const u32x2 v1 = read_v<D>(vt, 16 * k + 8 + 4 * half, d, lane);
                acc[d] = E::mfma(u32x4{v0.x, v0.y, v1.x, v1.y}, pt[k], acc[d]);
            }
        }
    }

    l += other_half(l);
    if (!live) return;
    const int64_t out = (p.cu_seqlens ? row0 + tok : (int64_t)u.n * p.T + tok) * p.HQ + head;
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const u32x2 w = {E::pack(acc[d][i] * inv, acc[d][i + 1] * inv),
                             E::pack(acc[d][i + 2] * inv, acc[d][i + 3] * inv)};
            *reinterpret_cast<u32x2*>(p.o + out * D + 32 * d + 2 * i + 4 * half) = w;
        }
    if (p.lse && half == 0)
        p.lse[out] = l > 0.f ? (m * c + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
}

template <class E, int D>
hipError_t launch(const PagedParams& p, hipStream_t stream) {
    // at most this many (packed sequences each leave one tile unfilled)
    const int64_t tiles = p.cu_seqlens ? ((int64_t)p.T * p.G) / MT + p.N : (int64_t)p.N * (((int64_t)p.T * p.G + MT - 1) / MT);
    paged_attn_kernel<E, D><<<dim3((unsigned)(tiles * p.HKV)), dim3(256), 0, stream>>>(p);
    return hipGetLastError();
}

}  // namespace

size_t paged_attn_workspace(const PagedParams&, int) { return 0; }

hipError_t launch_paged_attn(const PagedParams& p, int D, hipStream_t stream) {
    if (D == 128) return p.fp16 ? launch<FP16, 128>(p, stream) : launch<BF16, 128>(p, stream);
    return p.fp16 ? launch<FP16, 64>(p, stream) : launch<BF16, 64>(p, stream);
}

}  // namespace kda
