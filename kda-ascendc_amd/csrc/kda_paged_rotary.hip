// The append to a paged cache with the position rotation on the way
// (kda_paged_hip.h): every pair (a, b) of the queries' and the new keys' turned
// elements by the angle x = position * inv_freq,
//   a' = a cos x - b sin x,  b' = b cos x + a sin x,
// in fp32, rounded once to the cache's type.
//
// A far position turns a pair thousands of times, and only what is left of the
// last turn counts: 32 bits have none of it at a position of 10^6 (an angle of
// 10^6 in fp32 is off by 0.03).  So the turns are counted in 64 bits, off by
// 4e-8 at the farthest position (2^30), and the fraction of the last one goes on
// in 32, to the sine and cosine instructions, which count in turns and are off by
// 1.3e-7 at most (measured at 2^22 fractions of a turn).
#include "kda_common.h"
#include "kda_paged.h"

namespace kda {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Eight elements as floats and back (to the nearest, ties to even).
template <bool FP16>
__device__ __forceinline__ void unpack(u32x4 x, float (&f)[8]) {
    if constexpr (FP16) {
        const f16x8 h = __builtin_bit_cast(f16x8, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = lo_f(x[i]);
            f[2 * i + 1] = hi_f(x[i]);
        }
    }
}
template <bool FP16>
__device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (FP16)
            x[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{f[2 * i], f[2 * i + 1]}, f16x2));
        else
            x[i] = pack2(f[2 * i], f[2 * i + 1]);
    }
    return x;
}

// cos and sin of the angle of 8 pairs from `freq` on, at position `pos`.
__device__ __forceinline__ void angles(const float* freq, int pos, float (&cs)[8], float (&sn)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double turns = (double)pos * (double)freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
        const float part = (float)(turns - __builtin_rint(turns));
        cs[i] = __builtin_amdgcn_cosf(part);
        sn[i] = __builtin_amdgcn_sinf(part);
    }
}

__device__ __forceinline__ void turn(float& a, float& b, float cs, float sn) {
    const float x = a, y = b;
    a = fmaf(x, cs, -(y * sn));
    b = fmaf(y, cs, x * sn);
}

// The sequence of this lane's packed token t, of the wave's tokens t0 to t1:
// one load of the offsets instead of a chain of them where they are few.
__device__ __forceinline__ int sequence_in_wave(const PagedParams& p, int t, int t0, int t1, int lane) {
    if (p.N > 256) return sequence_of(p, t);
    int n = 0;
    int cu[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) cu[c] = 64 * c + lane < p.N ? paged_cu(p, 64 * c + lane) : 0x7fffffff;
    for (int x = t0; x <= t1; ++x) {
        int upto = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) upto += __popcll(__ballot(cu[c] <= x));
        if (t == x) n = max(upto - 1, 0);
    }
    return n;
}

// A thread turns (or moves) a unit, 16 elements of one head of a token.  Of the
// turned units both pieces of 8 belong to the same 8 pairs: elements 8 u and
// rotary_dim / 2 + 8 u on, or, interleaved, 16 u and 16 u + 8 on.
// Few tokens are bound by the chain of loads (offsets, length, table entry),
// many by HBM: on the GPU one token of 32 + 8 + 8 heads 2.5 us, 128 3.1, 16 packed
// prompts of 2311 tokens together (24 + 4 + 4 heads of 64, 19 MB) 6.2, 8192 tokens
// 36.2 (201 MB, 5.6 TB/s; a large copy reaches 5.2).  Two or four heads a thread,
// which need the angles once, were slower (single tokens 3.0 and 3.8 us, 8192 the
// same): the angles are not what bounds it.  Stores past the caches' lines:
// 8192 tokens 37.9 us without; with the attention that reads what was stored
// right after, 2048 tokens take 70.2 us instead of 69.1, 16 packed prompts 165.4
// instead of 166.0, 128 single tokens 40.1 instead of 40.4.
template <int D, bool FP16>
__global__ __launch_bounds__(256) void paged_append_rotary_kernel(RotaryParams p, int total) {
    constexpr int UNITS = D / 16;
    const int lane = threadIdx.x & 63;
    const int id = blockIdx.x * 256 + threadIdx.x;
    if (id - lane >= total) return;
    const bool live = id < total;
    const int heads = p.HQ + 2 * p.HKV;
    const int unit = id % UNITS, x = min(id, total - 1) / UNITS;
    const int head = x % heads, t = x / heads, h = head - p.HQ;
    const bool packed = p.cu_seqlens != nullptr;
    int n = packed ? 0 : t / p.T;
    const int64_t row = n, at = packed ? t : t - n * p.T;

    // The elements first: they do not wait for where they go.
    const bool turned = unit < p.units && h < p.HKV;
    const int first = turned && !p.interleaved ? 8 * unit : 16 * unit;
    const int second = first + (turned && !p.interleaved ? 8 * p.units : 8);
    const uint16_t* from = h < 0       ? p.q + row * p.q_row + at * p.q_token + head * p.q_head
                           : h < p.HKV ? p.nk + row * p.nk_row + at * p.nk_token + h * p.nk_head
                                       : p.nv + row * p.nv_row + at * p.nv_token + (h - p.HKV) * p.nv_head;
    u32x4 lo = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + first));
    u32x4 hi = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + second));
    if (packed) n = sequence_in_wave(p, t, __builtin_amdgcn_readfirstlane(t), __builtin_amdgcn_readlane(t, 63), lane);
    const NewTokens s = new_tokens(p, n);
    const int tok = packed ? t - s.first : (int)at;
    if (!live || tok < 0 || tok >= s.count) return;
    const int pos = s.pos + tok;
    uint16_t* to;
    if (h < 0) {
        to = p.q_out + row * p.out_row + at * p.out_token + head * p.out_head;
    } else {
        if (pos < 0) return;
        const int64_t page = table_entry(p, n, pos >> p.page_shift);
        if (!is_page(p, (int)page)) return;
        const int64_t in = pos & ((1 << p.page_shift) - 1);
        to = h < p.HKV ? p.k + page * p.k_page + in * p.k_token + h * p.k_head
                       : p.v + page * p.v_page + in * p.v_token + (h - p.HKV) * p.v_head;
    }
    if (turned) {
        float cs[8], sn[8], a[8], b[8];
        angles(p.inv_freq + 8 * unit, pos, cs, sn);
        unpack<FP16>(lo, a);
        unpack<FP16>(hi, b);
        if (p.interleaved) {
            // (neighbours: pairs 0 to 3 in the first piece, 4 to 7 in the second)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                turn(a[2 * i], a[2 * i + 1], cs[i], sn[i]);
                turn(b[2 * i], b[2 * i + 1], cs[i + 4], sn[i + 4]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) turn(a[i], b[i], cs[i], sn[i]);
        }
        lo = pack<FP16>(a);
        hi = pack<FP16>(b);
    }
    __builtin_nontemporal_store(lo, reinterpret_cast<u32x4*>(to + first));
    __builtin_nontemporal_store(hi, reinterpret_cast<u32x4*>(to + second));
}

template <int D>
hipError_t launch(const RotaryParams& p, hipStream_t stream) {
    const int64_t tokens = p.cu_seqlens ? p.T : (int64_t)p.N * p.T;
    const int64_t total = tokens * (p.HQ + 2 * p.HKV) * (D / 16);
    const dim3 grid((unsigned)((total + 255) / 256));
    if (p.fp16) paged_append_rotary_kernel<D, true><<<grid, 256, 0, stream>>>(p, (int)total);
    else paged_append_rotary_kernel<D, false><<<grid, 256, 0, stream>>>(p, (int)total);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append_rotary(const RotaryParams& p, int D, hipStream_t stream) {
    return D == 128 ? launch<128>(p, stream) : launch<64>(p, stream);
}

}  // namespace kda
