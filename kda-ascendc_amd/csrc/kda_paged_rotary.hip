// The append to a paged cache with the position rotation on the way
// (kda_paged_hip.h): every pair (a, b) of the queries' and the new keys' turned
// elements by the angle x = position * inv_freq,
//   a' = a cos x - b sin x,  b' = b cos x + a sin x,
// in fp32, rounded once to the cache's type.
//
// A far position turns a pair thousands of times, and only what is left of the
// last turn counts: 32 bits have none of it at a position of 10^6 (an angle of
// 10^6 in fp32 is off by 0.03).  So the turns are counted in 64 bits, off by
// 4e-8 at the farthest position (2^30), and the fraction of the last one goes
// on in 32.
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
        sincospif(2.f * part, &sn[i], &cs[i]);
    }
}

// One thread a unit: 16 elements of one head of a token.  Of the turned units
// both pieces of 8 belong to the same 8 pairs: elements 8 u and rotary_dim / 2 +
// 8 u on, or, interleaved, 16 u and 16 u + 8 on.
template <int D, bool FP16>
__global__ __launch_bounds__(256) void paged_append_rotary_kernel(RotaryParams p, int total) {
    constexpr int UNITS = D / 16;
    const int id = blockIdx.x * 256 + threadIdx.x;
    if (id >= total) return;
    const int heads = p.HQ + 2 * p.HKV;
    const int unit = id % UNITS, x = id / UNITS;
    const int head = x % heads, t = x / heads;
    const int n = p.cu_seqlens ? sequence_of(p, t) : t / p.T;
    const NewTokens s = new_tokens(p, n);
    const int tok = p.cu_seqlens ? t - s.first : t - n * p.T;
    if (tok < 0 || tok >= s.count) return;
    const int pos = s.pos + tok;
    const int64_t row = p.cu_seqlens ? 0 : n, at = p.cu_seqlens ? t : tok;

    const bool turned = unit < p.units && head < p.HQ + p.HKV;
    const int first = !turned || p.interleaved ? 16 * unit : 8 * unit;
    const int second = !turned || p.interleaved ? first + 8 : first + 8 * p.units;
    const uint16_t* from;
    uint16_t* to;
    if (head < p.HQ) {
        from = p.q + row * p.q_row + at * p.q_token + head * p.q_head;
        to = p.q_out + row * p.out_row + at * p.out_token + head * p.out_head;
    } else {
        if (pos < 0) return;
        const int64_t page = table_entry(p, n, pos >> p.page_shift);
        if (!is_page(p, (int)page)) return;
        const int64_t in = pos & ((1 << p.page_shift) - 1);
        const int h = head - p.HQ;
        if (h < p.HKV) {
            from = p.nk + row * p.nk_row + at * p.nk_token + h * p.nk_head;
            to = p.k + page * p.k_page + in * p.k_token + h * p.k_head;
        } else {
            from = p.nv + row * p.nv_row + at * p.nv_token + (h - p.HKV) * p.nv_head;
            to = p.v + page * p.v_page + in * p.v_token + (h - p.HKV) * p.v_head;
        }
    }
    u32x4 lo = *reinterpret_cast<const u32x4*>(from + first), hi = *reinterpret_cast<const u32x4*>(from + second);
    if (turned) {
        float cs[8], sn[8], a[8], b[8];
        angles(p.inv_freq + 8 * unit, pos, cs, sn);
        unpack<FP16>(lo, a);
        unpack<FP16>(hi, b);
        if (p.interleaved) {
            // (neighbours: pairs 0 to 3 in the first piece, 4 to 7 in the second)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a0 = a[2 * i], a1 = a[2 * i + 1], b0 = b[2 * i], b1 = b[2 * i + 1];
                a[2 * i] = fmaf(a0, cs[i], -(a1 * sn[i]));
                a[2 * i + 1] = fmaf(a1, cs[i], a0 * sn[i]);
                b[2 * i] = fmaf(b0, cs[i + 4], -(b1 * sn[i + 4]));
                b[2 * i + 1] = fmaf(b1, cs[i + 4], b0 * sn[i + 4]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a0 = a[i], b0 = b[i];
                a[i] = fmaf(a0, cs[i], -(b0 * sn[i]));
                b[i] = fmaf(b0, cs[i], a0 * sn[i]);
            }
        }
        lo = pack<FP16>(a);
        hi = pack<FP16>(b);
    }
    *reinterpret_cast<u32x4*>(to + first) = lo;
    *reinterpret_cast<u32x4*>(to + second) = hi;
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
