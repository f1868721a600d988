// vxs_attn_core.h — what the attention kernels share: tiles of a paged cache on their way into LDS, and a wave's
// products with them on the matrix cores.
//
// A wave holds 32 query rows as the columns of 32x32x16 products. Scores come transposed, S^T = K Q^T: lane l has
// column c = l % 32 and, of each 32 keys, those 8 j + 4 (l / 32) + 0..3, j = 0..3, in 16 registers. So a query's
// maximum and sum stay within two lanes, rescaling is one factor per lane, and the weights are the second product's
// right operand where they are: O^T = V^T P^T, whose sum over keys may take them in any order as long as V^T's
// operand has the same one. V^T comes from the row-major tile through the transposing LDS read (16 lanes give four
// rows of 16 entries and get four keys of one entry each).
//
// A tile in LDS has its rows' 16-byte units at their index xor swizzle(row): the 16 rows at one unit that a K read
// touches at a time, and the 4 rows at 4 units of a V read, then lie in different banks. Tiles are loaded straight into
// LDS, 1 KiB a wave instruction in lane order; the swizzle is in the addresses that the lanes load from, whose rows
// stay whole.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vxs_attn.h"

namespace vxs {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Vec;
template <>
struct Vec<__bf16> {
    using v4 = bf4;
    using v8 = bf8;
    static constexpr unsigned kExponent = 0x7F80u;  // all ones: infinity or NaN
    static constexpr float kAbove = 8.0f;           // = kLag: m over the maximum when it is set
    static constexpr int kParts = 3;                // of an fp32 value: 8 bits each
    static constexpr float kPart = 1.0f;            // each part is multiplied by this more than the one before
    static __device__ __forceinline__ f16v mfma(bf8 a, bf8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Vec<_Float16> {
    using v4 = h4;
    using v8 = h8;
    static constexpr unsigned kExponent = 0x7C00u;
    static constexpr float kAbove = -7.0f;
    static constexpr int kParts = 2;  // 11 bits each
    static constexpr float kPart = 2048.0f;
    static __device__ __forceinline__ f16v mfma(h8 a, h8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Vec<float> {
    using v4 = f4;
};

// Whether one of the 8 entries of x (16 bits each) is infinite or NaN: its exponent's carry reaches the sign's place.
template <typename T>
__device__ __forceinline__ bool any_odd(u4 x) {
    constexpr unsigned kOne = 0x8000u - Vec<T>::kExponent, kBoth = kOne << 16 | kOne;
    unsigned y = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) y |= (x[i] & 0x7fff7fffu) + kBoth;
    return (y & 0x80008000u) != 0;
}

// The largest of three, NaN if one of them is: one instruction. The compiler has to know it, as every one that reads the result of
// a matrix product: it keeps the wait states between them, and sees no operands in inline assembly.
__device__ __forceinline__ float max3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }
// The larger of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.0e38f;  // a running maximum before any key
// Weights are exp2(score - m), and the sums are rescaled only when some query's maximum has grown by more than kLag since
// m was set: for bf16 to kLag above the maximum, so that no weight passes 1; for fp16, whose values end at 2^16 and whose
// precision ends at 2^-14, to 7 below it: weights reach 2^15, and those down to 2^-21 of the largest keep fp16's bits.
constexpr float kLag = 8.0f;

template <int N>
__device__ __forceinline__ void wait_vm() {  // all but the N youngest loads into LDS have arrived
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ const char* uniform_ptr(const char* p) {
    const uint64_t x = (uint64_t)p;
    return (const char*)((uint64_t)(unsigned)uniform((int)(x >> 32)) << 32 | (unsigned)uniform((int)x));
}

template <int D>
struct TileGeom {
    static constexpr int kRow = 2 * D;           // bytes
    static constexpr int kUnits = D / 8;         // 16-byte units of a row
    static constexpr int kRows = 64 / kUnits;    // rows of one load instruction
    static constexpr int kLoads = 16 / kRows;    // of 16 rows
    static __device__ __forceinline__ int swizzle(int row) {
        return D >= 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    }
};

// Loads of 16 rows (a granule: always within one page) of a cache into LDS.
template <int D>
struct Loader {
    using G = TileGeom<D>;
    unsigned off[G::kLoads];  // this lane's byte offsets within a granule
    __device__ __forceinline__ void init(const PagedCache& c, int lane) {
#pragma unroll
        for (int j = 0; j < G::kLoads; j++) {
            const int row = j * G::kRows + lane / G::kUnits;
            off[j] = (unsigned)row * (unsigned)c.token_stride + 16u * (unsigned)((lane % G::kUnits) ^ G::swizzle(row));
        }
    }
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is no register that the compiler would save: it only has to know)
    // base: the granule's first row (uniform); lds: where its rows go
    __device__ __forceinline__ void load(const char* base, unsigned lds) const {
        base = uniform_ptr(base);
        lds = uniform((int)lds);
#pragma unroll
        for (int j = 0; j < G::kLoads; j++)
            // (inline, or the compiler would wait for all of them before any read of LDS; a base that a vector instruction has just
            // written needs five wait states before the load, m0 one, and the compiler counts none here)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds + 1024u * j), "v"(off[j]), "s"(base)
                         : "m0", "memory");
    }
#pragma clang diagnostic pop
};

// Read-only memory of the launch, read with scalar loads: they are not counted with the loads into LDS.
template <typename A>
using Constant = const __attribute__((address_space(4))) A;
__device__ __forceinline__ int scalar(const int32_t* p, int64_t i) { return ((Constant<int32_t>*)p)[i]; }
// The kernel's arguments (of type A, the first) read again: kept from the start they would hold registers throughout.
template <typename A>
__device__ __forceinline__ A arguments_again() {
#ifdef __HIP_DEVICE_COMPILE__
    Constant<A>* p = (Constant<A>*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
#else
    return A{};
#endif
}

// Byte offset, from k or v at `head`, of the granule that begins at token t (uniform) of a slot whose table entries are
// `pages`, the last of them at `last`. Granules past a sequence's end read what is there in the pool.
__device__ __forceinline__ uint64_t granule_offset(const PagedCache& c, const int32_t* pages, int last, int t) {
    return cache_offset(c, scalar(pages, min(t >> c.page_bits, last)), 0, t);
}

// BYTES of a tile of values in LDS (whole rows, the first of which is key `row0` of the tile) before weights of zero meet
// them: rows from `end` on, which nobody sees and which may hold anything, become zero, and with `each` so do entries
// that are not finite, since some query does not see them; true in a lane that found such.
template <int D, typename T, int BYTES>
__device__ __forceinline__ bool scrub(char* rows, int row0, int end, bool each, int lane) {
    asm volatile("" : "+v"(lane));  // (few tiles come here: addresses are formed here too, and hold no registers of the others)
    bool found = false;
#pragma unroll
    for (int i = 0; i < BYTES / 1024; i++) {
        const int at = 16 * (64 * i + lane);
        u4* p = reinterpret_cast<u4*>(rows + at);
        if (row0 + at / (2 * D) >= end) {
            *p = u4{0, 0, 0, 0};
        } else if (each) {
            u4 x = *p;
            if (any_odd<T>(x)) {
                found = true;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if ((x[e] & Vec<T>::kExponent) == Vec<T>::kExponent) x[e] &= 0xffff0000u;
                    if ((x[e] >> 16 & Vec<T>::kExponent) == Vec<T>::kExponent) x[e] &= 0xffffu;
                }
                *p = x;
            }
        }
    }
    return found;
}

// A wave's 32 queries: operand, running maximum, sum of its own keys' weights, and outputs O^T.
template <int D, typename T, int PARTS>
struct Queries {
    using G = TileGeom<D>;
    using v8 = typename Vec<T>::v8;
    v8 q[D / 16];
    f16v o[D / 32];
    float m, l;

    __device__ __forceinline__ void init() {
        m = kLowest;
        l = 0.f;
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[b][i] = 0.f;
    }
    // row: this lane's query (null: zeros); the 8 entries at 16 t + 8 (lane / 32) are the lane's for step t
    __device__ __forceinline__ void load(const T* row, int lane) {
#pragma unroll
        for (int t = 0; t < D / 16; t++) {
            v8 x{};
            if (row) x = *reinterpret_cast<const v8*>(row + 16 * t + 8 * (lane >> 5));
            q[t] = x;
        }
    }
    __device__ __forceinline__ void loaded() {  // the wait for load() is here (and for every load into LDS before)
#pragma unroll
        for (int t = 0; t < D / 16; t++) asm volatile("" : "+v"(q[t]));
    }

    // S^T of 32 keys at `tile`
    __device__ __forceinline__ f16v scores(const char* tile, int lane) const {
        const int row = lane & 31;
        const char* p = tile + row * G::kRow;
        const int u = ((lane >> 5) ^ G::swizzle(row)) << 4;
        f16v s{};
#pragma unroll
        for (int t = 0; t < D / 16; t++) s = Vec<T>::mfma(*reinterpret_cast<const v8*>(p + ((32 * t) ^ u)), q[t], s);
        return s;
    }

    // Weights of NB x 32 keys from their scores; c = scale log2 e. The sums are rescaled when they have to be.
    template <int NB>
    __device__ __forceinline__ void weigh(f16v (&s)[NB], float c) {
        float top = kLowest;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i += 2) top = max3(top, s[b][i], s[b][i + 1]);
        top = max_halves(top) * c;
        if (__ballot(top > m + (kLag - Vec<T>::kAbove))) {
            // (where a score is NaN so are the weight and the sums, whatever m is: it stays)
            const float next = fmaxf(m, top + Vec<T>::kAbove), shrink = __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= shrink;
#pragma unroll
            for (int b = 0; b < D / 32; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[b][i] *= shrink;
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], c, -m));
                part[i & 3] += s[b][i];
            }
            l += (part[0] + part[1]) + (part[2] + part[3]);
        }
    }

    // Unseen keys of a tile have no weight: this lane's query sees `seen` of its keys (which may be negative or more).
    template <int NB>
    static __device__ __forceinline__ void hide(f16v (&s)[NB], int seen, int lane) {
        seen -= 4 * (lane >> 5);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (32 * b + 8 * (i >> 2) + (i & 3) >= seen) s[b][i] = -__builtin_inff();
    }

    // Four keys of 32 entries of V^T, twice: rows 16 t + 8 u + 4 (lane / 32) + 0..3 of `tile`, entries 32 b + lane % 32.
    static __device__ __forceinline__ s8 values(const char* tile, int t, int b, int lane) {
        const int i = lane & 15, g = lane >> 4;
        const int row = 4 * (g >> 1) + (i >> 2);
        const int unit = (2 * (g & 1) + ((i & 3) >> 1)) ^ G::swizzle(row);
        const char* p = tile + row * G::kRow + 8 * (i & 1);
        using lds_s4 = __attribute__((address_space(3))) s4;
        // (8 rows further the swizzle differs in bit 1)
        const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 16 * t * G::kRow + ((64 * b) ^ (unit << 4))));
        const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + (16 * t + 8) * G::kRow + ((64 * b) ^ (unit << 4) ^ 32)));
        return s8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    }
    // Eight weights in PARTS of T's bits, each the rounded rest of those before, times kPart: an fp16 rest would have nothing left
    // of its bits for all but the largest weights.
    static __device__ __forceinline__ void weights(const f16v& s, int t, v8 (&part)[PARTS]) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float rest = s[8 * t + e];
#pragma unroll
            for (int i = 0; i < PARTS; i++) {
                part[i][e] = (T)rest;
                rest = (rest - (float)part[i][e]) * Vec<T>::kPart;
            }
        }
    }

    // O^T += V^T P^T over NB x 32 keys. The weights are rounded to T once, as the outputs are: half an ulp of each weight, at random,
    // is as much of the output as its own rounding (an fp16 weight below 2^-21 of the largest has an error of 2^-32 of that, so a
    // million of them stay below the output's rounding). Outputs in fp32 take PARTS products instead, of all the weights' bits that
    // matter to them: 24 (bf16), or 22, down to 2^-44 of the largest weight (fp16, whose second products have sums of their own until
    // the end of the tile). A weight of zero hides values that are finite only: see scrub().
    template <int NB>
    __device__ __forceinline__ void add(const char* tile, const f16v (&s)[NB], int lane) {
        v8 part[2 * NB][PARTS];
#pragma unroll
        for (int k = 0; k < 2 * NB; k++) weights(s[k >> 1], k & 1, part[k]);
#pragma unroll
        for (int b = 0; b < D / 32; b++) {
            if constexpr (PARTS == 1 || Vec<T>::kPart == 1.0f) {
#pragma unroll
                for (int k = 0; k < 2 * NB; k++) {
                    const v8 v = __builtin_bit_cast(v8, values(tile, k, b, lane));
#pragma unroll
                    for (int i = PARTS - 1; i >= 0; i--) o[b] = Vec<T>::mfma(v, part[k][i], o[b]);
                }
            } else {
                static_assert(PARTS == 2);
                f16v rest{};
#pragma unroll
                for (int k = 0; k < 2 * NB; k++) {
                    const v8 v = __builtin_bit_cast(v8, values(tile, k, b, lane));
                    rest = Vec<T>::mfma(v, part[k][1], rest);
                    o[b] = Vec<T>::mfma(v, part[k][0], o[b]);
                }
#pragma unroll
                for (int i = 0; i < 16; i++) o[b][i] = __builtin_fmaf(rest[i], 1.0f / Vec<T>::kPart, o[b][i]);
                if (D == 256) __builtin_amdgcn_sched_barrier(0);  // (one block's rest at a time, or registers spill)
            }
        }
    }

    // Adds a key's values that are not finite (row: its values in memory), where this lane's query sees it.
    __device__ __forceinline__ void add_odd(const char* row, bool sees, int lane) {
        row += 8 * (lane >> 5);
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const s4 x = *reinterpret_cast<const s4*>(row + 64 * b + 16 * j);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (((unsigned short)x[e] & Vec<T>::kExponent) == Vec<T>::kExponent && sees)
                        o[b][4 * j + e] += (float)__builtin_bit_cast(T, (short)x[e]);
            }
    }

    __device__ __forceinline__ void finish_sum() { l += __shfl_xor(l, 32); }
};

}  // namespace vxs
