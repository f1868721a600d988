// vxs_attn_core8.h — what the attention kernels do otherwise over a cache of 8-bit entries (e4m3, a power of two for each
// block of 16 keys and head).
//
// Four significant bits are exact in bf16 and fp16, so entries become the queries' type where they leave LDS (v_cvt_scalef32_pk,
// two a lane and instruction at half rate) and the products are those of 16-bit caches. A block is 16 keys, a half of a lane's
// scores of 32: the keys' scale is a uniform factor in the exponent's argument, 8 scores at a time, and costs nothing; the values'
// is applied by their conversion, to bf16 whatever the queries are, since fp16's range may not hold them. A value is exact from
// a scale of 2^-117 on; below, bf16 rounds it to its least 2^-133.
//
// V^T comes from the row-major tile by the transposing LDS read of bytes: 16 lanes give 8 rows of 16 entries and get 8 keys
// of one entry each, the 8 of a lane's weights. A K read takes 16 entries of a key, those of two products (the queries' order of entries
// is the same). Rows' 16-byte units lie at their index xor swizzle(row): both reads then touch different banks.
#pragma once

#include <type_traits>

#include "vxs_attn_core.h"

namespace vxs {

typedef int i2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

template <int D>
struct TileGeom8 {
    static constexpr int kRow = D;               // bytes
    static constexpr int kUnits = D / 16;        // 16-byte units of a row
    static constexpr int kRows = 64 / kUnits;    // rows of one load instruction
    static constexpr int kLoads = 16 / kRows;    // of 16 rows
    // A K read is 16 rows at one unit, a V read rows 4 h + 0..3 and 8 + 4 h + 0..3 at two neighbouring ones: bit 2 of the row is in the
    // lowest bit, the others above it, as far as rows do not already differ in their place among the 256 bytes of all banks.
    static __device__ __forceinline__ int swizzle(int row) {
        if (D == 64) return (((row >> 3) & 1) << 1) | ((row >> 2) & 1);
        if (D == 128) return (((row >> 3) & 1) << 2) | (((row >> 1) & 1) << 1) | ((row >> 2) & 1);
        return (((row >> 3) & 1) << 3) | ((row & 3) << 1) | ((row >> 2) & 1);
    }
};

template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 widen(i2 x, float scale);
template <>
__device__ __forceinline__ bf8 widen<__bf16>(i2 x, float scale) {
    const bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[0], scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[0], scale, true);
    const bf2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[1], scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[1], scale, true);
    return bf8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <>
__device__ __forceinline__ h8 widen<_Float16>(i2 x, float scale) {
    const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)x[0], scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)x[0], scale, true);
    const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)x[1], scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)x[1], scale, true);
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The scale's byte of token t's block (uniform), of keys or values: scalar loads are of whole words.
__device__ __forceinline__ unsigned scale_byte(const uint8_t* scales, uint64_t index) {
    return ((unsigned)scalar(reinterpret_cast<const int32_t*>(scales), (int64_t)(index >> 2)) >> (8 * (index & 3))) & 255u;
}
// Scales of a tile of N granules; those that begin at `end` or after, which may hold anything, count as 1.
template <int N>
struct Scales {
    unsigned k[N], v[N];
    __device__ __forceinline__ void read(const PagedCache& c, const CacheScales& scales, int g, int page, int head, int t, int end) {
        const uint64_t at = scale_index(c, page, head, t);
        const unsigned kb = scale_byte(scales.k, at), vb = scale_byte(scales.v, at);
        k[g] = t < end ? kb : 127u;
        v[g] = t < end ? vb : 127u;
    }
};
// Scales of a tile of N granules on their way through LDS, as its entries: scalar loads would be waited for with the reads of LDS, a round
// trip to memory for each tile. [2 N] words at `at` are those that hold the bytes, keys' first.
template <int N>
struct ScaleWords {
    unsigned shift[N];  // a granule's byte in its words
    // One load, older than those of the tile that the caller asks for next. page[g]: of granule t + 16 g (uniform).
    __device__ __forceinline__ void ask(const PagedCache& c, const CacheScales& scales, const int (&page)[N], int head, int t, unsigned at, int lane) {
        int mine = page[0];
#pragma unroll
        for (int g = 0; g < N; g++) {
            shift[g] = 8 * ((unsigned)scale_index(c, page[g], head, t + 16 * g) & 3u);
            if (lane % N == g) mine = page[g];
        }
        const uint8_t* const p = ((lane / N) & 1 ? scales.v : scales.k) + (scale_index(c, mine, head, t + 16 * (lane % N)) & ~uint64_t(3));
        at = uniform((int)at);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dword %1, off" ::"s"(at), "v"(p) : "m0", "memory");
#pragma clang diagnostic pop
    }
    // The bytes of keys and values, once they are there; granules that begin at `end` or after, which may hold anything, count as 1.
    __device__ __forceinline__ void read(const char* at, int t, int end, unsigned (&k)[N], unsigned (&v)[N]) const {
        unsigned w[2 * N];
#pragma unroll
        for (int i = 0; i < 2 * N; i += 4) {
            const u4 x = *reinterpret_cast<const u4*>(at + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; e++) w[i + e] = x[e];
        }
#pragma unroll
        for (int g = 0; g < N; g++) {
            const bool there = t + 16 * g < end;
            k[g] = there ? (w[g] >> shift[g]) & 255u : 127u;
            v[g] = there ? (w[N + g] >> shift[g]) & 255u : 127u;
        }
    }
};
__device__ __forceinline__ float power(unsigned byte) { return __uint_as_float(byte << 23); }
// c 2^(byte - 127) > 0: what a key's product is multiplied by; never zero, which times the -inf of an unseen key would be NaN
__device__ __forceinline__ float score_factor(float c, unsigned byte) { return fmaxf(__builtin_ldexpf(c, (int)byte - 127), 0x1p-149f); }

// Into how many parts the weights go: as many as the outputs' bits need (vxs_attn_core.h), of bf16 over 8-bit entries.
template <typename T, typename TO, bool E8>
constexpr int weight_parts = E8 ? (sizeof(TO) == 4 ? 3 : std::is_same_v<TO, _Float16> ? 2 : 1) : sizeof(TO) == 4 ? Vec<T>::kParts : 1;

// NaN entries among 4 bytes: 0x80 in each.
__device__ __forceinline__ unsigned odd8(unsigned x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// scrub() of a tile of 8-bit values: rows of D bytes.
template <int D, int BYTES>
__device__ __forceinline__ bool scrub8(char* rows, int row0, int end, bool each, int lane) {
    asm volatile("" : "+v"(lane));
    bool found = false;
#pragma unroll
    for (int i = 0; i < BYTES / 1024; i++) {
        const int at = 16 * (64 * i + lane);
        u4* p = reinterpret_cast<u4*>(rows + at);
        if (row0 + at / D >= end) {
            *p = u4{0, 0, 0, 0};
        } else if (each) {
            u4 x = *p;
            unsigned any = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const unsigned odd = odd8(x[e]);
                any |= odd;
                x[e] &= ~((odd >> 7) * 255u);
            }
            if (any) {
                found = true;
                *p = x;
            }
        }
    }
    return found;
}

// A granule of 8-bit keys and values that a wave asks for, and later leaves in LDS in 16 bits, laid out as Loader's tiles: keys of
// bf16 times their scale, fp16's range may not hold that, so keys of fp16 as they are; values bf16 times their scale.
template <int D, typename T>
struct Stager {
    using G = TileGeom8<D>;
    u4 k[G::kLoads], v[G::kLoads];
    unsigned off[G::kLoads];
    int lane;
    __device__ __forceinline__ void init(const PagedCache& c, int l) {
        lane = l;
#pragma unroll
        for (int j = 0; j < G::kLoads; j++) off[j] = (unsigned)row(j) * (unsigned)c.token_stride + 16u * (unsigned)unit();
    }
    __device__ __forceinline__ int row(int j) const { return j * G::kRows + lane / G::kUnits; }
    __device__ __forceinline__ int unit() const { return lane % G::kUnits; }
    __device__ __forceinline__ void load(const char* keys, const char* values) {
#pragma unroll
        for (int j = 0; j < G::kLoads; j++) k[j] = *reinterpret_cast<const u4*>(keys + off[j]);
#pragma unroll
        for (int j = 0; j < G::kLoads; j++) v[j] = *reinterpret_cast<const u4*>(values + off[j]);
    }
    // vxs_attn_core.h's scrub() of the values, the first of which is key `row0`.
    __device__ __forceinline__ bool scrub(int row0, int end) {
        unsigned any = 0;
#pragma unroll
        for (int j = 0; j < G::kLoads; j++) {
            const bool there = row0 + row(j) < end;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const unsigned odd = odd8(v[j][e]);
                any |= there ? odd : 0u;
                v[j][e] = there ? v[j][e] & ~((odd >> 7) * 255u) : 0u;
            }
        }
        return any != 0;
    }
    __device__ __forceinline__ void store(char* keys, int values, const Scales<1>& scales) const {
        constexpr bool kFold = std::is_same_v<T, __bf16>;
        const float ks = kFold ? power(scales.k[0]) : 1.0f, vs = power(scales.v[0]);
#pragma unroll
        for (int j = 0; j < G::kLoads; j++) {
            const int r = row(j), u = (2 * unit()) ^ TileGeom<D>::swizzle(r);
            char* const p = keys + r * TileGeom<D>::kRow;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                *reinterpret_cast<typename Vec<T>::v8*>(p + ((u ^ i) << 4)) = widen<T>(i2{(int)k[j][2 * i], (int)k[j][2 * i + 1]}, ks);
                *reinterpret_cast<bf8*>(p + values + ((u ^ i) << 4)) = widen<__bf16>(i2{(int)v[j][2 * i], (int)v[j][2 * i + 1]}, vs);
            }
        }
    }
};

// Queries (vxs_attn_core.h) of type T over 8-bit keys and values; weights are bf16, in PARTS. STAGED: the tiles are in 16 bits.
template <int D, typename T, int PARTS, bool STAGED>
struct Queries8 : Queries<D, __bf16, PARTS> {
    using G = TileGeom8<D>;
    using Base = Queries<D, __bf16, PARTS>;
    using v8 = typename Vec<T>::v8;
    using Base::l;
    using Base::m;
    using Base::o;
    v8 q[D / 16];

    // row: this lane's query (null: zeros); entries 32 t + 16 (lane / 32) + 0..7 and + 8..15 are the lane's for steps 2 t and 2 t + 1
    // (staged: the 8 at 16 t + 8 (lane / 32) for step t)
    __device__ __forceinline__ void load(const T* row, int lane) {
#pragma unroll
        for (int t = 0; t < D / 16; t++) {
            v8 x{};
            if (row) x = *reinterpret_cast<const v8*>(row + (STAGED ? 16 * t + 8 * (lane >> 5) : 32 * (t >> 1) + 16 * (lane >> 5) + 8 * (t & 1)));
            q[t] = x;
        }
    }
    __device__ __forceinline__ void loaded() {
#pragma unroll
        for (int t = 0; t < D / 16; t++) asm volatile("" : "+v"(q[t]));
    }

    // S^T of 32 keys at `tile`, over their scales
    __device__ __forceinline__ f16v scores(const char* tile, int lane) const {
        const int row = lane & 31;
        f16v s{};
        if constexpr (STAGED) {
            const char* p = tile + row * TileGeom<D>::kRow;
            const int u = ((lane >> 5) ^ TileGeom<D>::swizzle(row)) << 4;
#pragma unroll
            for (int t = 0; t < D / 16; t++) s = Vec<T>::mfma(*reinterpret_cast<const v8*>(p + ((32 * t) ^ u)), q[t], s);
            return s;
        }
        const char* p = tile + row * G::kRow;
        const int u = ((lane >> 5) ^ G::swizzle(row)) << 4;
#pragma unroll
        for (int t = 0; t < D / 32; t++) {
            const u4 x = *reinterpret_cast<const u4*>(p + ((32 * t) ^ u));
            s = Vec<T>::mfma(widen<T>(i2{(int)x[0], (int)x[1]}, 1.0f), q[2 * t], s);
            s = Vec<T>::mfma(widen<T>(i2{(int)x[2], (int)x[3]}, 1.0f), q[2 * t + 1], s);
        }
        return s;
    }

    // Weights of NB x 32 keys from their scores; f: the factors of their blocks of 16.
    template <int NB>
    __device__ __forceinline__ void weigh(f16v (&s)[NB], const float (&f)[2 * NB]) {
        float top = kLowest;
#pragma unroll
        for (int g = 0; g < 2 * NB; g++) {
            float y = s[g >> 1][8 * (g & 1)];
#pragma unroll
            for (int i = 1; i < 7; i += 2) y = max3(y, s[g >> 1][8 * (g & 1) + i], s[g >> 1][8 * (g & 1) + i + 1]);
            y = __builtin_elementwise_maximum(y, s[g >> 1][8 * (g & 1) + 7]);
            top = __builtin_elementwise_maximum(top, y * f[g]);
        }
        top = max_halves(top);
        if (__ballot(top > m + (kLag - Vec<__bf16>::kAbove))) {
            const float next = fmaxf(m, top + Vec<__bf16>::kAbove), shrink = __builtin_amdgcn_exp2f(m - next);
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
                s[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], f[2 * b + (i >> 3)], -m));
                part[i & 3] += s[b][i];
            }
            l += (part[0] + part[1]) + (part[2] + part[3]);
        }
    }

    // Eight keys of 32 entries of V^T: rows 16 t + 8 u + 4 (lane / 32) + 0..3 of `tile` for u = 0, 1, entries 32 b + lane % 32.
    static __device__ __forceinline__ bf8 values(const char* tile, int t, int b, float scale, int lane) {
        const int i = lane & 15, g = lane >> 4;
        const int row = 4 * (g >> 1) + ((i >> 1) & 3) + 8 * (i >> 3);
        const int unit = (g & 1) ^ G::swizzle(row);
        const char* p = tile + row * G::kRow + 8 * (i & 1);
        using lds_i2 = __attribute__((address_space(3))) i2;
        return widen<__bf16>(__builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2*)(p + 16 * t * G::kRow + ((32 * b) ^ (unit << 4)))), scale);
    }

    using Base::add;
    // O^T += V^T P^T over NB x 32 keys; scale: of their values' blocks.
    template <int NB>
    __device__ __forceinline__ void add(const char* tile, const f16v (&s)[NB], const float (&scale)[2 * NB], int lane) {
        bf8 part[2 * NB][PARTS];
#pragma unroll
        for (int k = 0; k < 2 * NB; k++) Base::weights(s[k >> 1], k & 1, part[k]);
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int k = 0; k < 2 * NB; k++) {
                const bf8 v = values(tile, k, b, scale[k], lane);
#pragma unroll
                for (int i = PARTS - 1; i >= 0; i--) o[b] = Vec<__bf16>::mfma(v, part[k][i], o[b]);
            }
    }
};

// Adds a key's values that are not finite (row: its values in memory, of 8 bits with E8), where this lane's query sees it.
template <bool E8, int D, typename T, int PARTS>
__device__ __forceinline__ void add_odd(Queries<D, T, PARTS>& w, const char* row, bool sees, int lane) {
    if constexpr (E8) {
        row += 4 * (lane >> 5);
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned odd = odd8(*reinterpret_cast<const unsigned*>(row + 32 * b + 8 * j));
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if ((odd >> (8 * e)) & 128u && sees) w.o[b][4 * j + e] = __builtin_nanf("");
            }
    } else {
        w.add_odd(row, sees, lane);
    }
}

}  // namespace vxs
