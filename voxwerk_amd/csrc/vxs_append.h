// vxs_append.h — a head's norm and rotation, as the appends to 16-bit and 8-bit caches form them.
//
// D/8 lanes hold a head, each two runs of four entries, so that both entries of every pair are in one lane: for pairs
// (i, i + rot/2) runs 4u and 4u + rot/2, past the rotated part 4u' and 4u' + (D - rot)/2 of the rest; for interleaved pairs
// two neighbouring runs. An angle is position * inv_freq / 2pi in fp64, whose fraction (exact to 2^-20 of a turn at any int32
// position) goes to the fp32 sine and cosine, which take turns. With several axes each frequency takes the position of its own.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "vxs_attn.h"

namespace vxs {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Four;
template <>
struct Four<float> { using type = f4; };
template <>
struct Four<__bf16> { using type = bf4; };
template <>
struct Four<_Float16> { using type = h4; };

template <typename T>
__device__ __forceinline__ f4 load4(const T* p) {
    const typename Four<T>::type x = *reinterpret_cast<const typename Four<T>::type*>(p);
    return f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}
template <typename T>
__device__ __forceinline__ void store4(T* p, f4 v) {  // conversions round to nearest even
    *reinterpret_cast<typename Four<T>::type*>(p) = typename Four<T>::type{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
}

// A lane's place in a head: its runs at ra and rb, whether their pairs turn.
template <int D>
struct HeadLane {
    static constexpr int kLanes = D / 8;
    int u, ra, rb;
    bool inter, turned;
    __device__ __forceinline__ HeadLane(const vxs_kv_prep& p, int lane) {
        const int rot = p.rot_dim;
        u = lane % kLanes;
        inter = p.interleaved;
        turned = 8 * u < rot;
        ra = inter ? 8 * u : turned ? 4 * u : rot + (4 * u - rot / 2);
        rb = inter ? 8 * u + 4 : ra + (turned ? rot / 2 : (D - rot) / 2);
    }

    // Cosines and sines of token t's four pairs (1 and 0 where the lane's do not turn).
    template <typename Args>
    __device__ __forceinline__ void angles(const Args& a, int t, f4& c, f4& s) const {
        c = f4{1.f, 1.f, 1.f, 1.f};
        s = f4{0.f, 0.f, 0.f, 0.f};
        if (!turned) return;
        const f4 w = *reinterpret_cast<const f4*>(a.prep.inv_freq + 4 * u);
        int p[4];
        bool one = true;
        if constexpr (std::is_base_of_v<AppendAxesArgs, Args>) {
            one = a.axes.axes == 0;
            if (!one) {
                const i4 x = *reinterpret_cast<const i4*>(a.axes.d_axis + 4 * u);
#pragma unroll
                for (int e = 0; e < 4; e++) p[e] = a.pos[min(max(x[e], 0), a.axes.axes - 1) * a.axes.ld_pos + t];
            }
        }
        if (one) p[0] = p[1] = p[2] = p[3] = a.pos[t];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double turns = (double)p[e] * ((double)w[e] * 0.15915494309189533577);
            const float part = (float)(turns - __builtin_floor(turns));
            c[e] = __builtin_amdgcn_cosf(part) * a.prep.rope_scale;
            s[e] = __builtin_amdgcn_sinf(part) * a.prep.rope_scale;
        }
    }

    // x, y: the lane's runs of a head (all of its lanes are here); weight: of the norm.
    __device__ __forceinline__ void norm(f4& x, f4& y, const float* weight, float eps) const {
        const f4 wa = *reinterpret_cast<const f4*>(weight + ra), wb = *reinterpret_cast<const f4*>(weight + rb);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) sum = __builtin_fmaf(x[e], x[e], __builtin_fmaf(y[e], y[e], sum));
#pragma unroll
        for (int m = kLanes / 2; m >= 1; m /= 2) sum += __shfl_xor(sum, m);
        const float r = 1.0f / __builtin_sqrtf(sum * (1.0f / D) + eps);
        x = x * r * wa;
        y = y * r * wb;
    }
    __device__ __forceinline__ void rotate(f4& x, f4& y, f4 c, f4 s) const {
        if (!turned) return;
        if (inter) {
            const f4 xx{x[0] * c[0] - x[1] * s[0], x[0] * s[0] + x[1] * c[0], x[2] * c[1] - x[3] * s[1], x[2] * s[1] + x[3] * c[1]};
            const f4 yy{y[0] * c[2] - y[1] * s[2], y[0] * s[2] + y[1] * c[2], y[2] * c[3] - y[3] * s[3], y[2] * s[3] + y[3] * c[3]};
            x = xx;
            y = yy;
        } else {
            const f4 xx = x * c - y * s;
            y = x * s + y * c;
            x = xx;
        }
    }
};

// Where a token's block of pages lies: its page, or -1 where its slot, place or page lies outside the cache.
__device__ __forceinline__ int place_page(const PagedCache& c, int slot, int place) {
    if ((unsigned)slot >= (unsigned)c.slots || place < 0 || (place >> c.page_bits) >= c.ld_table) return -1;
    const int page = c.table[(int64_t)slot * c.ld_table + (place >> c.page_bits)];
    return (unsigned)page < (unsigned)c.pages ? page : -1;
}

}  // namespace vxs
