// vxs_attn_types.h — a call's instance of a kernel, by head size and types.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/vxs_sampler.h"

namespace vxs {

// F<D, T, TO>::go(a, stream) for head_dim D, the cache's type T and the outputs' type TO.
template <template <int, typename, typename> class F, typename A>
hipError_t by_type(const A& a, int head_dim, int dtype, int out_dtype, hipStream_t stream) {
    auto dim = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (dtype == VXS_BF16) return out_dtype == VXS_F32 ? F<D, __bf16, float>::go(a, stream) : F<D, __bf16, __bf16>::go(a, stream);
        return out_dtype == VXS_F32 ? F<D, _Float16, float>::go(a, stream) : F<D, _Float16, _Float16>::go(a, stream);
    };
    switch (head_dim) {
        case 64: return dim(std::integral_constant<int, 64>{});
        case 128: return dim(std::integral_constant<int, 128>{});
        default: return dim(std::integral_constant<int, 256>{});
    }
}

}  // namespace vxs
