// vxs_attn_types.h — a call's instance of a kernel, by head size and types.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <type_traits>

#include "../../include/vxs_sampler.h"

namespace vxs {

// Lets a kernel have `bytes` of dynamic LDS on the current device, once for each of them (`devices`: the kernel's own).
inline hipError_t allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& devices) {
    int d = 0;
    if (const hipError_t e = hipGetDevice(&d); e != hipSuccess) return e;
    const uint64_t bit = uint64_t(1) << (d & 63);
    if (d < 64 && (devices.load(std::memory_order_relaxed) & bit)) return hipSuccess;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) devices.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

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
