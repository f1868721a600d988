// The C entry points of the paged caches (vxs_attn_api.cpp, compiled with this file) on a host without a GPU: a context that only keeps
// the last error, and launchers that count how often they are reached. Built and driven by tests/test_attention8_host.py.
#include "../voxwerk_amd/csrc/vxs_attn.h"

#include "../voxwerk_amd/csrc/vxs_attn_plan.h"
#include "../voxwerk_amd/csrc/vxs_internal.h"

struct vxs_ctx {
    const char* error;
};
static vxs_ctx the_context{""};
static int launches;

extern "C" {
__attribute__((visibility("default"))) vxs_ctx* test_context() { return &the_context; }
__attribute__((visibility("default"))) int test_launches() { return launches; }
void* vxs_get_stream(const vxs_ctx*) { return nullptr; }
__attribute__((visibility("default"))) const char* vxs_last_error(const vxs_ctx* ctx) { return ctx->error; }
}

namespace vxs {
int ctx_fail(vxs_ctx* ctx, int code, const char* msg) {
    ctx->error = msg;
    return code;
}
int ctx_hip_fail(vxs_ctx* ctx, hipError_t, const char* what) { return ctx_fail(ctx, VXS_ERR_HIP, what); }
hipError_t ctx_use(vxs_ctx*) { return hipSuccess; }
int ctx_ok(vxs_ctx* ctx) {
    ctx->error = "";
    return VXS_OK;
}
hipError_t launch_kv_append(const AppendArgs&, int, int, hipStream_t) { return launches++, hipSuccess; }
hipError_t launch_kv8_append(const AppendArgs&, int, int, hipStream_t) { return launches++, hipSuccess; }
hipError_t launch_attn_prompt(const PromptArgs&, const CacheScales&, bool, int, int, hipStream_t) { return launches++, hipSuccess; }
hipError_t launch_attn_step(const StepArgs&, const CacheScales&, int, int, hipStream_t) { return launches++, hipSuccess; }
int64_t attn_step_work_bytes(const StepArgs& a) { return work_bytes(a); }
}  // namespace vxs
