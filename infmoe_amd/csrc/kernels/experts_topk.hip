// Choice of the type's launch sequence for the experts' products (experts_topk_run.h).
#include "kernels.h"

namespace infmoe {

hipError_t launch_experts_topk_f32(int T, int k, int E, int d, int h, int ffn, const void* x, long long x_stride, const int* ids, const float* weights, const void* wi, const void* wi_1,
                                  const void* wo, long long wi_stride, long long wo_stride, void* y, long long y_stride, void* workspace, hipStream_t stream);
hipError_t launch_experts_topk_f16(int T, int k, int E, int d, int h, int ffn, const void* x, long long x_stride, const int* ids, const float* weights, const void* wi, const void* wi_1,
                                  const void* wo, long long wi_stride, long long wo_stride, void* y, long long y_stride, void* workspace, hipStream_t stream);
hipError_t launch_experts_topk_bf16(int T, int k, int E, int d, int h, int ffn, const void* x, long long x_stride, const int* ids, const float* weights, const void* wi, const void* wi_1,
                                  const void* wo, long long wi_stride, long long wo_stride, void* y, long long y_stride, void* workspace, hipStream_t stream);

hipError_t launch_experts_topk(int T, int k, int E, int d, int h, int ffn, int dtype, const void* x, long long x_stride, const int* ids,
                               const float* weights, const void* wi, const void* wi_1, const void* wo, long long wi_stride,
                               long long wo_stride, void* y, long long y_stride, void* workspace, hipStream_t stream) {
    if (T <= 0) return hipSuccess;
    const auto launch = dtype == DTYPE_F32 ? launch_experts_topk_f32 : dtype == DTYPE_F16 ? launch_experts_topk_f16 : launch_experts_topk_bf16;
    return launch(T, k, E, d, h, ffn, x, x_stride, ids, weights, wi, wi_1, wo, wi_stride, wo_stride, y, y_stride, workspace, stream);
}

}  // namespace infmoe
