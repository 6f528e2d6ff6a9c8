// The products of experts_topk_run.h for _Float16.
#include "experts_topk_run.h"

namespace infmoe {

hipError_t launch_experts_topk_f16(int T, int k, int E, int d, int h, int ffn, const void* x, long long x_stride, const int* ids, const float* weights, const void* wi, const void* wi_1,
                                  const void* wo, long long wi_stride, long long wo_stride, void* y, long long y_stride, void* workspace, hipStream_t stream) {
    using E_ = _Float16;
    return run<E_>(T, k, E, d, h, ffn, static_cast<const E_*>(x), x_stride, ids, weights, static_cast<const E_*>(wi), static_cast<const E_*>(wi_1),
                   static_cast<const E_*>(wo), wi_stride, wo_stride, static_cast<E_*>(y), y_stride,
                   carve(T, k, E, d, h, DTYPE_F16, static_cast<char*>(workspace)), stream);
}

}  // namespace infmoe
