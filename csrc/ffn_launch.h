// What the launches of the feed-forward operators have in common.
#pragma once
#include <hip/hip_runtime.h>
#include "ffn_ops.h"
#include "ffn_common.h"
#include <c10/hip/HIPStream.h>

#define FFN_OK() do { hipError_t _e = hipGetLastError(); \
    TORCH_CHECK(_e == hipSuccess, "HIP error: ", hipGetErrorString(_e)); \
} while (0)

// runs the statement with T as the tensor's type
#define FFN_TYPES(type, ...) do { \
    if ((type) == at::kBFloat16) { typedef bf16_t T; __VA_ARGS__; } \
    else if ((type) == at::kHalf) { typedef f16_t T; __VA_ARGS__; } \
    else { typedef float T; __VA_ARGS__; } \
} while (0)

namespace ffn {

inline hipStream_t stream_now() {
    return c10::hip::getCurrentHIPStream().stream();
}

}  // namespace ffn
