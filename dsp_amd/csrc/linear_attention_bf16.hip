// linear_attention_bf16.hip -- the kernels of linear_attention_core.h for one sample type.
#include "linear_attention_core.h"

namespace dspgpu {
namespace la {

int launch_bf16(const Args &a, const Variant &v, hipStream_t s) {
    return launch_any<__bf16, __bf16>(a, v, s);
}

}  // namespace la
}  // namespace dspgpu
