// linear_attention_f32.hip -- the kernels of linear_attention_core.h for one sample type.
#include "linear_attention_core.h"

namespace dspgpu {
namespace la {

int launch_f32(const Args &a, const Variant &v, hipStream_t s) {
    return launch_any<float, float>(a, v, s);
}

}  // namespace la
}  // namespace dspgpu
