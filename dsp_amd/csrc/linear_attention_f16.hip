// linear_attention_f16.hip -- the kernels of linear_attention_core.h for one sample type.
#include "linear_attention_core.h"

namespace dspgpu {
namespace la {

int launch_f16(const Args &a, const Variant &v, hipStream_t s) {
    return launch_any<_Float16, float>(a, v, s);
}

}  // namespace la
}  // namespace dspgpu
