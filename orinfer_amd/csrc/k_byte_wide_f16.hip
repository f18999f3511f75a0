// Products by byte tiles of fp16 values, weights straight into registers.
#include "byte_wide_kernel.h"

namespace orx {

int launch_byte_wide_f16(const bytes::Product& p, int form, bool swiglu, uint32_t blocks, hipStream_t s) {
    return form == kWide128 ? launch_wide<F16, 8, true>(p, swiglu, blocks, s) : launch_wide<F16, 4, true>(p, swiglu, blocks, s);
}

}  // namespace orx
