// Products by byte tiles of bf16 values, weights straight into registers.
#include "byte_wide_kernel.h"

namespace orx {

int launch_byte_wide_bf16(const bytes::Product& p, int form, bool swiglu, uint32_t blocks, hipStream_t s) {
    return form == kWide128 ? launch_wide<BF16, 8, true>(p, swiglu, blocks, s) : launch_wide<BF16, 4, true>(p, swiglu, blocks, s);
}

}  // namespace orx
