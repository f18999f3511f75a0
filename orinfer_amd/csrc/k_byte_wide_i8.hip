// Products by byte tiles of 8-bit integers, weights straight into registers.
#include "byte_wide_kernel.h"

namespace orx {

int launch_byte_wide_i8(const bytes::Product& p, int form, bool grouped, bool swiglu, uint32_t blocks, hipStream_t s) {
    if (!grouped) return launch_wide<I8, 8, false>(p, swiglu, blocks, s);
    return form == kWide128 ? launch_wide<I8, 8, true>(p, swiglu, blocks, s) : launch_wide<I8, 4, true>(p, swiglu, blocks, s);
}

}  // namespace orx
