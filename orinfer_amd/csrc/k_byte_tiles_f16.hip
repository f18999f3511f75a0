// Products by byte tiles of fp16 values.
#include "byte_tiles_kernel.h"

namespace orx {

int launch_byte_tiles_f16(const bytes::Product& p, int form, bool swiglu, uint32_t blocks, hipStream_t s) {
    return with_form(form, [&](auto which) { return Launch<F16, true>()(which, p, swiglu, blocks, s); });
}

}  // namespace orx
