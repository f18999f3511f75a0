// Products by byte tiles of 8-bit integers; and what the forms of the tiles are.
#include <algorithm>

#include "byte_tiles_kernel.h"

namespace orx {

int launch_byte_tiles_i8(const bytes::Product& p, int form, bool grouped, bool swiglu, uint32_t blocks, hipStream_t s) {
    return with_form(form, [&](auto which) { return grouped ? Launch<I8, true>()(which, p, swiglu, blocks, s) : Launch<I8, false>()(which, p, swiglu, blocks, s); });
}
TilesShape byte_tiles_shape(int kind, int form, bool grouped) {
    TilesShape shape = {};
    with_form(form, [&](auto which) {
        using FORM = decltype(which);
        const int lds = kind != I8 ? FORM::template lds<F16, true>() : grouped ? FORM::template lds<I8, true>() : FORM::template lds<I8, false>();
        shape = {FORM::bm, FORM::bn, 64 * FORM::waves, lds, std::min(160 * 1024 / lds, FORM::rows <= 2 ? 3 : 8 / FORM::waves)};
        return 0;
    });
    return shape;
}

}  // namespace orx
