// The memory that an argument's rows span, for checks of overlap.
#pragma once

#include <cstdint>

namespace airkv {

// The bytes that n > 0 rows of `width` elements, `stride` >= 0 apart, span (up to the end of the address
// space: their number may pass 64 bits where no such memory can be).
struct Span {
    uintptr_t at, end;
    Span(const void *p, int64_t n, int64_t stride, int64_t width, int64_t bytes) : at((uintptr_t)p) {
        const unsigned __int128 size = ((unsigned __int128)(n - 1) * (unsigned __int128)stride + (unsigned __int128)width) * (unsigned __int128)bytes;
        end = size > UINTPTR_MAX - at ? UINTPTR_MAX : at + (uintptr_t)size;
    }
    bool meets(const Span &o) const { return at < o.end && o.at < end; }
};

}  // namespace airkv
