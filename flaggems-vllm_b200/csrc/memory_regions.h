// Whether two strided arguments share memory: used by the C entry points and the native front ends before a launch.
#pragma once

#include <stdint.h>

#include <initializer_list>

namespace dsv4 {

// The bytes of an argument: `row` contiguous ones at every combination of up to three indices, `count` of them at a distance of `stride` bytes.
struct Region {
    struct Dimension {
        int64_t count, stride;
    };
    __int128 at = 0, row = 0, end = 0;  // no bytes where row is 0; products of sizes that a caller names need not fit into 64 bits
    Dimension dims[3] = {{1, 0}, {1, 0}, {1, 0}};

    Region(const void* p, __int128 bytes, std::initializer_list<Dimension> outer = {}) : at(reinterpret_cast<uintptr_t>(p)), row(p ? bytes : 0) {
        Dimension* d = dims;
        for (const Dimension& o : outer) {
            if (o.count <= 0) row = 0;
            if (o.count > 1) {
                *d = o;
                if (o.stride < 0) at += static_cast<__int128>(o.count - 1) * o.stride, d->stride = -o.stride;
            }
            ++d;
        }
        end = at + span(0);
    }
    // Bytes from the first to behind the last one, dimensions whose stride is a multiple of `modulus` left out (0: none left out).
    __int128 span(int64_t modulus) const {
        __int128 n = row;
        for (const Dimension& d : dims)
            if (d.count > 1 && (modulus == 0 || d.stride % modulus != 0)) n += static_cast<__int128>(d.count - 1) * d.stride;
        return n;
    }
};

// True where they are shown to share no byte: they lie in ranges apart, or, modulo one of their strides, in ranges apart (slices of the columns of
// one wide buffer, say).  Interleaved in another way they count as overlapping.
inline bool regions_apart(const Region& a, const Region& b) {
    if (a.row <= 0 || b.row <= 0) return true;
    if (a.end <= b.at || b.end <= a.at) return true;
    for (const Region* r : {&a, &b})
        for (const Region::Dimension& d : r->dims) {
            if (d.count <= 1 || d.stride <= 0) continue;
            const __int128 m = d.stride, of_a = a.span(d.stride), of_b = b.span(d.stride), behind = ((b.at - a.at) % m + m) % m;
            if (behind >= of_a && behind + of_b <= m) return true;
        }
    return false;
}

// Whether `a` shares memory with none of `others`.
inline bool apart_from_all(const Region& a, std::initializer_list<const Region*> others) {
    for (const Region* o : others)
        if (!regions_apart(a, *o)) return false;
    return true;
}

}  // namespace dsv4
