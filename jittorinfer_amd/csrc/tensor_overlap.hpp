// Whether two strided tensors share bytes.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace mla {

// What a tensor covers: runs of `run` bytes, `size[i]` of them `step[i]` bytes apart in each dimension, the largest step first.  Dimensions of one, and those that do
// not step (expanded ones), are left out.
struct Extent {
    static constexpr int DIMS = 6;
    uint64_t at = 0;                 // address of the first byte
    int64_t  run = 0;
    int      dims = 0;               // DIMS + 1: more than there is room for
    int64_t  step[DIMS], size[DIMS];

    // sizes and strides in elements, strides not negative
    Extent() = default;
    Extent(const void * data, int64_t element, int n, const int64_t * sizes, const int64_t * strides) : at((uint64_t) (uintptr_t) data), run(element) {
        for (int i = 0; i < n; i++) {
            if (sizes[i] == 0) { run = 0; dims = 0; return; }
            if (sizes[i] == 1 || strides[i] == 0) continue;
            if (dims >= DIMS) { dims = DIMS + 1; return; }
            int k = dims++;
            for (; k > 0 && step[k - 1] < strides[i] * element; k--) { step[k] = step[k - 1]; size[k] = size[k - 1]; }
            step[k] = strides[i] * element; size[k] = sizes[i];
        }
        while (dims > 0 && step[dims - 1] <= run) { run += step[dims - 1] * (size[dims - 1] - 1); dims--; }      // runs that follow each other are one
    }
    // bytes from the first to behind the last of dimensions d, d + 1, ..
    int64_t length(int d) const {
        int64_t n = run;
        for (int i = d; i < dims; i++) n += step[i] * (size[i] - 1);
        return n;
    }
};

enum class Shares { NO, YES, UNKNOWN };

// Dimensions da.. of a at offset 0 against db.. of b at offset `off`.  Where both step alike, two places of one beside the other are looked at; where they do not, a
// few; what stays open after `budget` looks is unknown.
inline Shares shares(const Extent & a, int da, const Extent & b, int db, int64_t off, int & budget) {
    const int64_t la = a.length(da), lb = b.length(db);
    if (off >= la || off + lb <= 0) return Shares::NO;
    if (da == a.dims && db == b.dims) return Shares::YES;
    if (--budget < 0) return Shares::UNKNOWN;
    Shares found = Shares::NO;
    auto look = [&](Shares s) { if (s != Shares::NO && found != Shares::YES) found = s; };
    const int64_t sa = da < a.dims ? a.step[da] : 0, sb = db < b.dims ? b.step[db] : 0;
    if (sa == sb) {
        const int64_t ia = a.length(da + 1), ib = b.length(db + 1);
        // b's place j less a's place i: m in (-size a, size b) with off + m sa in (-ib, ia)
        const int64_t na = a.size[da], nb = b.size[db];
        auto floor_div = [](int64_t x, int64_t y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
        const int64_t lo = std::max(1 - na, floor_div(-ib - off, sa) + 1), hi = std::min(nb - 1, -floor_div(off - ia, sa) - 1);
        for (int64_t m = lo; m <= hi && found != Shares::YES; m++) {
            look(shares(a, da + 1, b, db + 1, off + m * sa, budget));
            if (budget < 0) return found == Shares::YES ? found : Shares::UNKNOWN;
        }
        return found;
    }
    // the one of the larger step, place by place, as far as the other reaches
    const bool    first = sa > sb;
    const int64_t s = first ? sa : sb, n = first ? a.size[da] : b.size[db];
    const int64_t inner = first ? a.length(da + 1) : b.length(db + 1), from = first ? off : -off, to = from + (first ? lb : la);      // the other: [from, to)
    const int64_t lo = std::max<int64_t>(0, from - inner < 0 ? 0 : (from - inner) / s + 1), hi = std::min(n - 1, to <= 0 ? -1 : (to - 1) / s);
    for (int64_t i = lo; i <= hi && found != Shares::YES; i++) {
        look(first ? shares(a, da + 1, b, db, off - i * s, budget) : shares(a, da, b, db + 1, off + i * s, budget));
        if (budget < 0) return found == Shares::YES ? found : Shares::UNKNOWN;
    }
    return found;
}
inline Shares shares(const Extent & a, const Extent & b) {
    if (!a.run || !b.run || !a.at || !b.at) return Shares::NO;
    if (a.dims > Extent::DIMS || b.dims > Extent::DIMS) return Shares::UNKNOWN;
    int budget = 64;
    return shares(a, 0, b, 0, (int64_t) (b.at - a.at), budget);
}

}  // namespace mla
