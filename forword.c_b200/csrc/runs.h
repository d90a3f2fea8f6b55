// runs.h — where a tensor of strided rows lies, for the C entry points that write one.
#pragma once
#include <cstddef>
#include <cstdint>

namespace fwb {

// Three levels of runs, widest stride first; levels of one are left out.  false:
// the runs may overlap one another, each level not reaching past the stride of
// the next.
struct Runs {
    uint64_t n[3], stride[3], span;  // span: bytes from the first to the last
    int levels = 0;
    bool nested(uint64_t run, const size_t (&counts)[3], const size_t (&strides)[3]) {
        for (int i = 0; i < 3; ++i) {
            if (counts[i] == 1) continue;
            int at = levels++;
            for (; at > 0 && stride[at - 1] < strides[i]; --at) {
                n[at] = n[at - 1];
                stride[at] = stride[at - 1];
            }
            n[at] = counts[i];
            stride[at] = strides[i];
        }
        span = run;
        for (int i = levels - 1; i >= 0; --i) {
            uint64_t over;
            if (stride[i] < span || __builtin_mul_overflow(n[i] - 1, stride[i], &over) || over > (uint64_t)1 << 62) return false;
            span += over;
        }
        return true;
    }
    // Whether runs of the same layout, the first `off` bytes on, shares a byte with this one.
    bool meets(int64_t off, uint64_t run, int level = 0) const {
        if (level == levels) return off < (int64_t)run && off > -(int64_t)run;
        // the two multiples of the stride around it: the smaller levels reach no further than one stride
        const int64_t st = (int64_t)stride[level], q = off / st - (off % st < 0), most = (int64_t)n[level] - 1;
        for (int64_t i = q; i <= q + 1; ++i)
            if (i >= -most && i <= most && meets(off - i * st, run, level + 1)) return true;
        return false;
    }
};

}  // namespace fwb
