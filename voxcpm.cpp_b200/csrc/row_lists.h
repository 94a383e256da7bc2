// Row lists: runs of `bytes` bytes at base + i * stride[0] + j * stride[1] + ..., as a call's scores and row positions lie in memory.
// Host code without CUDA: whether two of a call's lists, or a list and another buffer, share bytes.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <initializer_list>
#include <utility>

namespace vox {

struct RowLists {
    static constexpr int kDims = 3;
    uint64_t base, bytes;
    int64_t  n[kDims];
    uint64_t stride[kDims];

    RowLists(const void * at, size_t bytes_, std::initializer_list<std::pair<int64_t, size_t>> dims)
        : base(reinterpret_cast<uint64_t>(at)), bytes(bytes_) {
        int d = 0;
        for (const auto & x : dims) { n[d] = x.first; stride[d] = x.second; ++d; }
        for (; d < kDims; ++d) { n[d] = 1; stride[d] = 0; }
        for (d = 0; d < kDims; ++d)
            if (n[d] <= 1) stride[d] = 0;
        for (int a = 0; a < kDims; ++a)  // by falling extent: the first one is not walked below
            for (int b = a + 1; b < kDims; ++b)
                if (n[b] > n[a]) { std::swap(n[a], n[b]); std::swap(stride[a], stride[b]); }
    }
    uint64_t end() const {
        uint64_t e = base + bytes;
        for (int d = 0; d < kDims; ++d) e += (uint64_t) (n[d] - 1) * stride[d];
        return e;
    }

    // Every list clear of the sum of those of shorter strides: then no two meet, and a gap of `room` bytes is left behind each.
    bool nested(uint64_t room) const {
        uint64_t s[kDims], span = room;
        int64_t  m[kDims];
        int      order[kDims] = {0, 1, 2};
        std::sort(order, order + kDims, [&](int a, int b) { return stride[a] < stride[b]; });
        for (int d = 0; d < kDims; ++d) { s[d] = stride[order[d]]; m[d] = n[order[d]]; }
        for (int d = 0; d < kDims; ++d) {
            if (m[d] <= 1) continue;
            if (s[d] < span) return false;
            span += (uint64_t) (m[d] - 1) * s[d];
        }
        return true;
    }

    // Is there a difference of indices, other than none at all if `others`, that puts one list's start into (lo, hi) from
    // another's?  Two of the extents are walked, the third is divided.
    bool differ_by(int64_t lo, int64_t hi, bool others) const {
        for (int64_t c = 1 - n[2]; c < n[2]; ++c)
            for (int64_t b = 1 - n[1]; b < n[1]; ++b) {
                const int64_t x = c * (int64_t) stride[2] + b * (int64_t) stride[1], s = (int64_t) stride[0];
                auto in = [&](int64_t a) { return a > -n[0] && a < n[0] && !(others && a == 0 && b == 0 && c == 0) && x + a * s > lo && x + a * s < hi; };
                if (s == 0) {
                    if (in(0) || in(1)) return true;
                    continue;
                }
                // the smallest a with x + a s > lo, and the ones behind it (two: the first may be `none at all`)
                int64_t a = (lo - x) / s;
                while (x + a * s > lo) --a;
                while (x + a * s <= lo) ++a;
                a = std::max(a, 1 - n[0]);
                if (in(a) || in(a + 1)) return true;
            }
        return false;
    }

    // two of the lists share a byte
    bool overlap() const { return bytes > 0 && !nested(bytes) && differ_by(-(int64_t) bytes, (int64_t) bytes, true); }

    // A list shares a byte with one of the same lists `other` bytes further on (scores and positions of equal strides).
    bool overlap_shifted(const void * other) const {
        const uint64_t o = reinterpret_cast<uint64_t>(other);
        if (bytes == 0 || o >= end() || o + (end() - base) <= base) return false;
        const uint64_t gap = o > base ? o - base : base - o;
        if (gap >= bytes && nested(gap + bytes)) return false;  // side by side in every gap
        const int64_t d = (int64_t) (o - base);
        return differ_by(d - (int64_t) bytes, d + (int64_t) bytes, false);
    }

    // A list shares a byte with [at, at + size).
    bool meets(const void * at, size_t size) const {
        const uint64_t a = reinterpret_cast<uint64_t>(at);
        if (at == nullptr || size == 0 || bytes == 0 || a >= end() || a + size <= base) return false;
        for (int64_t c = 0; c < n[2]; ++c)
            for (int64_t b = 0; b < n[1]; ++b) {
                const uint64_t x = base + (uint64_t) c * stride[2] + (uint64_t) b * stride[1];
                // the first list of this walk that ends behind `a`
                uint64_t i = x + bytes > a || stride[0] == 0 ? 0 : (a - x - bytes) / stride[0] + 1;
                i = std::min(i, (uint64_t) n[0] - 1);
                const uint64_t y = x + i * stride[0];
                if (y < a + size && y + bytes > a) return true;
            }
        return false;
    }
};

inline bool ranges_meet(const void * a, size_t a_size, const void * b, size_t b_size) {
    const uint64_t x = reinterpret_cast<uint64_t>(a), y = reinterpret_cast<uint64_t>(b);
    return a != nullptr && b != nullptr && x < y + b_size && y < x + a_size && a_size > 0 && b_size > 0;
}

}  // namespace vox
