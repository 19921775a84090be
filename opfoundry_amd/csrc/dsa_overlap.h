// dsa_overlap.h - whether strided rows share memory, for the host's checks of a
// call's outputs (include/dsa_chunk.h).  Plain C++, which a host-only test includes.
#ifndef DSA_OVERLAP_H_
#define DSA_OVERLAP_H_

#include <stdint.h>

namespace dsa_overlap {

typedef __int128 wide;         // no product of a count and a stride passes it

// Rows (t, h), t < T and h < H, of `width` elements from t * st + h * sh on.
struct Rows {
    int64_t T, H, st, sh, width;
};

inline wide extent(const Rows& r) { return (wide)(r.T - 1) * r.st + (wide)(r.H - 1) * r.sh + r.width; }

// Two rows of r share an element (or a stride is too short, or negative).
inline bool within(const Rows& r) {
    if (r.T < 1 || r.H < 1) return false;
    if ((r.T > 1 && r.st < r.width) || (r.H > 1 && r.sh < r.width)) return true;
    if (r.T == 1 || r.H == 1) return false;
    if ((wide)(r.H - 1) * r.sh + r.width <= r.st || (wide)(r.T - 1) * r.st + r.width <= r.sh) return false;
    // Rows d steps of the shorter dimension and e of the other, the other way, apart
    const bool t_short = r.T < r.H;
    const int64_t n = t_short ? r.T : r.H, m = t_short ? r.H : r.T, a = t_short ? r.st : r.sh, b = t_short ? r.sh : r.st;
    for (int64_t d = 1; d < n; ++d) {
        const wide at = (wide)d * a, e = at / b;
        if ((e < m && at - e * b < r.width) || (e + 1 < m && (e + 1) * b - at < r.width)) return true;
    }
    return false;
}

// A row of a and one of b share an element; b starts `delta` elements after a, T and the width are the same,
// strides not negative and b's rows apart from each other.  Where the two lie among one another with different
// token strides, or with several heads a token of different strides, the answer is yes without a closer look.
inline bool between(const Rows& a, const Rows& b, int64_t delta) {
    if (a.T < 1 || a.H < 1 || b.H < 1) return false;
    if (delta >= extent(a) || -(wide)delta >= extent(b)) return false;
    if (a.T > 1 && (a.st != b.st || a.st == 0)) return true;
    const int64_t s = a.T > 1 ? a.st : 0, w = a.width;
    if (s) {
        // a token's rows of b between those of a of the same (or an earlier) token and of the next
        int64_t d = delta % s;
        if (d < 0) d += s;
        if ((wide)(a.H - 1) * a.sh + w <= d && d + (wide)(b.H - 1) * b.sh + w <= s) return false;
    }
    if (a.H > 1 && b.H > 1 && a.sh != b.sh) return true;
    const int64_t sh = a.H > 1 ? a.sh : b.sh;
    for (int64_t h = 1 - a.H; h < b.H; ++h) {             // heads of b less heads of a
        const wide c = delta + (wide)h * sh;
        if (!s) {
            if (c > -w && c < w) return true;
            continue;
        }
        wide k = -c / s;                                  // tokens of b less tokens of a that bring them next to one another
        for (wide i = k - 1; i <= k + 1; ++i) {
            const wide x = c + i * s;
            if (i > -a.T && i < a.T && x > -w && x < w) return true;
        }
    }
    return false;
}

}  // namespace dsa_overlap

#endif  // DSA_OVERLAP_H_
