// What the C entries of the operators on scores check before anything is queued.
#pragma once
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/thundergbm.h"
#include "tgbm_common.h"
#include "tgbm_scores.h"

namespace tgbm {

inline int size_of(int type) { return type == SCORE_F32 ? 4 : 2; }

inline ScoreView view_of(const char *what, const void *data, int type, int n, int k, long long row, long long cls, bool written) {
    const std::string w(what);
    TGBM_CHECK(type >= SCORE_F32 && type <= SCORE_BF16, w + ": unknown type");
    TGBM_CHECK(data != nullptr, w + ": null pointer");
    TGBM_CHECK(reinterpret_cast<uintptr_t>(data) % size_of(type) == 0, w + ": not aligned for its type");
    // (beyond SCORES_CLASS_MOST only where nothing else tells the layout: a slice of one such row is left to the kernels for any stride)
    const bool one_by_class = n == 1 && row >= 1 && (row == cls || (row < cls && k <= SCORES_CLASS_MOST));
    if (n == 1) row = k == 1 ? 1 : cls * k;   // a stride that no step takes
    if (k == 1) cls = row * n;
    TGBM_CHECK(row >= 0 && cls >= 0, w + ": negative stride");
    const long long most = LLONG_MAX / 16;
    TGBM_CHECK(row <= most / n && cls <= most / k, w + ": stride too large");
    if (written) TGBM_CHECK((row >= 1 && cls > (n - 1) * row) || (cls >= 1 && row > (k - 1) * cls), w + ": strides under which cells share memory");
    ScoreView v;
    v.data = const_cast<void *>(data); v.type = type; v.row = row; v.cls = cls; v.one_by_class = one_by_class;
    return v;
}

// whether two matrices of n x k share memory (true also where that is not easily told)
inline bool share_memory(const ScoreView &a, int a_size, const ScoreView &b, int b_size, int n, int k) {
    auto end = [&](const ScoreView &v, int size) { return reinterpret_cast<uintptr_t>(v.data) + size * (uintptr_t)((n - 1) * v.row + (k - 1) * v.cls + 1); };
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a.data), pb = reinterpret_cast<uintptr_t>(b.data);
    if (end(a, a_size) <= pb || end(b, b_size) <= pa) return false;
    if (a_size != b_size || a.row != b.row || a.cls != b.cls || (pa > pb ? pa - pb : pb - pa) % a_size) return true;
    // parts of one larger matrix, side by side: `d` cells apart are `over` lines and `in` cells
    const long long d = (long long)((pa > pb ? pa - pb : pb - pa) / a_size);
    const bool by_row = a.cls <= a.row;
    const long long line = by_row ? a.row : a.cls, step = by_row ? a.cls : a.row;
    const long long lines = by_row ? n : k, cells = by_row ? k : n;
    if (line <= 0) return true;
    const long long over = d / line, in = d % line, width = (cells - 1) * step + 1;
    return (in < width && over < lines) || (line - in < width && over + 1 < lines);
}

// Does [p, p + bytes) hold cells of the matrix?  (Where neither stride is 1 the gaps within a line count as cells.)
inline bool lies_in(const ScoreView &v, int size, int n, int k, const void *p, long long bytes) {
    if (!p || bytes <= 0) return false;
    const bool by_row = n > 1 && (k == 1 || v.cls <= v.row);
    const long long lines = by_row ? n : k, apart = size * (by_row ? v.row : v.cls), width = size * (by_row ? (k - 1) * v.cls + 1 : (n - 1) * v.row + 1);
    const long long lo = (long long)(reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(v.data)), hi = lo + bytes;
    if (hi <= 0 || lo >= (lines - 1) * apart + width) return false;
    return lo < width || ((lo - width) / apart + 1) * apart < hi;   // (the first line that ends behind `lo`)
}

inline void check_pointer(const char *what, const void *p, size_t size) {
    TGBM_CHECK(reinterpret_cast<uintptr_t>(p) % size == 0, std::string(what) + ": not aligned for its type");
}
inline void check_shape(int n, int k) {
    TGBM_CHECK(n >= 0, "negative number of rows");
    TGBM_CHECK(k >= 1 && k <= TGBM_SCORES_MAX_CLASSES, "number of classes outside [1, " + std::to_string(TGBM_SCORES_MAX_CLASSES) + "]");
}
inline void check_temperature(float t) { TGBM_CHECK(temperature_fits(t), "the temperature has to be a positive number"); }
inline void check_list(int top) { TGBM_CHECK(top >= 1 && top <= TGBM_SCORES_MAX_TOP, "length of a row's list outside [1, " + std::to_string(TGBM_SCORES_MAX_TOP) + "]"); }

inline void check_draws(int draws) {
    TGBM_CHECK(draws >= 1 && draws <= TGBM_SCORES_MAX_DRAWS, "draws of a row outside [1, " + std::to_string(TGBM_SCORES_MAX_DRAWS) + "]");
}
inline void check_limits(float temperature, int top_k, float top_p, float min_p) {
    TGBM_CHECK(temperature >= 0.f && temperature <= FLT_MAX, "the temperature has to be a number from 0 on");
    TGBM_CHECK(top_k >= 0, "top_k: negative");
    TGBM_CHECK(top_p >= 0.f && top_p <= 1.f, "top_p outside [0, 1]");
    TGBM_CHECK(min_p >= 0.f && min_p <= 1.f, "min_p outside [0, 1]");
}
inline void check_feedback(float clip_low, float clip_high, float kl, float entropy) {
    TGBM_CHECK(clip_low >= 0.f && clip_low <= 1.f && clip_high >= 0.f, "clip: the lower one outside [0, 1], or the upper one negative");
    TGBM_CHECK(kl >= 0.f && kl <= FLT_MAX && entropy >= 0.f && entropy <= FLT_MAX, "kl, entropy: negative or not finite");
}

template <typename F> int scores_call(F &&f) {
    try {
        set_last_error("");
        f();
        return 0;
    } catch (const std::exception &e) {
        set_last_error(e.what());
        return 1;
    }
}

}  // namespace tgbm
