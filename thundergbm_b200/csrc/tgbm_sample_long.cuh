// Classes drawn from long rows of scores.
#pragma once
#include <cfloat>
#include <climits>
#include <cmath>

#include <cooperative_groups.h>

#include "tgbm_sample.cuh"

namespace tgbm {
namespace {
namespace cg = cooperative_groups;

// ---- long rows: a cluster of up to 8 blocks (or one) holds the row in its registers -------------------------------------------
// Classes stand in the order block, u, thread, place in the pack (Hold); a segment is what a warp has of one u, 32 packs side by side.
//
// Limits: as above the scores that can be left are those from a border on, which is raised by bisection over the registers while more than
// LONG_LIST reach it.  They go into a list in the first block, in class order, and that block alone goes on: every entry counts the larger ones,
// which is its place in descending order; prefix sums in that order tell where top_p ends, prefix sums in class order which class a random number
// falls on.  Where top_p alone leaves more, what is certainly left is told from what the end of it lies among, and only that goes into the list.
// Rows with more than a list, and rows without limits, take their draws from sums per segment.
//
// Bound by instructions and by waiting for the cluster: 256 x 131072 in 16 bits, limits of their own for all rows, 211 to 264 us by what these are (floor
// 10.2), 96 instructions a score, 14 of them of the fp64 units (every exponential that a mass takes is a double); 16 draws for each of 333 x 50021 without limits
// 124 us (5.1), 116 instructions a score, 19 of them fp64: what is left of them is the cluster's exchanges and registers that the limits' code spills.
// 64 registers, so that two blocks share an SM: with 128 and one block 425 us and 233 (before the lists were narrowed).
constexpr int LONG_LIST = 1024;

template <int W, int S> struct LongRow {
    Powers powers;
    double sums[W], slot_sum[2], sum, front;          // of the warps, of this block (read by the others), of the row, of the blocks in front
    float lows[W], highs[W], slot_low[2], slot_high[2], low, high;
    int counts[W], slot_count[2], count, front_count;
    double segment[S];                                // of a segment, then of all in front of it
    int segment_count[S];
    int tie, last;
    float tie_score, at;
    __align__(16) unsigned key[LONG_LIST];
    int k[LONG_LIST];
    double w[LONG_LIST], upto[LONG_LIST];
};

// The list of a row, `size` entries in class order: what is left of it (w[i] > 0), prefix sums in class order (upto), its mass.  `base`: mass of what is
// larger than all entries (only where `border`: then the last entry that is left is told, in at and last).  All threads of a block.
template <int W, int S>
__device__ __noinline__ double settle_list(LongRow<W, S> &sh, const Exponent &weight, float top, int size, double min_p, int top_k, bool by_mass, bool of_list, double top_p,
                                           double all, double base, bool border) {
    constexpr int TH = 32 * W, Q = LONG_LIST / TH;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // exclusive prefix of the threads' sums
    auto scan = [&](double own, double &whole) {
        double upto = own;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const double v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        __syncthreads();
        if (lane == 31) sh.sums[warp] = upto;
        __syncthreads();
        double before = 0;
        whole = 0;
        for (int v = 0; v < W; ++v) {
            if (v == warp) before = whole;
            whole += sh.sums[v];
        }
        return before + (upto - own);
    };
    auto count = [&](int own) {
        own = warp_sum(own);
        __syncthreads();
        if (lane == 0) sh.counts[warp] = own;
        __syncthreads();
        int s = 0;
        for (int v = 0; v < W; ++v) s += sh.counts[v];
        return s;
    };
    if (tid < 4 && size + tid < LONG_LIST) sh.key[size + tid] = 0;   // (read four at a time)
    __syncthreads();
    int place[Q], heavy = 0;
    double mine[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = q * TH + tid;
        place[q] = size;
        mine[q] = 0;
        if (i < size) {
            const unsigned own = sh.key[i];
            mine[q] = weight(sh.powers, key_score(own), top);
            heavy += mine[q] >= min_p;
            int larger = 0;   // entries in front of this one in descending order: of equal ones those of lower classes
            for (int j = 0; j < size; j += 4) {
                const uint4 o = *reinterpret_cast<const uint4 *>(&sh.key[j]);
                const unsigned over = own + (j + 4 > i);
                larger += (o.x >= over) + (o.y >= over) + (o.z >= over) + (o.w >= over);
            }
            for (int j = i & ~3; j < i; ++j) larger += sh.key[j] == own;
            place[q] = larger;
        }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (place[q] < size) sh.w[place[q]] = mine[q];
    int keep = min(count(heavy), top_k);   // in descending order
    if (by_mass) {
        // entries tid Q + q in descending order: prefix sums
        double s = 0, whole;
#pragma unroll
        for (int q = 0; q < Q; ++q) s += tid * Q + q < keep ? sh.w[tid * Q + q] : 0.0;
        double upto = base + scan(s, whole);
        const double target = top_p * (of_list ? whole : all);
        int before = 0;   // entries in front of which the target is not reached
#pragma unroll
        for (int q = 0; q < Q; ++q)
            if (tid * Q + q < keep) {
                before += tid * Q + q == 0 || upto < target;
                upto += sh.w[tid * Q + q];
            }
        keep = count(before);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = q * TH + tid;
        if (i < size) {
            sh.w[i] = place[q] < keep ? mine[q] : 0.0;   // in class order now
            if (border && place[q] == keep - 1) { sh.at = key_score(sh.key[i]); sh.last = sh.k[i]; }
        }
    }
    __syncthreads();
    double s = 0, mass;
#pragma unroll
    for (int q = 0; q < Q; ++q) s += tid * Q + q < size ? sh.w[tid * Q + q] : 0.0;
    double upto = scan(s, mass);
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (tid * Q + q < size) {
            upto += sh.w[tid * Q + q];
            sh.upto[tid * Q + q] = upto;
        }
    __syncthreads();
    return sh.upto[size - 1];
}

template <typename T, int TH, int P, bool EVEN>
__global__ void __launch_bounds__(TH, 1024 / TH) k_sample_long(SampleArgs a, Scores<T> in) {
    typedef Hold<T, TH, P, EVEN> H;
    constexpr int V = H::V, W = TH / 32, S = P * W;
    __shared__ __align__(16) LongRow<W, S> sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long n = blockIdx.x / C;
    const int lo = rank * H::CELLS, cells = min(a.k - lo, H::CELLS);
    H hold;
    hold.read(in.at(n, lo), cells);
    if (warp == 0) sh.powers.fill();
    const Limits l = limits_of(a, n);
    // f(score, class - lo) in class order within u; -inf behind the last class
    auto each_of = [&](int u, auto &&f) {
        float v[V];
        if (H::first(u) < cells) hold.get(u, v);
#pragma unroll
        for (int i = 0; i < V; ++i) f(H::first(u) < cells ? v[i] : minus_inf(), H::first(u) + i);
    };
    auto each = [&](auto &&f) {
#pragma unroll
        for (int u = 0; u < P; ++u) each_of(u, f);
    };
    // of all threads of all blocks, the same everywhere; front, front_count: of the blocks in front of this one
    int turn = 0;
    double front = 0;
    int front_count = 0;
    auto total = [&](double &sum, float &low, float &high, int &count) {
        sum = warp_sum(sum); low = lanes_min<32>(low); high = lanes_max<32>(high); count = warp_sum(count);
        if (lane == 0) { sh.sums[warp] = sum; sh.lows[warp] = low; sh.highs[warp] = high; sh.counts[warp] = count; }
        __syncthreads();
        if (warp == 0) {
            sum = lanes_sum<W>(sh.sums[lane & (W - 1)]); count = lanes_sum<W>(sh.counts[lane & (W - 1)]);
            low = lanes_min<W>(sh.lows[lane & (W - 1)]); high = lanes_max<W>(sh.highs[lane & (W - 1)]);
            if (lane == 0) { sh.slot_sum[turn] = sum; sh.slot_low[turn] = low; sh.slot_high[turn] = high; sh.slot_count[turn] = count; }
        }
        if (C > 1) cluster.sync();
        if (warp == 0) {
            double before = 0, its = sum;
            int before_count = 0, its_count = count;
            if (C > 1) {
                const LongRow<W, S> *o = cluster.map_shared_rank(&sh, lane < C ? lane : 0);
                its = o->slot_sum[turn]; its_count = o->slot_count[turn]; low = o->slot_low[turn]; high = o->slot_high[turn];
                low = lanes_min<LONG_CLUSTER>(low); high = lanes_max<LONG_CLUSTER>(high);
                sum = 0; count = 0;
                for (int b = 0; b < C; ++b) {   // one after the other: where one block's part ends the next one's begins
                    if (b == rank) { before = sum; before_count = count; }
                    sum += __shfl_sync(0xffffffffu, its, b);
                    count += __shfl_sync(0xffffffffu, its_count, b);
                }
            }
            if (lane == 0) { sh.sum = sum; sh.low = low; sh.high = high; sh.count = count; sh.front = before; sh.front_count = before_count; }
        }
        __syncthreads();
        sum = sh.sum; low = sh.low; high = sh.high; count = sh.count; front = sh.front; front_count = sh.front_count;
        turn ^= 1;
    };
    // sums of the segments become those of all segments in front; returns the block's
    auto prefix = [&](auto *of) {
        auto before = of[0] - of[0];
        __syncthreads();
        if (warp == 0) {
            for (int s = 0; s < S; s += 32) {
                const auto own = s + lane < S ? of[s + lane] : before - before;
                auto upto = own;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const auto v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                if (s + lane < S) of[s + lane] = before + (upto - own);
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        __syncthreads();
    };
    float top = minus_inf(), low = -minus_inf(), none = 0;
    double sum = 0;
    int count = 0;
    if constexpr (EVEN) {
        top = hold.largest(cells);
        if (top != top) { count = 1; top = minus_inf(); }
    } else {
        each([&](float x, int) {
            top = fmaxf(top, x);
            count |= x != x;
        });
    }
    // Each group of lanes that holds a score has a largest one, and the least of these is reached by as many scores as there are groups: the first
    // guess of a border.  Groups are as large as they may be to be top_k.
    const int top_k = l.greedy ? 1 : l.top_k, groups = max(1, a.k / H::E);   // (threads that hold all their scores)
    {
        float its = top;
#pragma unroll
        for (int o = 1; o < 32; o *= 2)
            if (groups / (2 * o) >= max(top_k < a.k ? top_k : 0, 96)) its = fmaxf(its, __shfl_xor_sync(0xffffffffu, its, o));
        low = its > minus_inf() ? its : low;
    }
    total(sum, low, top, count);
    const bool bad = l.broken || count || top == -minus_inf();
    if (bad || top == minus_inf()) {   // (the same for all blocks; none reads another's memory any more than it did before the last barrier)
        const float v = bad ? __int_as_float(0x7fffffff) : minus_inf();
        if (rank == 0)
            for (int d = tid; d < a.draws; d += TH) put_draw(a, n * a.draws + d, -1, v, v);
        if (C > 1) cluster.sync();
        return;
    }
    const Exponent weight(l);
    auto weight_of = [&](float v) { return weight(sh.powers, v, top); };
    const bool by_count = top_k < a.k, by_mass = l.top_p < 1 && !l.greedy, by_share = l.min_p > 0 && !l.greedy;
    const float guess = low;
    double all = 0;
    // what is left: larger than `at`, or equal to it and a class up to `last`
    float at = minus_inf();
    int last = a.k;
    auto left = [&](float x, int k) { return x > at || (x == at && x > minus_inf() && lo + k <= last); };
    // masses of segments, of what is left
    auto segments = [&] {
        double s[P], mine = 0;
#pragma unroll
        for (int u = 0; u < P; ++u) {
            s[u] = 0;
            each_of(u, [&](float x, int k) { s[u] += left(x, k) ? weight_of(x) : 0.0; });
        }
        constexpr int PER = 32 / P;
        mine = sums_spread<P>(s);
        if (lane % PER == 0) {
            sh.segment[lane / PER * W + warp] = mine;
            sh.segment_count[lane / PER * W + warp] = mine > 0;
        }
        mine = lane % PER == 0 ? mine : 0.0;
        float f0 = 0, f1 = 0;
        int c0 = 0;
        total(mine, f0, f1, c0);
        prefix(sh.segment);
        return mine;
    };
    double mass = 0;
    bool listed = false;
    if (by_count || by_mass || by_share) {
        const float c = (float)(l.inv_t * 1.4426950408889634);
        const bool told = floats_tell(l);
        auto rough = [&](float x) { return exp2_fast(__fsub_rn(x, top) * c); };
        float f0 = 0, f1 = 0;
        int count_of_row = 0;   // (not looked at)
        unsigned reach = 0;   // scores from the border on
        // sum of floats over this thread's scores
        auto look = [&] {
            float2 part = make_float2(0.f, 0.f);
#pragma unroll
            for (int u = 0; u < P; ++u) {
                if (H::first(u) >= cells) continue;
                float v[V];
                hold.get(u, v);
                if constexpr (V == 1) {
                    part.x += rough(v[0]);
                } else {
                    const float2 mt = make_float2(-top, -top), c2 = make_float2(c, c);
#pragma unroll
                    for (int i = 0; i < V; i += 2) part = add2(part, exp_pair(make_float2(v[i], v[i + 1]), mt, c2));
                }
            }
            return (double)__fadd_rn(part.x, part.y);
        };
        const bool exact = !by_count && !by_share;   // top_p alone: a share of the whole mass (by floats at first)
        if (exact && told) {
            all = look();
            count = 0;
            total(all, f0, f1, count);
        }
        // the border, rounded down as in k_sample_limited, and by what the sum of floats is off, less than 2^-18; what lies 750 T below the largest score has no mass in any case
        const float t = (float)(1.0 / l.inv_t);
        float down = -750.f * t;
        if (by_share) down = logf((float)l.min_p) * t;
        else if (exact && told) down = logf((float)((1 - l.top_p) * all / a.k)) * t;
        low = __fadd_rn(top, down) - ((fabsf(down) + 5.f * t + fabsf(top)) * 2e-6f + 1e-44f);
        if (l.greedy) low = top;
        if (!(low <= top)) low = minus_inf();
        low = fmaxf(low, -FLT_MAX);
        const float base = low;
        if (by_count && guess <= top) low = fmaxf(low, guess);
        auto mark = [&](float border) {
            reach = 0;
            int bit = 0;
            each([&](float x, int) {
                reach |= x >= border ? 1u << bit : 0u;
                ++bit;
            });
        };
        mark(low);
        count = __popc(reach);
        if (exact) {
            total(sum, f0, f1, count);
        } else {
            each([&](float x, int) { all += weight_of(x); });
            total(all, f0, f1, count);
        }
        if (l.greedy) all = 1.0;
        if (by_count && count < top_k && low > base) {   // (groups without a score: the guess was too high)
            low = base;
            mark(low);
            count = __popc(reach);
            total(sum, f0, f1, count);
        }
        float high = top;
        const bool narrowing = by_count ? top_k <= LONG_LIST : by_mass && !by_share && told;
        // top_p alone: masses by floats, each off by less than 2^-18 (chains of up to 16), tell what certainly reaches the target and what certainly does not
        const double enough = l.top_p * all * (1 + 2e-5), short_of = l.top_p * all * (1 - 2e-5);
        int above = 0;   // scores larger than `high`, which are left in any case
        bool first = !by_count && guess > low && guess < top, moved = false;
        // An entry of the list is compared with all others: one block alone narrows on for less than that, a cluster, whose blocks wait for one another
        // every time, not as far.  At 160 and at 512 (us): one block, 1 x 2000 with top_p 0.9 29 and 38, 32 x 4000 42 and 40; clusters, 256 x 131072 with
        // top_k 50 198 and 195, top_p 0.9 742 and 720, 333 x 50021 with top_p 0.95 634 and 606.
        const int want = max(C == 1 ? 160 : 512, by_count ? top_k : 0);
        while (narrowing && count - above > want && low < high) {
            const float mid = first ? guess : middle(low, high);
            first = false;
            float up = -minus_inf(), below = minus_inf();
            int c = 0;
            sum = 0;
#pragma unroll
            for (int u = 0; u < P; ++u) {
                if (!__any_sync(0xffffffffu, reach >> (u * V) & ((1ull << V) - 1))) continue;   // (nothing from the border on)
                float part = 0;
                each_of(u, [&](float x, int) {
                    if (x >= mid) {
                        ++c;
                        up = fminf(up, x);
                        if (!by_count) part += rough(x);
                    } else if (x >= low) {
                        below = fmaxf(below, x);
                    }
                });
                sum += (double)part;
            }
            total(sum, up, below, c);
            if (by_count ? c >= top_k : sum >= enough) { low = up; count = c; moved = true; }
            else if (below > minus_inf() && (by_count || sum < short_of)) {
                high = below;
                if (!by_count) above = c;
            } else break;
        }
        // whole: all that can be left stands in the list; part: so does the border, and what is larger is left
        const bool whole = count <= LONG_LIST, part = !whole && narrowing && !by_count && count - above <= LONG_LIST;
        listed = whole;
        if (whole) above = 0;
        if (whole || part) {
            double base = 0;
            if (!part) high = top;
            if (exact) {   // now by doubles: the whole mass, and that of what is larger
                all = 0;
                each([&](float x, int) {
                    const double w = weight_of(x);
                    all += w;
                    if (x > high) base += w;
                });
                count_of_row = 0;
                total(all, f0, f1, count_of_row);
            }
            auto inside = [&](float x) { return x >= low && x <= high; };
            if (moved || part) {
                reach = 0;
                int bit = 0;
                each([&](float x, int) {
                    reach |= inside(x) ? 1u << bit : 0u;
                    ++bit;
                });
            }
            // into the first block's list, in class order
            auto bits = [&](int u) { return (unsigned)(reach >> (u * V) & ((1ull << V) - 1)); };
            int mine = __popc(reach);
#pragma unroll
            for (int u = 0; u < P; ++u) {
                const int s = __reduce_add_sync(0xffffffffu, __popc(bits(u)));
                if (lane == 0) sh.segment_count[u * W + warp] = s;
            }
            total(base, f0, f1, mine);
            prefix(sh.segment_count);
            LongRow<W, S> *to = C > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
#pragma unroll
            for (int u = 0; u < P; ++u) {
                const int c = __popc(bits(u));
                if (!__any_sync(0xffffffffu, c)) continue;
                int upto = c;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                int place = front_count + sh.segment_count[u * W + warp] + upto - c;
                each_of(u, [&](float x, int k) {
                    if (inside(x)) { to->key[place] = plain_key(x); to->k[place] = lo + k; ++place; }
                });
            }
            if (C > 1) cluster.sync();
            else __syncthreads();
            if (rank == 0) {
                const int size = count - above;
                mass = settle_list(sh, weight, top, size, l.min_p, top_k, by_mass, by_count || by_share, l.top_p, all, base, part);
                if (part && tid < C) {   // the border, for all blocks
                    LongRow<W, S> *o = C > 1 ? cluster.map_shared_rank(&sh, tid) : &sh;
                    o->tie_score = sh.at; o->tie = sh.last;
                }
                count = size;
            } else if (whole) {
                return;
            }
            if (part) {
                if (C > 1) cluster.sync();
                else __syncthreads();
                at = sh.tie_score; last = sh.tie;
                mass = segments();
            }
        } else {
            // over all scores
            if (by_share) {
                float lightest = -minus_inf();
                each([&](float x, int) {
                    if (x >= low && weight_of(x) >= l.min_p) lightest = fminf(lightest, x);
                });
                count = 0;
                total(sum, lightest, f1, count);
                at = lightest;
            } else {
                each([&](float x, int) { at = fminf(x > minus_inf() ? x : -minus_inf(), at == minus_inf() ? -minus_inf() : at); });
                count = 0;
                total(sum, at, f1, count);
            }
            auto together = [&](double &s, float &up, float &below) {
                int c = 0;
                total(s, up, below, c);
            };
            // the first r of the scores that equal `at`
            auto cut_ties = [&](int r) {
                int mine = 0;
#pragma unroll
                for (int u = 0; u < P; ++u) {
                    int c = 0;
                    each_of(u, [&](float x, int k) { c += x == at && lo + k <= last; });
                    mine += c;
                    const int s = __reduce_add_sync(0xffffffffu, c);
                    if (lane == 0) sh.segment_count[u * W + warp] = s;
                }
                total(sum, f0, f1, mine);
                prefix(sh.segment_count);
#pragma unroll
                for (int u = 0; u < P; ++u) {
                    int c = 0;
                    each_of(u, [&](float x, int k) { c += x == at && lo + k <= last; });
                    int upto = c;
#pragma unroll
                    for (int o = 1; o < 32; o *= 2) {
                        const int v = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += v;
                    }
                    int seen = front_count + sh.segment_count[u * W + warp] + upto - c;
                    each_of(u, [&](float x, int k) {
                        if (x == at && lo + k <= last && ++seen == r)
                            for (int b = 0; b < C; ++b) (C > 1 ? cluster.map_shared_rank(&sh, b) : &sh)->tie = lo + k;
                    });
                }
                if (C > 1) cluster.sync();
                else __syncthreads();
                last = sh.tie;
            };
            auto measured = [&](bool masses) {
                return [&, masses](auto &&f) {
                    each([&](float x, int k) {
                        if (left(x, k)) f(x, masses ? weight_of(x) : 1.0);
                    });
                };
            };
            auto settle = [&](bool masses, double target) {
                const float found = reached(true, target, at, top, measured(masses), together);
                double above = 0;
                int ties = 0;
                measured(masses)([&](float x, double m) {
                    if (x > found) above += m;
                    ties += x == found;
                });
                total(above, f0, f1, ties);
                const int r = masses ? ties_left(target, above, weight_of(found), ties) : (int)(target - above);
                if (found > at) { at = found; last = a.k; }
                if (r < ties) cut_ties(r);
            };
            if (by_count) {
                count = 0;
                each([&](float x, int k) { count += left(x, k); });
                total(sum, f0, f1, count);
                if (top_k < count) settle(false, (double)top_k);
            }
            if (by_mass) {
                sum = 0;
                measured(true)([&](float, double m) { sum += m; });
                count = 0;
                total(sum, f0, f1, count);
                if (exact) all = sum;
                settle(true, l.top_p * sum);
            }
            mass = segments();
        }
    } else {
        mass = all = segments();
    }
    auto put = [&](long long i, int cls, float score, double log_mass, double log_all) {
        const double lw = ((double)score - (double)top) * l.inv_t;
        put_draw(a, i, cls, (float)(lw - log_mass), (float)(lw - log_all));
    };
    if (!listed) {
        // this block's draws: those that fall into [front, front + its mass), and where nothing is left behind it also what rounding leaves there
        const double log_mass = log(mass), log_all = log(all), own_end = front + sh.slot_sum[turn ^ 1];   // (the last total was of the masses)
        bool behind = false;
        for (int b = rank + 1; b < C; ++b) behind |= cluster.map_shared_rank(&sh, b)->slot_sum[turn ^ 1] > 0;
        const bool some = own_end > front;
        for (int d = warp; d < a.draws; d += W) {
            const long long i = n * a.draws + d;
            const double target = uniform_of(a, i) * mass;
            if (!(some && front <= target && (own_end > target || !behind))) continue;
            // the last segment that begins at or before the target; the one in front of it (or behind) where it is empty
            int from = 0, to = S;
            while (to - from > 1) {
                const int mid = (from + to) / 2;
                if (front + sh.segment[mid] <= target) from = mid;
                else to = mid;
            }
            while (from > 0 && !sh.segment_count[from]) --from;
            while (from < S - 1 && !sh.segment_count[from]) ++from;
            const int cell = ((from / W) * TH + (from % W) * 32 + lane) * V;
            float x[V];
            double w[V], own = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x[j] = cell < cells ? in(n, lo + cell + j) : minus_inf();
                w[j] = left(x[j], cell + j) ? weight_of(x[j]) : 0.0;
                own += w[j];
            }
            double upto = own;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            double before = front + sh.segment[from] + (upto - own);
            const unsigned has = __ballot_sync(0xffffffffu, own > 0), hit = __ballot_sync(0xffffffffu, own > 0 && before + own > target);
            const int src = hit ? __ffs(hit) - 1 : 31 - __clz(has);
            if (lane == src) {
                int cls = 0;
                float s = 0;
                bool found = false;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (!found && w[j] > 0) {
                        before += w[j];
                        cls = lo + cell + j;
                        s = x[j];
                        found = before > target;
                    }
                put(i, cls, s, log_mass, log_all);
            }
        }
        if (C > 1) cluster.sync();   // (others look at this block's sums)
        return;
    }
    const int size = count;
    for (int d = tid; d < a.draws; d += TH) {
        const long long i = n * a.draws + d;
        const double target = uniform_of(a, i) * mass;
        int from = 0, to = size - 1;   // the first entry beyond the target, or the last that is left
        while (from < to) {
            const int mid = (from + to) / 2;
            if (sh.upto[mid] > target || sh.upto[mid] >= mass) to = mid;
            else from = mid + 1;
        }
        while (from > 0 && !(sh.w[from] > 0)) --from;   // (prefix sums by different threads are not rounded alike)
        put(i, sh.k[from], key_score(sh.key[from]), log(mass), log(all));
    }
}
}  // namespace

// false: no cluster holds the row
template <typename T> bool sample_long(const SampleArgs &a, cudaStream_t stream) {
    const Scores<T> in = scores_of<T>(a.in);
    const bool even = a.k % Pack<T>::V == 0 && on_16(in.p, in.row, sizeof(T));
    bool done = false;
    // the smallest blocks that hold a row in a cluster of up to 8
    auto go = [&](auto th, auto p, auto ev) {
        constexpr bool EVEN = decltype(ev)::value;
        constexpr int TH = decltype(th)::value, P = decltype(p)::value;
        const int c = (a.k + Hold<T, TH, P, EVEN>::CELLS - 1) / Hold<T, TH, P, EVEN>::CELLS;
        if (done || c > LONG_CLUSTER) return;
        launch_long(k_sample_long<T, TH, P, EVEN>, a.n, c, TH, stream, 0, a, in);
        done = true;
    };
    using std::integral_constant;
    auto all = [&](auto ev) {
        constexpr int S = decltype(ev)::value ? sizeof(T) == 2 ? 1 : 2 : 8;   // 8 scores
        if (a.k <= 2048) go(integral_constant<int, 256>{}, integral_constant<int, S>{}, ev);
        go(integral_constant<int, 512>{}, integral_constant<int, S>{}, ev);
        go(integral_constant<int, 512>{}, integral_constant<int, 2 * S>{}, ev);
        go(integral_constant<int, 512>{}, integral_constant<int, 4 * S>{}, ev);
    };
    even ? all(std::true_type{}) : all(std::false_type{});
    return done;
}

}  // namespace tgbm
