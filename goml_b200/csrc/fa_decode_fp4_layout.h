// fa_decode_fp4_layout.h — how fa_decode_fp4 divides the keys: teams, plans, and the choice between them.  Plain C++: no GPU is needed to ask what a call would do.
#pragma once
#include <math.h>

#include <algorithm>

#ifdef __CUDACC__
#define FP4_HOST_DEVICE __host__ __device__
#else
#define FP4_HOST_DEVICE
#endif

namespace fa_fp4 {

constexpr int CHUNK = 64;        // keys per unit of work (page sizes are multiples of it)
constexpr int THREADS = 128;
constexpr int WARPS = THREADS / 32;
// What a pair costs beyond its chunks, in chunks: on the line it takes so many units more, ahead of its first chunk.  A long one costs its sum and its queries (about 5 of a CTA's
// chunks of 1.1k clocks); one of a single key is a chain of latencies of 7 to 11k clocks.
constexpr int PAIR_LEAST = 12, PAIR_MORE = 5, PAIR_LEAST_ALONE = 2, PAIR_MORE_ALONE = 1;
template <bool ALONE>
FP4_HOST_DEVICE constexpr int pair_cost(int chunks) {
    const int least = ALONE ? PAIR_LEAST_ALONE : PAIR_LEAST, more = ALONE ? PAIR_MORE_ALONE : PAIR_MORE;
    return more > least - chunks ? more : least - chunks;
}
constexpr int ctas_per_sm(int nq) { return nq == 1 ? 3 : 2; }

// Plans.
//  PAIR:  a team to a pair: no search, no cuts.
//  LINE:  the chunks of all pairs form one line that is cut into equal pieces, one per resident team, so sequences of very different
//         lengths load all SMs alike.
enum Plan : int { PAIR, LINE };

struct Layout {
    int plan, grid, rows;
    bool alone;
    int pieces() const { return grid * (alone ? WARPS : 1); }
    int sums() const { return 2 * (pieces() / 8 + 1); }   // of eight teams' pieces
    int slots() const { return 2 * pieces() + sums(); }
};
// Teams and plan: what costs least by an estimate, in units of a warp's time for a chunk on a full SM (2.6 us for head dim 128), at lengths of all that the cache has room for, of which the line, which
// shares the keys there are, is expected to see 0.8.  Cutting pairs and adding their pieces up makes the line dear, a last round with few teams and unequal lengths whole pairs.
// The constants are from 300 shapes of 8 to 4096 pairs of 64 to 8000 keys, all of one length and drawn from zero on; the choice is 2 % off the best of the four on
// the mean.  us, CTAs on the line / a pair each / warps on the line / a pair each, 4 query heads to a kv head of 128: 8 pairs of 4096 keys 10.8 / 22.6 / 16 / 79.8, 288 pairs of 512 keys 15.1 / 7.63 / 15.2 / 14.1,
// 288 pairs of 4096 keys 40.7 / 35.3 / 42.5 / 82.1, 592 pairs of 256 keys 12.2 / 10.5 / 15.2 / 9.57, 960 pairs of 512 keys 27.5 / 23.6 / 27.8 / 21.1,
// 960 pairs of 4096 keys 105 / 104 / 106 / 122, 1184 pairs of 1024 keys 46 / 41.9 / 46.7 / 36.6.
struct Estimate {
    double pairs, resident;   // CTAs of all SMs
    int nq, group, per_sm;
    double unit() const { return 2.0 / per_sm; }   // of what does not take longer where more CTAs share an SM
    double line(bool alone, double chunks) const {
        const double units = pairs * (alone ? chunks + pair_cost<true>((int)chunks) + 1.8 * nq : chunks + pair_cost<false>((int)chunks));
        return unit() * (alone ? 1.5 + 1.3 * std::min(group, 4) : 6) + units / (WARPS * resident);
    }
    double whole_pairs(bool alone, int steps) const {
        const double teams = alone ? WARPS * resident : resident, full = std::floor(pairs / teams), rest = pairs - full * teams;
        const int on_sm = (int)std::ceil(rest * per_sm / teams);   // CTAs that an SM has in the last round: the fewer, the faster
        const double last = on_sm == 0 ? 0 : on_sm == per_sm ? 1 : per_sm == 2 ? 0.6 : on_sm == 1 ? 0.45 : 0.72;
        return unit() * ((alone ? 1.7 : 0.8) * nq * (full + (rest > 0)) + (alone ? 0 : 0.8)) + steps * (full + last);
    }
};
// rows: of the whole cache.  Tables are often wide enough for one sequence to have all pages; a sequence is expected to have its share of them at most, and the longest twice that.
inline Layout layout_of(int batch, int q_heads, int kv_heads, int span, long long rows, int sms) {
    Layout x;
    const int group = q_heads / kv_heads, per_sm = ctas_per_sm(group <= 8 ? 1 : 2), resident = per_sm * sms;
    x.rows = group <= 8 ? 8 : 16;
    const long long pairs = (long long)batch * kv_heads, chunks = ((long long)span + CHUNK - 1) / CHUNK;
    const Estimate e{(double)pairs, (double)resident, x.rows / 8, group, per_sm};
    const long long share = (rows / batch + CHUNK - 1) / CHUNK, longest = std::min(chunks, 2 * share);
    const double mean = std::min(0.8 * chunks, (double)share);
    const double line = e.line(false, mean), line_alone = 3 * pairs < 2 * resident ? INFINITY : e.line(true, mean);
    const double whole = e.whole_pairs(false, (int)((longest + WARPS - 1) / WARPS)), whole_alone = e.whole_pairs(true, (int)longest);
    x.alone = std::min(line_alone, whole_alone) < std::min(line, whole);
    const int teams = x.alone ? WARPS : 1;
    // a line has to have no more units than an int counts (a paged cache whose capacity is far above what it holds)
    if (pairs * (chunks + PAIR_LEAST) > 0x7fffffffLL || std::min(whole, whole_alone) <= std::min(line, line_alone)) {
        x.plan = PAIR;
        x.grid = (int)((pairs + teams - 1) / teams);
    } else {
        x.plan = LINE;
        const long long units = (pairs * chunks + teams - 1) / teams;
        x.grid = (int)(units < resident ? (units > 0 ? units : 1) : resident);
    }
    return x;
}

}  // namespace fa_fp4
