// fa_line_pieces.h — how a line of units is cut into equal pieces, one for every CTA (fa_decode_stream_sm100.cu); also for the host, so that it can be asked without a GPU.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define FA_LINE_FN __host__ __device__ __forceinline__
#else
#define FA_LINE_FN inline
#endif

namespace fa_sm100 {

// Division of lines: their numbers nearly always fit 32 bits, and of 64 a division takes some hundred instructions.
FA_LINE_FN long long quotient(long long a, long long b) { return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b; }
// equal pieces of a line, the first `r` of them one unit longer
struct Pieces {
    long long q, r;
    FA_LINE_FN Pieces(long long total, int pieces) : q(quotient(total, pieces)), r(total - q * pieces) {}
    FA_LINE_FN long long begin(int i) const { return i * q + (i < r ? i : r); }
    // the piece that holds unit u of the line
    FA_LINE_FN int piece_of(long long u) const { return (int)(u < r * (q + 1) ? quotient(u, q + 1) : r + quotient(u - r * (q + 1), q)); }
    // The pieces that the n units from u on are in: the first one, and their number.  Units that are not on the line (of lengths that have changed since it was cut) count as the nearest
    // one that is, so that the places of the pieces' states are those of CTAs that there are whatever u and n.  The line has a unit.
    struct Span {
        int first, count;
    };
    FA_LINE_FN Span pieces_of(long long u, long long n, int pieces) const {
        const long long last = q * pieces + r - 1, from = u < 0 ? 0 : u < last ? u : last, to = n < 1 ? from : from + n - 1 < last ? from + n - 1 : last;
        Span s;
        s.first = piece_of(from);
        s.count = piece_of(to) - s.first + 1;
        return s;
    }
};

}  // namespace fa_sm100
