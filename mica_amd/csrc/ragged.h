// Sequences of different lengths packed one behind the other: rows starts[b] .. starts[b + 1] - 1 of T are sequence b's.
#pragma once

#include "common.h"

// starts: int32 [B + 1] in device memory, which nothing on the host has seen: every value is clamped, so that whatever it
// holds no row outside 0 .. T - 1 is touched.
struct Ragged {
    const int *starts;
    int B, T;
    MICA_DEVICE int at(int b) const { return min(max(starts[b], 0), T); }
    MICA_DEVICE int rows(int b) const { return max(at(b + 1) - at(b), 0); }
};

// a wave's running sums
MICA_DEVICE int wave_scan(int x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d, 64);
        x += (int)(threadIdx.x & 63) >= d ? y : 0;
    }
    return x;
}

// Sequence b has units(b) units of work.  The sequence and the unit at place `at` in the row of all sequences' units; false
// where there are fewer (b is then their number).  All lanes of a wave call and get the same; a lane reads every 64th
// sequence's lengths.  (In two levels, a lane 1 / 64 of the sequences at first: 1000 prompts of up to 60 tokens 199 -> 179 us, 400
// and 256 the same, 128 of 512 tokens 483 -> 491.)
template <class F>
MICA_DEVICE bool find_unit(int B, F units, int at, int &b, int &u) {
    int before = 0;
    for (int base = 0; base < B; base += 64) {
        const int i = base + (int)(threadIdx.x & 63);
        const int x = i < B ? units(i) : 0, sum = wave_scan(x);
        const unsigned long long past = __builtin_amdgcn_ballot_w64(before + sum > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            b = base + l;
            // (starts that are no running sum may wrap these round: the unit stays one of the sequence's)
            u = min(max(at - before - __builtin_amdgcn_readlane(sum - x, l), 0), __builtin_amdgcn_readlane(x, l) - 1);
            return u >= 0;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    b = before;
    return false;
}
