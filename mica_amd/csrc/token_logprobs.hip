// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits, in one pass over them.
//
//   M = max_v x_v,  S = sum_v e^(x_v - M),  lp(v) = (x_v - M) - ln S,  H = ln S - (sum_v e^(x_v - M) (x_v - M)) / S
//   top: the `top` largest by (value, then lowest index); NaN counts as the largest value, -0 equals 0
//
// (in log2 units, see Stat).  A workgroup walks a row's (or a part's) logits in blocks of 256 threads (a
// short row's: 64) x 64 bytes, the next block's loads in flight while it works on one.  Every thread keeps a running (m, s, t) of its own elements in fp32, so
// the statistics need no barrier.  For the alternatives the workgroup keeps a list of candidates in LDS and a threshold, of
// which it knows that `top` elements reach it: at first the top-th largest of 64 group maxima of the first block (found bit
// by bit with ballots), later the top-th largest candidate.  The 16-byte vectors whose maximum reaches it go into a queue
// whole; when 32 of them wait, their elements are looked at, four threads a vector, and the best of the list found anew
// (with the elements looked at where they were found, a wave took 400 cycles for each, and 2048 x 151936 bf16 with 20
// alternatives 157 us instead of 135).  A block of which too many vectors reach the threshold (long runs of ties) is
// selected exactly, bit by bit over values and then indices.
//
// Few rows are divided over several workgroups each; lp_merge_kernel then joins their (m, s, t) and candidates.
#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;
constexpr int U = 4;                   // 16-byte vectors a thread holds of a block
template <int NT> constexpr int kCap = 4 * NT; // candidates in LDS, of a workgroup of NT threads
template <int NT> constexpr int kQueue = NT > 64 ? NT : 128; // vectors in LDS that hold an element that reaches the threshold
constexpr int kFlush = 32;             // as many wait for the next look at their elements
constexpr int kMaxParts = 64;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr float kFar = -1.0e4f;        // 2^-10000 is 0 in fp32: differences are cut here, so that 0 x inf never is
constexpr float kNear = 131072.0f;     // references up to here take one fma an element (Stat)
constexpr float kRaise = 16.0f;        // e^16 times the elements of a row is far from fp32's range

struct Stat;
struct LpParams {
    const void *x; long long ldx;      // logits [T][V], rows ldx elements apart
    const void *tok; int tok64;        // given tokens, int32 or int64 [T][C]
    int T, V, C, top;
    int parts, bpp;                    // workgroups a row, blocks each
    float *lp;                         // [T][C]
    float *ent;                        // [T]
    long long *ids;                    // [T][top]
    float *tlp;                        // [T][top]
    Stat *pm;                          // partial sums [T][parts]
    unsigned long long *pk;            // partial candidates [T][parts][top], the best first
};

// values in order as whole numbers: NaN above all, -0 as 0
MICA_DEVICE uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
MICA_DEVICE float value_of(uint32_t o) {
    return o == 0xffffffffu ? __builtin_nanf("") : __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
// larger: the larger value, then the lower index; every element of a row has a key of its own, and none is 0
MICA_DEVICE unsigned long long key_of(float v, int idx) {
    return ((unsigned long long)order_of(v) << 32) | (uint32_t)~idx;
}

template <int DT> struct Elem; // the logits' type: elements in 16 bytes, the bits of order_of() that a threshold is found to
template <> struct Elem<MICA_BF16> {
    static constexpr int N = 8, kBits = 16;
    static MICA_DEVICE float get(const u32x4 &w, int e) { return (e & 1) ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]); }
    static MICA_DEVICE float load(const void *p, long long i) { return bf16_to_f32(((const uint16_t *)p)[i]); }
    static constexpr uint32_t kLow = 0xff80ff80u; // -inf
};
template <> struct Elem<MICA_FP16> {
    static constexpr int N = 8, kBits = 19;
    static MICA_DEVICE float get(const u32x4 &w, int e) { return f16_to_f32((uint16_t)(w[e >> 1] >> (16 * (e & 1)))); }
    static MICA_DEVICE float load(const void *p, long long i) { return f16_to_f32(((const uint16_t *)p)[i]); }
    static constexpr uint32_t kLow = 0xfc00fc00u;
};
template <> struct Elem<MICA_FP32> {
    static constexpr int N = 4, kBits = 19;
    static MICA_DEVICE float get(const u32x4 &w, int e) { return __uint_as_float(w[e]); }
    static MICA_DEVICE float load(const void *p, long long i) { return ((const float *)p)[i]; }
    static constexpr uint32_t kLow = 0xff800000u;
};

// s = sum 2^y, t = sum 2^y y over elements y = (x - m) log2(e) + r.  m is the reference, at the end the largest element, and
// -inf before the first; with c = m log2(e) rounded and r = m log2(e) - c (exact), y is one fma of x, fma(x, log2(e), -c).  Where |m| is so large
// that r would count (kNear), r is 0 and y takes the difference first.
struct Stat {
    float m, r, s, t;
    MICA_DEVICE static float rest(float m) { return __builtin_fabsf(m) <= kNear ? __builtin_fmaf(m, kLog2e, -(m * kLog2e)) : 0.0f; }
    MICA_DEVICE void rebase(float to) { // to >= m
        const float r2 = rest(to);
        // (also for m = to = -inf, whose difference is NaN)
        const float d = __builtin_fmaxf(__builtin_fmaf(m - to, kLog2e, r2 - r), kFar);
        const float f = __builtin_amdgcn_exp2f(d);
        t = f * __builtin_fmaf(s, d, t);
        s *= f;
        m = to, r = r2;
    }
    MICA_DEVICE void add(float y) {
        const float e = __builtin_amdgcn_exp2f(y);
        s += e;
        t = __builtin_fmaf(e, __builtin_fmaxf(y, kFar), t);
    }
    MICA_DEVICE float y_of(float x) const { return __builtin_fmaf(x - (m == -__builtin_inff() ? 0.0f : m), kLog2e, r); }
    // ln S, S = sum e^(x - m): not below 0, and 0 where one element alone has a weight (its own 2^r divided by 2^r)
    MICA_DEVICE float ln_sum() const {
        const float q = s / __builtin_amdgcn_exp2f(r);
        return q < 1.0f ? 0.0f : logf(q);
    }
    MICA_DEVICE float logprob(float x) const { return (x - m) - ln_sum(); }
    MICA_DEVICE float entropy() const { // (t and r s round alike where one element alone has a weight)
        const float h = ln_sum() - (t - r * s) / s * kLn2;
        return h < 0.0f ? 0.0f : h;
    }
};
constexpr Stat kNone = {-__builtin_inff(), 0.0f, 0.0f, 0.0f};

// the order number of the n-th largest of 64 lanes' values, bit by bit from the top; lower bits than BITS are 0
template <int BITS>
MICA_DEVICE uint32_t nth_of_wave(uint32_t o, int n) {
    uint32_t at = 0;
#pragma unroll
    for (int b = 31; b > 31 - BITS; --b) {
        const uint32_t c = at | (1u << b);
        if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(o >= c)) >= n) at = c;
    }
    return at;
}

// The best `top` of the list's n keys, in order, at its start (n <= kCap; every thread calls).  Returns how many.
// QUADS: up to 64 keys take four threads each (64 x 151936 fp32 21.9 -> 20.3 us; the 16-bit rows' kernel would spill for it,
// 8192 x 16000 with 5 alternatives 66.4 -> 71.1).
template <bool QUADS, int NT>
MICA_DEVICE int keep_best(unsigned long long *list, int n, int top) {
    if (QUADS && n <= NT / 4) { // four threads a key
        const int at = threadIdx.x >> 2;
        const unsigned long long k = at < n ? list[at] : 0;
        int r = 0;
        for (int i = threadIdx.x & 3; i < n; i += 16)
#pragma unroll
            for (int x = 0; x < 16; x += 4) r += list[i + x] > k && i + x < n;
        r += __shfl_xor(r, 1, 64);
        r += __shfl_xor(r, 2, 64);
        __syncthreads();
        if (at < n && (threadIdx.x & 3) == 0 && r < top) list[r] = k;
        __syncthreads();
        return n < top ? n : top;
    }
    unsigned long long mine[kCap<NT> / NT];
    int rank[kCap<NT> / NT];
#pragma unroll
    for (int j = 0; j < kCap<NT> / NT; ++j) {
        const int at = threadIdx.x + j * NT;
        rank[j] = kCap<NT>;
        if (j * NT < n && at < n) {
            const unsigned long long k = list[at];
            int r = 0;
            for (int i = 0; i < n; i += 8) // 8 reads at a time; those past n do not count
#pragma unroll
                for (int x = 0; x < 8; ++x) r += list[i + x] > k && i + x < n;
            mine[j] = k, rank[j] = r;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kCap<NT> / NT; ++j)
        if (rank[j] < top) list[rank[j]] = mine[j];
    __syncthreads();
    return n < top ? n : top;
}

// the logit of a row's given token c; NaN for an id that is no token (no access)
template <int DT>
MICA_DEVICE float given(const LpParams &p, int row, int c) {
    const long long at = (long long)row * p.C + c;
    const long long id = p.tok64 ? ((const long long *)p.tok)[at] : ((const int *)p.tok)[at];
    const void *x = (const char *)p.x + (long long)row * p.ldx * (DT == MICA_FP32 ? 4 : 2);
    return id >= 0 && id < p.V ? Elem<DT>::load(x, id) : __builtin_nanf("");
}

// the results of a row from its whole statistics; every thread of a workgroup calls, with its given() logit c = threadIdx.x
template <int DT, int NT>
MICA_DEVICE void finish(const LpParams &p, int row, const Stat &a, const unsigned long long *best, float tok) {
    for (int c = threadIdx.x; c < p.C; c += NT) {
        if (c >= NT) tok = given<DT>(p, row, c);
        p.lp[(long long)row * p.C + c] = a.logprob(tok);
    }
    if (threadIdx.x == 0) p.ent[row] = a.entropy();
    if ((int)threadIdx.x < p.top) {
        const unsigned long long k = best[threadIdx.x];
        const long long at = (long long)row * p.top + threadIdx.x;
        p.ids[at] = (long long)(uint32_t)~(uint32_t)k;
        p.tlp[at] = a.logprob(value_of((uint32_t)(k >> 32)));
    }
}

// one (m, s, t) of the workgroup's NT; every thread gets it
template <int NT>
MICA_DEVICE Stat block_stat(Stat a, Stat *red) {
    a.rebase(wave_max(a.m));
    a.s = wave_sum(a.s), a.t = wave_sum(a.t);
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = a;
    __syncthreads();
    float m = red[0].m;
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) m = __builtin_fmaxf(m, red[w].m);
    Stat r = {m, Stat::rest(m), 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        Stat b = red[w];
        b.rebase(m);
        r.s += b.s, r.t += b.t;
    }
    return r;
}

// One pass over the row, bound by HBM without alternatives: 4096 x 151936 bf16 take 197 us, 6.3 TB/s; with 20 of them nearly
// as much by VALU issue, 2048 rows 130 us, 4.8 TB/s (calls one behind the other: a call by itself takes 147 to 160).  Rows
// of a block or two are bound by their latency (load, threshold, candidates, join): 64 x 151936 fp32 with 20 alternatives
// 19.3 us, without 12; one row 11.  Rows of which nearly everything is -inf are slower: lanes that have seen nothing else
// send their wave through the loop of single elements, and with fewer than `top` groups of the first block that hold a
// finite element the exact selection runs: 30 finite elements of 151936, 20 alternatives, one row 102 us, 2048 rows 447 (139
// without alternatives); 3000 finite ones 12.5 and 148.
// (six workgroups a CU; five leave fp32 the registers that it would spill: 1024 x 151936 with 20 alternatives 117.5 -> 107.9 us)
template <int DT, bool TOP, int NT>
__global__ __launch_bounds__(NT, DT == MICA_FP32 ? 5 : 6) void lp_rows_kernel(LpParams p) {
    using E = Elem<DT>;
    constexpr int kSize = 16 / E::N;
    __shared__ Stat red[NT / 64];
    __shared__ float gmax[NT / 2];
    __shared__ unsigned long long list[TOP ? kCap<NT> : 8];
    __shared__ u32x4 queue[TOP ? kQueue<NT> : 1];
    __shared__ int queue_at[TOP ? kQueue<NT> : 1];
    __shared__ int counts[3], listed, wcount[NT / 64];
    const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts, tid = threadIdx.x;
    const char *x = (const char *)p.x + (long long)row * p.ldx * kSize;
    // the row as up to N - 1 single elements, 16-byte vectors from the first aligned address, up to N - 1 single ones
    const int head = min((int)((0 - (uintptr_t)x) & 15) / kSize, p.V), nv = (p.V - head) / E::N;
    const int tail = p.V - head - nv * E::N;
    const char *body = x + head * kSize;
    const int v0 = part * p.bpp * (NT * U), v1 = min(v0 + p.bpp * (NT * U), nv);
    const bool first_part = part == 0, last_part = part == p.parts - 1;
    if (TOP && tid == 0) counts[0] = listed = 0;

    auto load = [&](int v, u32x4 (&w)[U]) {
        if (v + NT * U <= v1) { // a full block
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = __builtin_nontemporal_load((const u32x4 *)(body + (v + u * NT + tid) * 16ll));
            return;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = v + u * NT + tid;
            w[u] = u32x4{E::kLow, E::kLow, E::kLow, E::kLow};
            if (at < v1) w[u] = __builtin_nontemporal_load((const u32x4 *)(body + at * 16ll));
        }
    };
    u32x4 cur[U], nxt[U];
    load(v0, cur);
    // a single element a thread: the head's in the first part, the tail's in the last
    float one = -__builtin_inff();
    int one_at = -1;
    if (first_part && tid < head) one_at = tid;
    if (last_part && tid >= 8 && tid < 8 + tail) one_at = p.V - tail + tid - 8;
    if (one_at >= 0) one = E::load(x, one_at);
    const float tok = p.parts == 1 && tid < p.C ? given<DT>(p, row, tid) : 0.0f;

    Stat a = kNone;
    float largest = -__builtin_inff();
    bool near = false; // every lane's reference is within kNear
    float thr = -__builtin_inff(); // elements not below it are candidates;
    bool above = false;            // or only those above it
    int kept = 0, queued = 0;      // candidates; vectors of earlier blocks in the queue
    int turn = 0;                  // the block's counter
    for (int v = v0; v == v0 || v < v1; v += NT * U) {
        const bool first = v == v0;
        if (v + NT * U < v1) load(v + NT * U, nxt);
        float vmax[U], mx = first ? one : -__builtin_inff(); // the largest of each vector, of the thread's elements
        // the reference of the sums follows the maximum when a lane's exceeds it by kRaise (with the maximum itself a wave
        // would rebase at most of its vectors, half a row's elements later still)
        auto raise = [&](float m) {
            if (__builtin_amdgcn_ballot_w64(m > a.m + kRaise)) {
                a.rebase(__builtin_fmaxf(a.m, m));
                near = __builtin_amdgcn_ballot_w64(__builtin_fabsf(a.m) > kNear) == 0;
            }
        };
        if (first) {
            raise(one);
            a.add(a.y_of(one));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vmax[u] = E::get(cur[u], 0);
#pragma unroll
            for (int e = 1; e < E::N; ++e) vmax[u] = __builtin_fmaxf(vmax[u], E::get(cur[u], e));
            mx = __builtin_fmaxf(mx, vmax[u]);
            raise(vmax[u]);
            if (near) {
                const float c = -(a.m * kLog2e);
#pragma unroll
                for (int e = 0; e < E::N; ++e) a.add(__builtin_fmaf(E::get(cur[u], e), kLog2e, c));
            } else { // (or a thread is without any element of its own yet)
#pragma unroll 1
                for (int e = 0; e < E::N; ++e) a.add(a.y_of(E::get(cur[u], e)));
            }
            __asm__ volatile("" : "+v"(a.s), "+v"(a.t)); // the sums here: left alone they follow all the exponentials
        }
        largest = __builtin_fmaxf(largest, mx);
        // keeps what the compiler makes of the elements (their unpacked values, their order numbers) from staying in
        // registers from one use to the next
        auto forget = [&] {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) __asm__ volatile("" : "+v"(cur[u][i]));
        };
        if constexpr (TOP) {
            forget();
            if (first) {
                // groups of lanes l and l + 32 of two waves: a short row fills as many as it has vectors (of four lanes side by
                // side, 300 elements filled 10, and everything was a candidate: 8192 rows with 20 alternatives 155 us, not 54)
                float g = mx;
                if constexpr (NT > 64) {
                    g = __builtin_fmaxf(g, __shfl_xor(g, 32, 64));
                    if ((tid & 32) == 0) gmax[(tid >> 6) * 32 + (tid & 31)] = g;
                    __syncthreads();
                    g = __builtin_fmaxf(gmax[tid & 63], gmax[64 + (tid & 63)]);
                } else {
                    __syncthreads(); // the counters' first values
                }
                thr = value_of(nth_of_wave<E::kBits>(order_of(g), p.top));
                if (thr != thr) thr = -__builtin_inff(); // (the number below -inf's is a NaN's)
            }
            auto reaches = [&](float xv) { return above ? !(xv <= thr) : !(xv < thr); }; // (as a NaN does)
            const bool more = v + NT * U < v1;
            auto push = [&](float xv, int idx) { list[atomicAdd(&listed, 1)] = key_of(xv, idx); };
            auto best = [&] { // the best of the list, and their threshold
                const bool full = kept >= p.top;
                kept = keep_best<DT == MICA_FP32, NT>(list, kept, p.top);
                if (full) {
                    const unsigned long long least = list[p.top - 1];
                    thr = value_of((uint32_t)(least >> 32));
                    if (thr != thr) thr = __builtin_inff();
                    // indices grow from block to block, but for the single elements of the row's end
                    above = (int)~(uint32_t)least < p.V - tail;
                }
                if (tid == 0) listed = kept;
                __syncthreads();
            };
            // the elements of the queue's first n vectors, four threads a vector, 64 vectors at a time
            auto expand = [&](int n) {
                kept = listed; // (with n = 0 the single elements)
                for (int q = 0; q < n; q += NT / 4) {
                    const int i = q + (tid >> 2);
                    if (i < n) {
                        const u32x4 w = queue[i];
                        const uint32_t word = (tid & 2) ? ((tid & 1) ? w[3] : w[2]) : ((tid & 1) ? w[1] : w[0]);
#pragma unroll
                        for (int e = 0; e < E::N / 4; ++e) {
                            const float xv = E::get(u32x4{word, 0, 0, 0}, e);
                            // (not below, also where `above`: that is for the blocks to come)
                            if (!(xv < thr)) push(xv, head + queue_at[i] * E::N + (tid & 3) * (E::N / 4) + e);
                        }
                    }
                    __syncthreads();
                    kept = listed;
                    if (q + NT / 4 < n || (more && kept > p.top + 16)) best();
                }
            };
            // Three counters in turn, so that one barrier a block is enough: the next block's is cleared here, before the
            // barrier, two blocks after its last reads.
            const int next = turn == 2 ? 0 : turn + 1;
            if (tid == 0) counts[next] = 0;
            // (the maxima pass over NaNs: a thread that has seen one looks at all its elements from then on)
            const bool odd = a.s != a.s;
            if (__builtin_amdgcn_ballot_w64(reaches(mx) || odd)) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int at = v + u * NT + tid;
                    if ((reaches(vmax[u]) || odd) && at < v1) { // (a queue that is full is only counted)
                        const int to = queued + atomicAdd(&counts[turn], 1);
                        if (to < kQueue<NT>) queue[to] = cur[u], queue_at[to] = at;
                    }
                }
                if (first && one_at >= 0 && reaches(one)) push(one, one_at);
            }
            __syncthreads();
            const int n = queued + counts[turn];
            const bool exact = n > kQueue<NT>;
            if (exact || n > kFlush || !more) {
                expand(exact ? queued : n);
                queued = 0;
            } else {
                queued = n;
            }
            if (exact) { // too many reach the threshold: the best of this block's vectors, exactly
                // the value of the top-th best element, then the index up to which elements of that value belong; the
                // block is read again for every bit (a loop of few registers beside the ordinary path's)
                auto each = [&](auto f) {
#pragma unroll 1
                    for (int u = 0; u < U; ++u) {
                        const int at = v + u * NT + tid;
                        if (at >= v1) break;
                        const u32x4 w = *(const u32x4 *)(body + (long long)at * 16);
#pragma unroll
                        for (int e = 0; e < E::N; ++e) f(E::get(w, e), head + at * E::N + e);
                    }
                };
                uint32_t o = 0, last = 0xffffffffu;
                auto belongs = [&](float xv, int idx) { // above order o, or at it with an index up to `last`
                    const uint32_t q = order_of(xv);
                    return q > o || (q == o && (uint32_t)idx <= last);
                };
                auto tally = [&] {
                    int c = 0;
                    each([&](float xv, int idx) { c += belongs(xv, idx); });
                    const float w = wave_sum((float)c); // (whole numbers below 2^24)
                    __syncthreads();
                    if ((tid & 63) == 0) wcount[tid >> 6] = (int)w;
                    __syncthreads();
                    int all = wcount[0];
#pragma unroll
                    for (int w = 1; w < NT / 64; ++w) all += wcount[w];
                    return all;
                };
#pragma unroll 1
                for (int b = 31; b >= 0; --b) {
                    o |= 1u << b;
                    if (tally() < p.top) o &= ~(1u << b);
                }
                last = 0xffffffffu >> __builtin_clz(p.V); // the least index that still gives `top` elements
#pragma unroll 1
                for (int b = 31 - __builtin_clz(p.V); b >= 0; --b) {
                    last &= ~(1u << b);
                    if (tally() < p.top) last |= 1u << b;
                }
                each([&](float xv, int idx) {
                    if (belongs(xv, idx)) push(xv, idx);
                });
                __syncthreads();
                kept = listed;
                if (more) best();
            }
            turn = next;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) cur[u] = nxt[u];
    }
    a.rebase(largest);
    const Stat all = block_stat<NT>(a, red);
    if constexpr (TOP) kept = keep_best<DT == MICA_FP32, NT>(list, kept, p.top);
    if (p.parts == 1) {
        finish<DT, NT>(p, row, all, list, tok);
        return;
    }
    if (tid == 0) p.pm[blockIdx.x] = all;
    if (TOP && tid < p.top) p.pk[(long long)blockIdx.x * p.top + tid] = tid < kept ? list[tid] : 0ull;
}

// The parts of a row joined: their sums by one wave's reduction, their candidates, which come best first, by a bound that
// `top` keys reach.  4 to 5 us, a launch and two loads' latency.
template <int DT>
__global__ __launch_bounds__(kThreads) void lp_merge_kernel(LpParams p) {
    __shared__ unsigned long long list[kCap<kThreads>], all[kMaxParts * kMaxTop];
    __shared__ int count;
    const int row = blockIdx.x, tid = threadIdx.x;
    Stat a = kNone;
    if ((tid & 63) < p.parts) a = p.pm[(long long)row * p.parts + (tid & 63)];
    const float tok = tid < p.C ? given<DT>(p, row, tid) : 0.0f;
    a.rebase(wave_max(a.m));
    a.s = wave_sum(a.s), a.t = wave_sum(a.t);
    if (p.top > 0) {
        const int n = p.parts * p.top;
        const unsigned long long *pk = p.pk + (long long)row * n;
        for (int i = tid; i < n; i += kThreads) all[i] = pk[i];
        if (tid == 0) count = 0;
        __syncthreads();
        // with r = top / parts rounded up, the (top / r rounded up)-th largest of the parts' r-th best: at least top keys
        // reach it
        const int r = (p.top + p.parts - 1) / p.parts, want = (p.top + r - 1) / r;
        const unsigned long long own = (tid & 63) < p.parts ? all[(tid & 63) * p.top + r - 1] : 0;
        int rank = 0;
        for (int c = 0; c < p.parts; c += 8) // 8 reads at a time (past the last part within `all`); those do not count
#pragma unroll
            for (int x = 0; x < 8; ++x) rank += all[(c + x) * p.top + r - 1] > own && c + x < p.parts;
        const unsigned long long at = __builtin_amdgcn_ballot_w64(rank == want - 1);
        unsigned long long least = 0; // (parts without that many keys)
        if (at) {
            const int l = __builtin_ctzll(at);
            least = (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(own >> 32), l) << 32 |
                    (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)own, l);
        }
        // At most top^2 keys reach it: with up to top parts there are no more; with more parts r is 1 and want is top, so
        // want - 1 parts have keys above `least`, and one more has it.
        static_assert(kMaxTop * kMaxTop <= kCap<kThreads>, "the keys that reach the bound fit the list");
        for (int i = tid; i < n; i += kThreads)
            if (all[i] >= least && all[i] != 0) list[atomicAdd(&count, 1)] = all[i];
        __syncthreads();
        keep_best<true, kThreads>(list, count, p.top);
    }
    finish<DT, kThreads>(p, row, a, list, tok);
}

// Workgroups a row, and whole blocks each: about 2048 in all, a third more than the chip holds at a time (256 CUs of six,
// fp32 five).  No more than it holds (1536, fp32 1280), rounded down, us, 2048 / those: 20 alternatives, bf16 100 x 151936
// 18.2 / 22.3, 300 37 / 33, 1000 75 / 70, fp32 300 x 151936 44 / 40; without, 300 x 151936 21.0 / 21.8, 700 41.8 / 44.5,
// 1000 56.7 / 53.2; fp16 517 x 32003 with 7 18.6 / 18.2.  Neither is better everywhere.
// A row that is short, or one of many, takes one workgroup and no join: up to 2 blocks with alternatives (which each block's
// candidates delay: 500 x 9000 bf16 with 20 16.6 -> 10.9 us, but 260 x 24000 14.4 -> 15.4), up to 4 without (260 x 24000
// 12.3 -> 8.8).
void divide(int T, int V, int elems, int top, int &parts, int &bpp) {
    const int blocks = max(1, (V / elems + kThreads * U - 1) / (kThreads * U));
    const int want = T >= 1024 || blocks <= (top ? 2 : 4) ? 1 : min((2048 + T - 1) / T, kMaxParts);
    bpp = (blocks + want - 1) / want;
    parts = (blocks + bpp - 1) / bpp;
}
long long part_bytes(int T, int parts, int top) { return parts > 1 ? (long long)T * parts * (16 + 8 * top) : 0; }

// Rows of one launch: a grid of 2^32 work-items or more wraps round without an error and leaves the rows behind it unwritten.
constexpr int kGridRows = 1 << 23;

template <int DT>
void launch(LpParams p, hipStream_t st) {
    constexpr int kSize = 16 / Elem<DT>::N;
    // A row of one block of 64 threads (two, where rows are so many that they wait for each other) takes a wave: 8192 x 300
    // bf16 with 20 alternatives 53.6 -> 23.9 us, 8192 x 4000 44.5 -> 36.1; but two blocks of 2000 x 4000 15.2 / 17.2.
    const bool wave = p.parts == 1 && p.V <= ((p.T >= 4096 ? 2 : 1) * 64 * U - 2) * Elem<DT>::N;
    if (wave) p.bpp *= kThreads / 64;
    for (int left = p.T; left > 0; left -= kGridRows) { // (rows of several parts are few)
        p.T = min(left, kGridRows);
        const dim3 grid((unsigned)(p.T * p.parts));
        if (p.top > 0 && wave) hipLaunchKernelGGL((lp_rows_kernel<DT, true, 64>), grid, dim3(64), 0, st, p);
        else if (p.top > 0) hipLaunchKernelGGL((lp_rows_kernel<DT, true, kThreads>), grid, dim3(kThreads), 0, st, p);
        else if (wave) hipLaunchKernelGGL((lp_rows_kernel<DT, false, 64>), grid, dim3(64), 0, st, p);
        else hipLaunchKernelGGL((lp_rows_kernel<DT, false, kThreads>), grid, dim3(kThreads), 0, st, p);
        if (p.parts > 1) hipLaunchKernelGGL((lp_merge_kernel<DT>), dim3(p.T), dim3(kThreads), 0, st, p);
        const long long n = p.T;
        p.x = (const char *)p.x + n * p.ldx * kSize;
        p.tok = (const char *)p.tok + n * p.C * (p.tok64 ? 8 : 4);
        p.lp += n * p.C, p.ent += n, p.ids += n * p.top, p.tlp += n * p.top;
    }
}

}  // namespace

extern "C" long long mica_token_logprobs_workspace_bytes(int T, int V, int dtype, int top) {
    if (T < 0 || V < 1 || top < 0 || top > kMaxTop || top > V) return -1;
    if (dtype != MICA_BF16 && dtype != MICA_FP16 && dtype != MICA_FP32) return -1;
    if (T == 0) return 0;
    int parts, bpp;
    divide(T, V, dtype == MICA_FP32 ? 4 : 8, top, parts, bpp);
    return part_bytes(T, parts, top);
}

extern "C" int mica_token_logprobs(const void *logits, int dtype, long long ldx, int T, int V, const void *tokens,
                                   int tokens_64, int C, int top, float *logprobs, float *entropy, long long *top_ids,
                                   float *top_logprobs, void *workspace, long long workspace_bytes,
                                   mica_stream_t stream) {
    if (dtype != MICA_BF16 && dtype != MICA_FP16 && dtype != MICA_FP32) return MICA_MISS_DTYPE;
    if (T < 0 || V < 1 || C < 0 || top < 0 || top > kMaxTop || top > V) return MICA_MISS_SHAPE;
    if (T == 0) return 0;
    if (!logits || !entropy || (C > 0 && (!tokens || !logprobs)) || (top > 0 && (!top_ids || !top_logprobs))) return MICA_MISS_ARG;
    if (ldx < V && T > 1) return MICA_MISS_STRIDE;
    const int size = dtype == MICA_FP32 ? 4 : 2;
    if ((uintptr_t)logits % size || (uintptr_t)tokens % (tokens_64 ? 8 : 4) || (uintptr_t)top_ids % 8 ||
        (uintptr_t)logprobs % 4 || (uintptr_t)entropy % 4 || (uintptr_t)top_logprobs % 4)
        return MICA_MISS_ALIGN;
    LpParams p{};
    p.x = logits; p.ldx = ldx; p.tok = tokens; p.tok64 = tokens_64 != 0; p.T = T; p.V = V; p.C = C; p.top = top;
    p.lp = logprobs; p.ent = entropy; p.ids = top_ids; p.tlp = top_logprobs;
    divide(T, V, 16 / size, top, p.parts, p.bpp);
    const long long need = part_bytes(T, p.parts, top);
    if (need && (!workspace || !mica_aligned16(workspace) || workspace_bytes < need)) return MICA_MISS_ARG;
    if (V > (1 << 30) || (long long)T * p.parts >= (1LL << 31)) return MICA_MISS_RANGE;
    p.pm = (Stat *)workspace;
    p.pk = (unsigned long long *)((char *)workspace + (long long)T * p.parts * 16);
    if (dtype == MICA_BF16) launch<MICA_BF16>(p, (hipStream_t)stream);
    else if (dtype == MICA_FP16) launch<MICA_FP16>(p, (hipStream_t)stream);
    else launch<MICA_FP32>(p, (hipStream_t)stream);
    return mica_err(hipGetLastError());
}
