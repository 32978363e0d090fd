// Attention of each sequence's newest rows over the paged 8-bit cache (mica_attention_paged), head dim 256, 4 query heads per
// key/value head; paged.h has the cache's layout.
//
//   o[t, h] = sum_{u <= p} softmax_u(scale q[t, h] . key_u[h / 4]) value_u[h / 4],   p = len - n + i  for row i of n
//   key_u = s_K q_u for a block's scale s_K and int8 q_u, bf16 in the rest; values likewise; zeros where p < 0
//
// The products are of whole numbers: int8 values are exact in bf16, so a block's key scale multiplies the scores and its value
// scale the weights, once each, and nothing is rounded that a bf16 cache would not round.
//
// Division: the tiles (pages, and the rest) of all units (a sequence's blocks of nb rows), one behind the other, are divided
// evenly over runs, and a worker takes a run for one key/value head: it may end one unit and begin the next, so that
// lengths that differ, or sequences that do not divide the chip, leave nothing idle.  pg_merge_kernel joins the partial
// softmax states (fp32) of the units that are divided.  Everything is found on the device from starts and lens.
//
// Two kernels: few rows (pg_few_kernel: a worker is a wave, which takes pages from memory into registers by itself) and more
// (pg_fwd_kernel: a worker is a workgroup, whose waves share each page through LDS).
#include "attn_common.h"
#include "paged.h"

namespace {

constexpr int kD = kPagedDim;
constexpr int kGroup = 4;               // query heads per key/value head
constexpr int kBK = kPage;              // keys of a tile: a page, or the rest
constexpr int kTile = kBK * kD * 2;     // 16 KB of K or V, in bf16
constexpr int kStage = 2 * kTile;

struct PagedParams {
    const uint16_t *q; long long shq, ldq; // head h of row t: q + h shq + t ldq
    uint16_t *o; long long sho, ldo;
    Ragged rows;
    Pages c;
    int fill;                              // rows of no sequence become zeros
    float scale_log2;                      // softmax scale x log2(e)
    int nb;                                // rows of a unit: a workgroup's (or a wave's) pairs are 4 nb
    int runs, least, begin;                // most runs; a run's fewest tiles; the tiles that a unit's beginning counts for
    float4 *part_o;                        // partial O: [part][64 fours of dims][4 nb pairs]
    float2 *part_ml;                       // partial (m, l): [part][4 nb pairs]
};

// zeros for rows i0 .. i0 + rows - 1 of those that no sequence has (the rows before the first and behind the last sequence)
MICA_DEVICE void fill_rows(const PagedParams &p, int hk, int i0, int rows, int tid, int threads) {
    const int before = p.rows.at(0), behind = p.rows.at(p.rows.B);
    for (int x = tid; x < rows * kGroup * (kD / 8); x += threads) {
        const int i = i0 + x / (kGroup * (kD / 8)), c = x % (kGroup * (kD / 8));
        const long long t = i < before ? i : (long long)behind + i - before;
        if (t < p.rows.T) *(u32x4 *)(p.o + (hk * kGroup + c / (kD / 8)) * p.sho + t * p.ldo + c % (kD / 8) * 8) = u32x4{0u, 0u, 0u, 0u};
    }
}

// The row of all units' tiles and its division.  All lanes of a wave call and get the same; a lane reads every 64th
// sequence's lengths.
struct Walk {
    int total, per;   // places in the row: tiles, and p.begin for each unit's beginning; those of a run
    int x, sum, base; // this lane's sequence of the 64 from `base` on: its places, those up to and with it
    MICA_DEVICE static int tiles(const PagedParams &p, int n, int len, int qb) {
        const int last = len - n + min(n, (qb + 1) * p.nb) - 1;
        return last < 0 ? 1 : last / kBK + 1; // (rows before the first token: a tile of which they see nothing)
    }
    MICA_DEVICE void take(const PagedParams &p, int from) {
        const int b = from + (int)(threadIdx.x & 63);
        base = from, x = 0;
        if (b < p.rows.B) {
            const int n = p.rows.rows(b), len = p.c.len(b);
            for (int qb = 0; qb * p.nb < n; ++qb) x += tiles(p, n, len, qb) + p.begin;
        }
        sum = wave_scan(x);
    }
    MICA_DEVICE Walk(const PagedParams &p) {
        total = 0;
        for (int from = (p.rows.B - 1) & ~63; from >= 0; from -= 64) { // (the first 64 last: they are kept)
            take(p, from);
            total += __builtin_amdgcn_readlane(sum, 63);
        }
        per = max((total + p.runs - 1) / p.runs, p.least + p.begin);
    }
    // the place where unit qb of sequence b begins; called once
    MICA_DEVICE int place(const PagedParams &p, int b, int qb) {
        int before = 0;
        for (int from = 0; from < b / 64 * 64; from += 64) {
            if (from) take(p, from);
            before += __builtin_amdgcn_readlane(sum, 63);
        }
        if (b >= 64) take(p, b / 64 * 64);
        before += __builtin_amdgcn_readlane(sum - x, b % 64);
        const int n = p.rows.rows(b), len = p.c.len(b);
        for (int q = 0; q < qb; ++q) before += tiles(p, n, len, q) + p.begin;
        return __builtin_amdgcn_readfirstlane(before);
    }
    // the unit at place `at` (below total), and the place where it begins; called once
    MICA_DEVICE void find(const PagedParams &p, int at, int &b, int &qb, int &from) {
        int before = 0;
        for (;;) {
            const unsigned long long past = __builtin_amdgcn_ballot_w64(before + sum > at);
            if (past != 0 || base + 64 >= p.rows.B) {
                const int l = past ? __builtin_ctzll(past) : 0;
                b = __builtin_amdgcn_readfirstlane(base + l);
                from = before + __builtin_amdgcn_readlane(sum - x, l);
                break;
            }
            before += __builtin_amdgcn_readlane(sum, 63);
            take(p, base + 64);
        }
        const int n = p.rows.rows(b), len = p.c.len(b);
        qb = 0;
        for (int t; (qb + 1) * p.nb < n && at >= from + (t = tiles(p, n, len, qb) + p.begin); ++qb) from += t;
        qb = __builtin_amdgcn_readfirstlane(qb), from = __builtin_amdgcn_readfirstlane(from);
    }
};

// A worker's place in its run: a unit, and the tiles of it that are this worker's
struct Piece {
    int b, qb;               // the unit
    int left;                // places of the run that are left
    int i0, i1, all;         // this worker's tiles; the unit's
    int part;                // where the partial state goes, for one head
    int n, len, first;       // the sequence's rows, tokens, first row
    MICA_DEVICE bool begin(const PagedParams &p, int run) {
        Walk w(p);
        const int at = run * w.per;
        if (at >= w.total) return false;
        int from;
        w.find(p, at, b, qb, from);
        left = __builtin_amdgcn_readfirstlane(min(w.per, w.total - at));
        i0 = __builtin_amdgcn_readfirstlane(at - from - p.begin);
        part = 2 * run;
        return open(p);
    }
    MICA_DEVICE bool next(const PagedParams &p) { // the run's next unit
        left -= i1 - i0;
        ++qb;
        if (qb * p.nb >= n) {
            qb = 0;
            do {
                if (++b >= p.rows.B) return false;
            } while (__builtin_amdgcn_readfirstlane(p.rows.rows(b)) == 0);
        }
        i0 = -p.begin;
        part |= 1; // (what lies between a run's first and last unit is whole)
        return open(p);
    }
    MICA_DEVICE bool whole() const { return i0 == 0 && i1 == all; }

private:
    MICA_DEVICE bool open(const PagedParams &p) {
        n = __builtin_amdgcn_readfirstlane(p.rows.rows(b));
        len = __builtin_amdgcn_readfirstlane(p.c.len(b));
        first = __builtin_amdgcn_readfirstlane(p.rows.at(b));
        all = Walk::tiles(p, n, len, qb);
        if (i0 < 0) left += i0, i0 = 0; // the rest of the unit's beginning
        i1 = min(i0 + left, all);
        return left > 0;
    }
};

// Pages and scales of 64 tiles of a sequence, a lane each: one round trip to memory for all of them.
struct Index {
    int base, page;
    float sk, sv;
    MICA_DEVICE void load(const PagedParams &p, int b, int hk, int whole, int from) {
        const int i = from + (int)(threadIdx.x & 63);
        base = from;
        page = i < whole ? p.c.page(b, i) : -1;
        // (a block without a page: NaN, for the rows that see it)
        sk = p.c.scale(page, 0, hk);
        sv = p.c.scale(page, 1, hk);
    }
    MICA_DEVICE int page_of(int i) const { return __builtin_amdgcn_readlane(page, i - base); }
    MICA_DEVICE float sk_of(int i) const { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sk), i - base)); }
    MICA_DEVICE float sv_of(int i) const { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sv), i - base)); }
};

// four int8 as two packed bf16 pairs
MICA_DEVICE u32x2 widen4(uint32_t w) {
    u32x2 x;
    x[0] = pack_bf16x2((float)(int8_t)w, (float)(int8_t)(w >> 8));
    x[1] = pack_bf16x2((float)(int8_t)(w >> 16), (float)((int32_t)w >> 24));
    return x;
}
MICA_DEVICE bf16x8 widen8(uint32_t a, uint32_t b) {
    const u32x2 x = widen4(a), y = widen4(b);
    return __builtin_bit_cast(bf16x8, u32x4{x[0], x[1], y[0], y[1]});
}

// The running softmax of a lane's pair, in log2 units relative to m
struct Softmax {
    float m, lsum;
    MICA_DEVICE void clear() { m = -__builtin_inff(), lsum = 0.0f; }
    // Scores sc of a tile (score r of a lane is key k0 + 8 (r / 4) + 4 hi + r % 4) become weights, unscaled ones in the sum and
    // sv times them in sc; `masked`: keys past pos get none.  A scale (the softmax's times a block's) may be 0 or negative: then
    // the least score is the largest product.  The reference moves only when the maximum exceeds it by more than
    // 8, and then O with it.
    MICA_DEVICE void add(f32x16 &sc, f32x16 (&O)[kD / 32], float scale, float sv, bool masked, int k0, int pos, int hi) {
        const float none = scale < 0.0f ? __builtin_inff() : -__builtin_inff();
        if (masked) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = k0 + 8 * (r >> 2) + 4 * hi + (r & 3) <= pos ? sc[r] : none;
        }
        float mx = none;
        if (scale < 0.0f) {
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = __builtin_fminf(mx, sc[r]);
            mx = half_swap_max(-mx) * -scale;
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = __builtin_fmaxf(mx, sc[r]);
            mx = half_swap_max(mx) * scale;
        }
        const bool grow = mx > m + 8.0f;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
        if (grow) m = mx;
        if (__builtin_amdgcn_ballot_w64(grow)) {
#pragma unroll
            for (int dt = 0; dt < kD / 32; ++dt) O[dt] *= alpha;
            lsum *= alpha;
        }
        const float ref = m == -__builtin_inff() ? 0.0f : m; // a row that has seen nothing yet: exp2(-inf - 0) = 0
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], scale, -ref));
        if (masked && !(scale > 0.0f && scale < __builtin_inff())) { // (a scale of 0 or NaN makes NaN of -inf)
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = k0 + 8 * (r >> 2) + 4 * hi + (r & 3) <= pos ? sc[r] : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < 16; r += 2) lsum += sc[r] + sc[r + 1];
        if (sv < __builtin_inff()) {
            sc *= sv;
        } else { // (a scale of NaN, and keys of no weight)
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = sc[r] == 0.0f ? 0.0f : sc[r] * sv;
        }
    }
};

// P^T operand of step s from the scores' place
MICA_DEVICE bf16x8 weights(const f32x16 &w, int s) {
    return __builtin_bit_cast(bf16x8, u32x4{pack_bf16x2(w[8 * s], w[8 * s + 1]), pack_bf16x2(w[8 * s + 2], w[8 * s + 3]),
                                            pack_bf16x2(w[8 * s + 4], w[8 * s + 5]), pack_bf16x2(w[8 * s + 6], w[8 * s + 7])});
}
// 2^127 in the place of every weight that is not zero
MICA_DEVICE bf16x8 indicators(const bf16x8 &x) {
    u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = ((w[e] & 0xffffu) ? 0x7f00u : 0u) | ((w[e] >> 16) ? 0x7f000000u : 0u);
    return __builtin_bit_cast(bf16x8, w);
}
// the values that are not finite of a V^T operand, see odd_value
MICA_DEVICE bf16x8 odd_values(const bf16x8 &x, uint32_t sign) {
    u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = odd_value(w[e] & 0xffffu, sign) | (odd_value(w[e] >> 16, sign) << 16);
    return __builtin_bit_cast(bf16x8, w);
}
MICA_DEVICE uint32_t without_odd(uint32_t w) {
    return w & ((odd_value(w & 0xffffu, 0) ? 0u : 0xffffu) | (odd_value(w >> 16, 0) ? 0u : 0xffff0000u));
}
// bits 15 and 31 are set where a packed value is not finite
MICA_DEVICE uint32_t odd_bits(uint32_t w) { return (w & 0x7f807f80u) + 0x00800080u; }

// A worker's state of its unit, left for pg_merge_kernel: (m, l) with l = -1 for a row that sees no key
MICA_DEVICE void leave(const PagedParams &p, long long part, int pair, int hi, bool blind, const f32x16 (&O)[kD / 32], float m,
                       float l) {
    const int np = kGroup * p.nb;
    if (pair >= np) return;
#pragma unroll
    for (int dt = 0; dt < kD / 32; ++dt)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const f32x16 x = O[dt];
            p.part_o[(part * 64 + (dt * 4 + r4) * 2 + hi) * np + pair] =
                blind ? float4{0.0f, 0.0f, 0.0f, 0.0f} : float4{x[4 * r4], x[4 * r4 + 1], x[4 * r4 + 2], x[4 * r4 + 3]};
        }
    if (hi == 0) p.part_ml[part * np + pair] = blind ? float2{-__builtin_inff(), -1.0f} : float2{m, l};
}

// ---- few rows: up to 8 G of a sequence ----
// A wave takes tiles by itself: a page's pieces go from memory straight into the registers of the matrix cores' operands, 16
// bytes a lane, each loaded for the next tile as soon as this one's has been widened, so that a wave has a page (16 KB) in
// flight all the time.  Nothing is shared and there is no barrier.  G waves take a run together, 8 rows each.
//
// Bound: up to 4 rows by HBM (64 single rows over up to 8192 tokens: 112 us, 4.9 TB/s, a copy's rate; 114 where the sequences' last
// blocks are not finished, whose tiles have nothing in flight beside them); then by instruction issue, about 800 for a page and
// wave, half of them to widen it, which all G waves repeat (64 x 8 rows 134 to 144 us, 16 177 to 181, 32 290 to 302).  Pages through
// LDS instead, by DMA of each wave: 126 us for single rows, 190 for 16.  Two waves a SIMD, queries in LDS: 16 rows 177 -> 187, 32 299
// -> 268, and twice the partial states to join (8 x 16 rows over 7000 58 -> 69); not built for G = 4 alone.
//
// Rounding: with one wave a run the weights are taken as two bf16 summands (hi and what it leaves), of pages and of the rest (64 x 8
// rows 131 -> 134 us, the rest's among them 137 -> 138.5); with more rows they are rounded to bf16 once (two summands: 32 x 32
// rows over up to 4096 97 -> 108 us).
template <int G>
__global__ __launch_bounds__(256, 1) void pg_few_kernel(PagedParams p) {
    __shared__ __attribute__((aligned(1024))) int8_t smem[4 * kTile]; // a wave's values of the rest
    const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int worker = blockIdx.x * (4 / G) + wave / G, rb = wave % G, hk = worker % p.c.HK, run = worker / p.c.HK;
    const int pair = rb * 32 + l32;
    if (run >= p.runs) return;
    if (p.fill && rb == 0) {
        const int none = p.rows.at(0) + p.rows.T - p.rows.at(p.rows.B);
        for (int i = run * 32; i < none; i += p.runs * 32) fill_rows(p, hk, i, 32, lane, 64);
    }
    int8_t *const mine = smem + wave * kTile;
    Piece w;
    if (!w.begin(p, run)) return;
    do {
        const int q0 = w.qb * p.nb, from = w.len - w.n, whole = w.len / kBK;
        const int t = q0 + (pair >> 2), head = hk * kGroup + (pair & 3), pos = from + t; // this lane's pair
        // Q fragments (B operand of S^T): step 2 c + e takes dims 32 c + 16 hi + 8 e .. + 7, as a page's bytes lie; rows past the
        // last repeat it
        bf16x8 qf[kD / 16];
        {
            const uint16_t *qr = p.q + head * p.shq + (long long)(w.first + min(t, w.n - 1)) * p.ldq + hi * 16;
#pragma unroll
            for (int s = 0; s < kD / 16; ++s) qf[s] = __builtin_bit_cast(bf16x8, *(const u32x4 *)(qr + (s >> 1) * 32 + (s & 1) * 8));
        }
        f32x16 O[kD / 32];
#pragma unroll
        for (int dt = 0; dt < kD / 32; ++dt) O[dt] = f32x16{};
        Softmax sm;
        sm.clear();
        const int end = min(w.i1, whole); // pages; then the rest
        auto left = [](const f32x16 &x) { // what the first summand of the weights leaves
            f32x16 lo = {};
            if constexpr (G == 1) {
#pragma unroll
                for (int r = 0; r < 16; ++r) lo[r] = x[r] - round_bf16(x[r]);
            }
            return lo;
        };
        if (w.i0 < end) {
            Index ix;
            ix.load(p, w.b, hk, whole, w.i0);
            const int at = l32 * 32 + hi * 16;
            auto source = [&](int page, int side) { // nothing of a block without a page: zeros
                return __builtin_amdgcn_make_buffer_rsrc((void *)p.c.block(max(page, 0), side, hk), 0, page >= 0 ? kPageBytes : 0,
                                                         kBufferFlags);
            };
            auto piece = [&](const __amdgpu_buffer_rsrc_t &r, int x) {
                return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at + x * 1024, 0, 0));
            };
            u32x4 rk[8], rv[8];
            {
                const int page = ix.page_of(w.i0);
                const __amdgpu_buffer_rsrc_t sk = source(page, 0), sv = source(page, 1);
#pragma unroll
                for (int x = 0; x < 8; ++x) rk[x] = piece(sk, x);
#pragma unroll
                for (int x = 0; x < 8; ++x) rv[x] = piece(sv, x);
            }
#pragma unroll 1
            for (int i = w.i0; i < end; ++i) {
                const float sk = ix.sk_of(i), sv = ix.sv_of(i);
                if (i + 1 - ix.base == 64) ix.load(p, w.b, hk, whole, i + 1);
                const int page = i + 1 < end ? ix.page_of(i + 1) : -1;
                const __amdgpu_buffer_rsrc_t nk = source(page, 0), nv = source(page, 1);
                f32x16 sc = {};
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const bf16x8 a = widen8(rk[x][0], rk[x][1]), c = widen8(rk[x][2], rk[x][3]);
                    rk[x] = piece(nk, x);
                    sc = mfma_bf16(a, qf[2 * x], sc);
                    sc = mfma_bf16(c, qf[2 * x + 1], sc);
                    __builtin_amdgcn_sched_barrier(0);
                }
                sm.add(sc, O, p.scale_log2 * sk, sv, (i + 1) * kBK - 1 > from + q0, i * kBK, pos, hi);
                const bf16x8 h0 = weights(sc, 0), h1 = weights(sc, 1);
                const f32x16 lo = left(sc);
                const bf16x8 g0 = weights(lo, 0), g1 = weights(lo, 1);
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const bf16x8 a = widen8(rv[x][0], rv[x][2]), c = widen8(rv[x][1], rv[x][3]);
                    rv[x] = piece(nv, x);
                    O[x] = mfma_bf16(a, h0, O[x]);
                    O[x] = mfma_bf16(c, h1, O[x]);
                    if constexpr (G == 1) {
                        O[x] = mfma_bf16(a, g0, O[x]);
                        O[x] = mfma_bf16(c, g1, O[x]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        if (w.i1 > end) {
            // The rest: keys from memory as operands, values by DMA into this wave's LDS (chunk c of row r at c ^ 4 (r % 4)),
            // from where they are read transposed; zeros past the last token.
            const int slot = __builtin_amdgcn_readfirstlane(p.c.slot(w.b)), have = slot < 0 ? 0 : w.len - whole * kBK;
            auto source = [&](int side) {
                return __builtin_amdgcn_make_buffer_rsrc((void *)p.c.rest(max(slot, 0), side, hk), 0, have * kD * 2, kBufferFlags);
            };
            const __amdgpu_buffer_rsrc_t kr = source(0), vr = source(1);
            f32x16 sc = {};
            u32x4 kf[kD / 16];
#pragma unroll
            for (int s = 0; s < kD / 16; ++s)
                kf[s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                      kr, l32 * (kD * 2) + hi * 32, (s >> 1) * 64 + (s & 1) * 16, 0));
#pragma unroll
            for (int x = 0; x < 16; ++x)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void *)(mine + x * 1024), 16,
                                                         (2 * x + hi) * (kD * 2) + ((l32 ^ (((2 * x + hi) & 3) << 2)) << 4), 0, 0, 0);
#pragma unroll
            for (int s = 0; s < kD / 16; ++s) sc = mfma_bf16(__builtin_bit_cast(bf16x8, kf[s]), qf[s], sc);
            const float one = slot < 0 ? __builtin_nanf("") : 1.0f;
            sm.add(sc, O, p.scale_log2 * one, one, true, whole * kBK, pos, hi);
            const bf16x8 pb[2] = {weights(sc, 0), weights(sc, 1)};
            const f32x16 lo = left(sc);
            const bf16x8 gb[2] = {weights(lo, 0), weights(lo, 1)};
            wait_vmcnt<0>();
            __asm__ volatile("" ::: "memory");
            uint32_t odd = 0;
#pragma unroll 4
            for (int x = 0; x < 16; ++x) {
                const u32x4 v = *(const u32x4 *)(mine + x * 1024 + lane * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) odd |= odd_bits(v[e]);
            }
            const uint32_t lds = (uint32_t)(uintptr_t)(lds_void *)mine;
            const int vrow = 4 * hi + ((l32 & 15) >> 2);
            const uint32_t vbase = lds + vrow * (kD * 2) + (((2 * (l32 >> 4) + ((l32 & 3) >> 1)) ^ ((vrow & 3) << 2)) << 4) + (l32 & 1) * 8;
            auto vfrag = [&](int s, int dt) {
                const uint32_t a = (vbase ^ (dt << 6)) + s * 16 * (kD * 2);
                const s16x4 x = tr_read((lds_s16x4 *)(uintptr_t)a, (lds_void *)smem);
                const s16x4 y = tr_read((lds_s16x4 *)(uintptr_t)(a + 8 * (kD * 2)), (lds_void *)smem);
                return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            // A value that is not finite must not reach the rows before its own (0 x inf = NaN): into the rows that give its key a
            // weight, then zeros in its place.
            if (__builtin_amdgcn_ballot_w64((odd & 0x80008000u) != 0)) {
                const bf16x8 i0 = indicators(pb[0]), i1 = indicators(pb[1]);
#pragma unroll
                for (int dt = 0; dt < kD / 32; ++dt)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        O[dt] = mfma_bf16(odd_values(vfrag(x & 1, dt), x & 2 ? 0x8000u : 0u), x & 1 ? i1 : i0, O[dt]);
                wait_lgkmcnt0();
                __asm__ volatile("" ::: "memory");
#pragma unroll 1
                for (int x = lane; x < kTile / 4; x += 64) ((uint32_t *)mine)[x] = without_odd(((uint32_t *)mine)[x]);
                wait_lgkmcnt0();
                __asm__ volatile("" ::: "memory");
            }
#pragma unroll
            for (int x = 0; x < 2 * (kD / 32); ++x) {
                const bf16x8 a = vfrag(x & 1, x >> 1);
                O[x >> 1] = mfma_bf16(a, pb[x & 1], O[x >> 1]);
                if constexpr (G == 1) O[x >> 1] = mfma_bf16(a, gb[x & 1], O[x >> 1]);
            }
            wait_lgkmcnt0();
        }
        const float l = half_swap_sum(sm.lsum);
        if (!w.whole()) {
            leave(p, (long long)w.part * p.c.HK + hk, pair, hi, pos < 0, O, sm.m, l);
        } else if (t < w.n && (pair >> 2) < p.nb) {
            // (a row whose scores are all -inf has no softmax: 0 / 0; one that sees no key: zeros)
            const float inv = 1.0f / l;
            uint16_t *out = p.o + head * p.sho + (long long)(w.first + t) * p.ldo + 4 * hi;
#pragma unroll
            for (int dt = 0; dt < kD / 32; ++dt)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const f32x16 x = O[dt];
                    u32x2 v = {pack_bf16x2(x[4 * r4] * inv, x[4 * r4 + 1] * inv), pack_bf16x2(x[4 * r4 + 2] * inv, x[4 * r4 + 3] * inv)};
                    if (pos < 0) v = u32x2{0u, 0u};
                    *(u32x2 *)(out + dt * 32 + 8 * r4) = v;
                }
        }
    } while (w.next(p));
}

// ---- more rows ----
// A workgroup of 8 waves shares each page, one workgroup a CU.  A page's 16 pieces come by LDS DMA, two of them by each wave,
// three tiles ahead into a ring; when its two have landed a wave widens them to bf16, once for all waves, into one of two
// stages, from which every operand is one contiguous 16-byte read a lane.  A wave holds 32 (row, head) pairs, 64 rows a
// workgroup: it computes S^T = K Q^T (32 keys x 32 pairs, v_mfma_f32_32x32x16_bf16), the online softmax of its pairs (a lane
// holds 16 of a pair's 32 scores, lane l ^ 32 the others) and O^T += V^T P^T.
//
// Bound: the matrix cores beside widening and softmax (2048 rows over 18001 tokens 530 to 560 us and 31 for the join, 1000 TFLOP/s; the
// library's 8192^3 product reaches 1400).  Pages widened in registers by the waves that use them, before the ring: 1234 us; the
// next page widened beside this one's PV, for one phase less: 636 against 605.
constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kOwn = 16 / kWaves;       // pieces of a page a wave brings
constexpr int kRing = 4;                // pages in the ring: one being widened, three on their way
constexpr int kRaw = 2 * kPageBytes;

__global__ __launch_bounds__(kThreads, 2) void pg_fwd_kernel(PagedParams p) {
    constexpr int NDT = kD / 32;            // 32-dim tiles of O
    constexpr int kSmem = 2 * kStage + kRing * kRaw; // the stages and the ring; the output, in the end
    static_assert(kSmem >= kWaves * 32 * kD * 2, "the output is staged in their place");
    // (one array: with several the compiler lets every operand read wait for all DMA in flight)
    __shared__ __attribute__((aligned(1024))) int8_t smem[kSmem + kWaves * 64 * 16 + 16];
    int *const index = (int *)(smem + kSmem) + (threadIdx.x >> 6) * 256; // this wave's: page and scales of 64 tiles, i at i % 64
    int *const odd_rest = (int *)(smem + kSmem + kWaves * 64 * 16);      // whether the rest holds a value that is not finite

    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int hk = blockIdx.x % p.c.HK, run = blockIdx.x / p.c.HK;
    if (p.fill) {
        const int none = p.rows.at(0) + p.rows.T - p.rows.at(p.rows.B);
        for (int i = run * 32; i < none; i += p.runs * 32) fill_rows(p, hk, i, 32, threadIdx.x, kThreads);
    }
    Piece w;
    if (!w.begin(p, run)) return;
    do {
        // what depends on the lane alone is made here, from an opaque copy of its id: the compiler would make it before the loop
        // and hold it in registers that the tiles need
        int tid = threadIdx.x;
        __asm__ volatile("" : "+v"(tid));
        const int lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
        const int q0 = w.qb * p.nb, from = w.len - w.n, whole = w.len / kBK;
        const int slot = __builtin_amdgcn_readfirstlane(p.c.slot(w.b)), have = slot < 0 ? 0 : w.len - whole * kBK;
        const int end = min(w.i1, whole); // pages; then the rest
        // Pages and scales of tiles i .. i + 31 into this wave's index: one round trip to memory for all of them
        auto look_up = [&](int i) {
            const int j = i + (lane & 31), page = j < whole ? p.c.page(w.b, j) : -1;
            // (a block without a page: NaN, for the rows that see it)
            const float x = p.c.scale(page, hi, hk);
            index[(j & 63) * 4] = page;
            index[(j & 63) * 4 + 1 + hi] = __float_as_int(x);
        };
        auto found = [&](int i, int what) { return __builtin_amdgcn_readfirstlane(index[(i & 63) * 4 + what]); };
        int known = w.i0 + 32; // the first tile that is not in the index
        look_up(w.i0);
        // DMA of tile i's pieces (of this wave): 0 .. 7 of a page are keys (32 dims of each token), 8 .. 15 values (32 dims'
        // rows).  Past the last page, and for a block without one, from a zero-sized buffer: every step issues as many.
        auto fetch = [&](int i) {
            const int page = i < end ? found(i, 0) : -1;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                (void *)p.c.block(max(page, 0), wave * kOwn >> 3, hk), 0, page >= 0 ? kPageBytes : 0, kBufferFlags);
            int ln = lane;
            __asm__ volatile("" : "+v"(ln));
            int8_t *s = smem + 2 * kStage + ((i - w.i0) & (kRing - 1)) * kRaw + wave * kOwn * 1024;
#pragma unroll
            for (int x = 0; x < kOwn; ++x)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)(s + x * 1024), 16,
                                                         (ln & 31) * 32 + (ln >> 5) * 16 + (wave * kOwn & 7) * 1024 + x * 1024, 0, 0, 0);
        };
        // Q fragments (B operand of S^T): step 2 c + e takes dims 32 c + 16 hi + 8 e .. + 7, as a page's bytes lie; rows past the
        // last repeat it
        const int t = q0 + wave * 8 + (l32 >> 2), pos = from + t; // this lane's pair: row t, head l % 4
        bf16x8 qf[kD / 16];
        {
            const uint16_t *qr = p.q + (hk * kGroup + (l32 & 3)) * p.shq + (long long)(w.first + min(t, w.n - 1)) * p.ldq + hi * 16;
#pragma unroll
            for (int s = 0; s < kD / 16; ++s) qf[s] = __builtin_bit_cast(bf16x8, *(const u32x4 *)(qr + (s >> 1) * 32 + (s & 1) * 8));
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < kRing - 1; ++x) {
            fetch(w.i0 + x);
        }
        // The rest into stage st: bf16 rows, the same operands; zeros past its last token (the buffer's range check).
        auto stage_rest = [&](int st) {
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)p.c.rest(max(slot, 0), wave * kOwn >> 3, hk),
                                                                               0, have * kD * 2, kBufferFlags);
            uint32_t odd = 0;
            int ln = lane;
            __asm__ volatile("" : "+v"(ln));
            const int row = ln & 31, half = ln >> 5;
#pragma unroll 1
            for (int x = 0; x < kOwn; ++x) {
                const int dims = ((wave * kOwn + x) & 7) * 64; // the piece's dims, in bytes of a row
                u32x4 a, c;
                if (wave < 4) {
                    const int at = row * (kD * 2) + dims + half * 32;
                    a = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
                    c = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at + 16, 0, 0));
                } else {
                    const int at = 4 * half * (kD * 2) + dims + row * 2;
                    uint32_t v[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) // step e / 8, its token e % 8
                        v[e] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(
                            r, at + (16 * (e >> 3) + 8 * ((e >> 2) & 1) + (e & 3)) * (kD * 2), 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] = v[2 * e] | v[2 * e + 1] << 16, c[e] = v[8 + 2 * e] | v[9 + 2 * e] << 16;
#pragma unroll
                    for (int e = 0; e < 4; ++e) odd |= odd_bits(a[e]) | odd_bits(c[e]);
                }
                int8_t *s = smem + st * kStage + (wave * kOwn + x) * 2048 + ln * 16;
                *(u32x4 *)s = a;
                *(u32x4 *)(s + 1024) = c;
            }
            if (__builtin_amdgcn_ballot_w64((odd & 0x80008000u) != 0) && ln == 0) *odd_rest = 1;
        };
        const uint32_t base = (uint32_t)(uintptr_t)(lds_void *)smem + lane * 16;
        // (opaque: as a constant it would be put into lds_read itself, which then says nothing)
        lds_void *none = (lds_void *)smem;
        __asm__ volatile("" : "+s"(none));
        auto kfrag = [none](uint32_t a, int s) { return __builtin_bit_cast(bf16x8, lds_read(a + s * 1024, none)); };
        auto vfrag = [none](uint32_t a, int s, int dt) { return __builtin_bit_cast(bf16x8, lds_read(a + dt * 2048 + s * 1024, none)); };
        f32x16 O[NDT];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) O[dt] = f32x16{};
        Softmax sm;
        sm.clear();
        if (tid == 0) *odd_rest = 0;
        wait_vmcnt<(kRing - 1) * kOwn>(); // the queries are there (said here, or the loop's first use waits for all DMA at every tile)
        wait_lgkmcnt0();
        meet();
#pragma unroll 1
        for (int i = w.i0; i < w.i1; ++i) {
            const uint32_t at = base + ((i - w.i0) & 1) * kStage;
            float sk, sv;
            if (i < whole) {
                // Tile i's pieces of this wave have landed (those of the next two, 2 kOwn, may still be out): each becomes two
                // operands.  Keys: bytes 8 e .. 8 e + 7 are step 2 c + e's; values: fours s and s + 2 are step s's (tokens 16 s + 4
                // hi .. + 3 and 8 more on: P^T's accumulator rows).
                wait_vmcnt<2 * kOwn>();
                __builtin_amdgcn_sched_barrier(0);
                const uint32_t src = base + 2 * kStage + ((i - w.i0) & (kRing - 1)) * kRaw + wave * kOwn * 1024;
                u32x4 raw[kOwn];
#pragma unroll
                for (int x = 0; x < kOwn; ++x) raw[x] = lds_read(src + x * 1024, none);
#pragma unroll
                for (int x = 0; x < kOwn; ++x) {
                    const uint32_t m1 = wave < 4 ? raw[x][1] : raw[x][2], m2 = wave < 4 ? raw[x][2] : raw[x][1];
                    const bf16x8 a = widen8(raw[x][0], m1), c = widen8(m2, raw[x][3]);
                    const uint32_t to = at + (wave * kOwn + x) * 2048;
                    *(lds_u32x4 *)(uintptr_t)to = __builtin_bit_cast(u32x4, a);
                    *(lds_u32x4 *)(uintptr_t)(to + 1024) = __builtin_bit_cast(u32x4, c);
                }
                sk = __int_as_float(found(i, 1)), sv = __int_as_float(found(i, 2));
            } else {
                stage_rest((i - w.i0) & 1);
                sk = sv = slot < 0 ? __builtin_nanf("") : 1.0f;
            }
            // the next tile of the ring, whose place this wave has read a step ago
            if (i + kRing - 1 == known && known < end) look_up(known), known += 32;
            fetch(i + kRing - 1);
            // every wave's pieces are there; nobody reads the other stage (tile i - 1) any more when tile i + 1 is written to it
            wait_lgkmcnt0();
            meet();
            // ---- S^T = K Q^T: rows = keys of the tile, column = this lane's pair ----
            constexpr int kPf = 3; // operands read ahead
            f32x16 sc = {};
            __builtin_amdgcn_s_setprio(1);
            bf16x8 kf[kPf];
#pragma unroll
            for (int s = 0; s < kPf; ++s) kf[s] = kfrag(at, s);
#pragma unroll
            for (int s = 0; s < kD / 16; ++s) {
                const bf16x8 a = kf[s % kPf];
                if (s + kPf < kD / 16) kf[s % kPf] = kfrag(at, s + kPf);
                __builtin_amdgcn_sched_barrier(0);
                sc = mfma_bf16(a, qf[s], sc);
            }
            __builtin_amdgcn_s_setprio(0);
            sm.add(sc, O, p.scale_log2 * sk, sv, (i + 1) * kBK - 1 > from + q0, i * kBK, pos, hi);
            // the matrix cores' operand type; the sum keeps the unrounded weights
            bf16x8 pb[2] = {weights(sc, 0), weights(sc, 1)};
            // A value of the rest that is not finite must not reach the rows before its own (0 x inf = NaN): zeros in its place, and
            // it goes into the rows that give its key a weight, by products of their own with what the ring then holds (nothing
            // else does: the rest is a unit's last tile).
            const bool odd = i >= whole && *odd_rest;
            if (odd) {
                wait_vmcnt<0>(); // (the empty loads)
                __syncthreads();
#pragma unroll 1
                for (int x = threadIdx.x; x < kTile / 4; x += kThreads) {
                    uint32_t *v = (uint32_t *)(smem + ((i - w.i0) & 1) * kStage + kTile) + x, *o = (uint32_t *)(smem + 2 * kStage) + x;
                    const uint32_t lo = *v & 0xffffu, hh = *v >> 16;
                    o[0] = odd_value(lo, 0) | odd_value(hh, 0) << 16;
                    o[kTile / 4] = odd_value(lo, 0x8000u) | odd_value(hh, 0x8000u) << 16;
                    *v = without_odd(*v);
                }
                __syncthreads();
            }
            // ---- O^T += V^T P^T ----
            auto product = [&](uint32_t v) { // values at v
                __builtin_amdgcn_s_setprio(1);
                bf16x8 vf[kPf];
#pragma unroll
                for (int x = 0; x < kPf; ++x) vf[x] = vfrag(v, x / NDT, x % NDT);
#pragma unroll
                for (int x = 0; x < 2 * NDT; ++x) {
                    const bf16x8 a = vf[x % kPf];
                    if (x + kPf < 2 * NDT) vf[x % kPf] = vfrag(v, (x + kPf) / NDT, (x + kPf) % NDT);
                    __builtin_amdgcn_sched_barrier(0);
                    O[x % NDT] = mfma_bf16(a, pb[x / NDT], O[x % NDT]);
                }
                __builtin_amdgcn_s_setprio(0);
            };
            product(at + kTile);
            if (odd) {
                pb[0] = indicators(pb[0]), pb[1] = indicators(pb[1]);
#pragma unroll 1
                for (int x = 0; x < 2; ++x) product(base + 2 * kStage + x * kTile);
            }
        }
        wait_vmcnt<0>(); // the last (empty) loads have written before the ring is used again or given up
        const float l = half_swap_sum(sm.lsum);
        __asm__ volatile("" : "+v"(tid));
        const int ln = tid & 63, row = wave * 32 + (ln & 31), half = ln >> 5;
        if (!w.whole()) {
            leave(p, (long long)w.part * p.c.HK + hk, row, half, pos < 0, O, sm.m, l);
        } else {
            // ---- normalise (a row whose scores are all -inf has no softmax: 0 / 0; one that sees no key: zeros), stage, write ----
            const float inv = 1.0f / l;
            __syncthreads();
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const int d = dt * 32 + 8 * r4 + 4 * half;
                    const f32x16 x = O[dt];
                    u32x2 v = {pack_bf16x2(x[4 * r4] * inv, x[4 * r4 + 1] * inv), pack_bf16x2(x[4 * r4 + 2] * inv, x[4 * r4 + 3] * inv)};
                    if (pos < 0) v = u32x2{0u, 0u};
                    *(u32x2 *)(smem + row * (kD * 2) + (((d >> 3) ^ (ln & 31)) << 4) + (d & 4) * 2) = v;
                }
            __syncthreads();
#pragma unroll 2
            for (int x = tid; x < 32 * kWaves * 32; x += kThreads) {
                const int rr = x >> 5, ch = x & 31, tt = q0 + (rr >> 2);
                if (tt < w.n)
                    *(u32x4 *)(p.o + (long long)(hk * kGroup + (rr & 3)) * p.sho + (long long)(w.first + tt) * p.ldo + ch * 8) =
                        *(const u32x4 *)(smem + rr * (kD * 2) + ((ch ^ (rr & 31)) << 4));
            }
        }
        __syncthreads(); // everybody is done with the stages and the ring
    } while (w.next(p));
}

// The partial states of a divided unit joined: with M = max_c m_c, w_c = 2^(m_c - M), o = (sum w_c O_c) / (sum w_c l_c).  A
// workgroup goes by the units, or, where there may be more of them than runs, by the place where run r begins, and joins the
// unit there if it is the unit's first division; a thread has four dims of a pair, for K pairs, or W waves share the parts of
// theirs.  Bound: the partial states, read from the caches (2048 rows over 18001 tokens: about 100 MB, 31 us), or the launch,
// 5 us.  By units where these are fewer than runs: 32 x up to 16 rows over up to 4096 65 -> 60 us; four pairs a thread: 8 x up to
// 240 rows over 7152 186 -> 178.
template <int W, int K, bool UNITS>
__global__ __launch_bounds__(256) void pg_merge_kernel(PagedParams p) {
    __shared__ float4 accs[W > 1 ? 4 : 1][64];
    __shared__ float2 mls[W > 1 ? 4 : 1][64];
    const int np = kGroup * p.nb, blocks = np * W / (4 * K); // workgroups that share a unit's 64 x np fours
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int x0 = (blockIdx.x % blocks * 4 + wave) / W * (64 * K) + lane;
    const int hk = blockIdx.x / blocks % p.c.HK, y = blockIdx.x / blocks / p.c.HK;
    Walk all(p);
    int b, qb, from;
    if constexpr (UNITS) {
        if (!find_unit(p.rows.B, [&](int i) { return (p.rows.rows(i) + p.nb - 1) / p.nb; }, y, b, qb)) return;
        from = all.place(p, b, qb);
    } else {
        const int at = (y + 1) * all.per;
        if (at >= all.total) return;
        all.find(p, at, b, qb, from);
        const int start = from + p.begin;
        if (at <= start || start / all.per != y) return;
    }
    const int start = from + p.begin, g0 = start / all.per; // the unit's first tile, and the run that has it
    const int n = p.rows.rows(b), tiles = Walk::tiles(p, n, p.c.len(b), qb);
    const int parts = (start + tiles - 1) / all.per - g0 + 1;
    if (parts < 2) return; // its worker wrote it
    auto part = [&](int c) { // (a unit that begins within a run has the run's second place)
        const int g = min(max(g0 + c, 0), p.runs - 1); // (starts that are no running sum may wrap places round)
        return (2 * (long long)g + (g * all.per < from)) * p.c.HK + hk;
    };
    float mx[K], l[K];
    float4 acc[K];
    // no part has a key that counts: weights 1 on zeros (a sum that is NaN or -1 stays so)
    auto weight = [](float m, float top) { return top == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - top); };
    auto add = [&](int k, float w, float2 ml, float4 o) {
        l[k] += w * ml.y;
        acc[k].x += w * o.x;
        acc[k].y += w * o.y;
        acc[k].z += w * o.z;
        acc[k].w += w * o.w;
    };
#pragma unroll
    for (int k = 0; k < K; ++k) mx[k] = -__builtin_inff(), l[k] = 0.0f, acc[k] = float4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kBatch = W > 1 ? 8 : K > 1 ? 2 : 4; // parts whose loads are in flight together
    for (int c0 = wave % W; c0 < parts; c0 += W * kBatch) {
        float2 ml[K][kBatch];
        float4 o[K][kBatch];
#pragma unroll
        for (int y = 0; y < kBatch; ++y) {
            const int c = c0 + y * W;
            const long long at = part(c < parts ? c : c0);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int x = x0 + k * 64;
                ml[k][y] = p.part_ml[at * np + x % np];
                o[k][y] = p.part_o[at * 64 * np + x];
                if (c >= parts) ml[k][y] = float2{-__builtin_inff(), 0.0f}, o[k][y] = float4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float top = mx[k];
#pragma unroll
            for (int y = 0; y < kBatch; ++y) top = __builtin_fmaxf(top, ml[k][y].x);
            const float w = weight(mx[k], top);
            l[k] *= w, acc[k].x *= w, acc[k].y *= w, acc[k].z *= w, acc[k].w *= w;
            mx[k] = top;
#pragma unroll
            for (int y = 0; y < kBatch; ++y) add(k, weight(ml[k][y].x, mx[k]), ml[k][y], o[k][y]);
        }
    }
    if constexpr (W > 1) {
        accs[wave][lane] = acc[0], mls[wave][lane] = float2{mx[0], l[0]};
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 1; w < W; ++w) mx[0] = __builtin_fmaxf(mx[0], mls[w][lane].x);
        l[0] = 0.0f, acc[0] = float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; ++w) add(0, weight(mls[w][lane].x, mx[0]), mls[w][lane], accs[w][lane]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int x = x0 + k * 64, pair = x % np, four = x / np, t = qb * p.nb + (pair >> 2);
        if (t >= n) continue;
        const float inv = l[k] < 0.0f ? 0.0f : 1.0f / l[k]; // (a row that sees no key: the parts' -1)
        const u32x2 w = {pack_bf16x2(acc[k].x * inv, acc[k].y * inv), pack_bf16x2(acc[k].z * inv, acc[k].w * inv)};
        *(u32x2 *)(p.o + (hk * kGroup + (pair & 3)) * p.sho + (long long)(p.rows.at(b) + t) * p.ldo + four * 4) = w;
    }
}

// ---- host side ----

constexpr int kCus = 256;

struct Plan {
    int G;                       // pg_few_kernel's waves of a run; 0: pg_fwd_kernel
    int nb, runs, least, begin;  // see PagedParams
    long long units, tiles, states; // most units; most places of the row; partial states
};

Plan plan(long long B, long long T, int HK, int width, int longest) {
    Plan pl{};
    // Unknown: as if all had as many rows (64 single tokens over up to 8192: 112 us, with T as the guess 305; 32 x up
    // to 16 over up to 4096 59 / 106).
    const long long guess = longest > 0 ? longest : B > 0 ? (T + B - 1) / B : T, hint = guess < T ? guess : T;
    // 8 rows a wave.  64 sequences of up to 8192 tokens, us with G = 1 / 2 / 4 / the workgroup kernel: 8 rows 134 / 169 / 274 / 306,
    // 16 rows 177 (G = 2) / 284 / 321, 32 rows 299 (G = 4) / 331; 8 x 32 rows over 7000 82 / 91.  All units of a call are as the longest
    // sequence asks.  Where most have fewer rows, smaller units can be faster, which the longest does not tell: with G = 2 / 4, 32 x
    // up to 32 rows over up to 4096 86 / 91, 64 x up to 32 over up to 8192 275 / 284, but 64 x up to 32 over 1000 80 / 75, 32 x 32
    // over up to 4096 99 / 96; 2048 rows beside 63 single ones 545 in one call, 269 + 111 in two.
    pl.G = hint <= 8 ? 1 : hint <= 16 ? 2 : hint <= 32 ? 4 : 0;
    // (a unit's rows are those of its partial states: single rows with nb = 1 / 2 / 4 / 8 112 / 114 / 120 / 128 us)
    pl.nb = hint <= 1 ? 1 : hint <= 2 ? 2 : hint <= 4 ? 4 : pl.G ? 8 * pl.G : 64;
    const long long most = (T + (pl.nb - 1) * B) / pl.nb;
    pl.units = most < T ? most : T;
    // What a unit's beginning costs, in tiles: few rows with 0 / 1 / 2 / 4 64 x 1 over up to 8192 117 / 114 / 112 / 112 us, 32 x up to 16
    // over up to 4096 64 / 60 / 58 / 58, and a run's one unit has none (1 x 500: 15.5 / 17.4 / 20.2 / 23.3); the workgroup kernel
    // with 0 / 2 / 4 / 8 64 x 64 over up to 4096 256 / 232 / 215 / 216.
    pl.begin = B == 1 && pl.units == 1 ? 0 : pl.G ? 2 : 4;
    // A run's fewest tiles: few rows 1 / 2 / 4, 1 x 500 15.5 / 18.5 / 21.2 us; the workgroup kernel 1 / 2 / 4 / 8, 64 rows over 2000
    // 55 / 44 / 36 / 35 (and as many partial states fewer to join).
    pl.least = pl.G ? 1 : 4;
    pl.tiles = pl.units * (width + 1ll + pl.begin);
    const long long slots = pl.G ? 4 * kCus / pl.G : kCus; // runs that the chip holds at once
    long long runs = slots / HK > 0 ? slots / HK : 1;
    const long long useful = pl.tiles / (pl.least + pl.begin) + 1; // (no more than can have tiles)
    pl.runs = (int)(runs < useful ? runs : useful);
    pl.states = B > 0 && pl.runs > 1 ? 2ll * pl.runs * HK : 0;
    return pl;
}
long long state_bytes(const Plan &pl) { return pl.states * kGroup * pl.nb * (kD * 4 + 8); }

}  // namespace

extern "C" int mica_attention_paged(const void *q, long long shq, long long ldq, void *o, long long sho, long long ldo,
                                    const int *starts, int B, int T, int HQ, const void *data, const float *scales,
                                    const void *recent, int pages, int n_slots, int HK, int head_dim, const int *table,
                                    long long ldt, int width, const int *lens, const int *slots, float scale, int fill,
                                    int longest, void *workspace, long long workspace_bytes, mica_stream_t stream) {
    if (B < 0 || T < 0) return MICA_MISS_SHAPE;
    if (!(scale > 0.0f) || !(scale * kLog2e < __builtin_inff())) return MICA_MISS_ARG;
    if (T == 0 || (B == 0 && !fill)) return 0;
    PagedParams p{};
    if (const int rc = mica_paged_check(p.c, (void *)data, (void *)scales, (void *)recent, pages, n_slots, HK, head_dim, table,
                                        ldt, width, lens, slots, B))
        return rc;
    if (HQ != HK * kGroup) return MICA_MISS_SHAPE;
    if (!q || !o || !starts) return MICA_MISS_ARG;
    for (long long x : {shq, ldq, sho, ldo})
        if (x < 0 || x % 8) return MICA_MISS_STRIDE;
    if (!mica_aligned16(q) || !mica_aligned16(o) || ((uintptr_t)starts & 3)) return MICA_MISS_ALIGN;
    const Plan pl = plan(B, T, HK, width, longest);
    if (pl.tiles >= (1ll << 30) || B >= (1 << 30) || T >= (1 << 29)) return MICA_MISS_RANGE; // (places are ints)
    if (pl.states && (!workspace || !mica_aligned16(workspace) || workspace_bytes < state_bytes(pl))) return MICA_MISS_ARG;
    p.q = (const uint16_t *)q; p.shq = shq; p.ldq = ldq;
    p.o = (uint16_t *)o; p.sho = sho; p.ldo = ldo;
    p.rows = Ragged{starts, B, T};
    p.fill = fill;
    p.scale_log2 = scale * kLog2e;
    p.nb = pl.nb, p.runs = pl.runs, p.least = pl.least, p.begin = pl.begin;
    p.part_o = (float4 *)workspace;
    p.part_ml = (float2 *)((char *)workspace + pl.states * kGroup * pl.nb * kD * 4);
    hipStream_t st = (hipStream_t)stream;
    const long long workers = (long long)pl.runs * HK;
    const unsigned few = pl.G ? (unsigned)((workers * pl.G + 3) / 4) : 0;
    if (pl.G == 1) hipLaunchKernelGGL(pg_few_kernel<1>, dim3(few), dim3(256), 0, st, p);
    else if (pl.G == 2) hipLaunchKernelGGL(pg_few_kernel<2>, dim3(few), dim3(256), 0, st, p);
    else if (pl.G == 4) hipLaunchKernelGGL(pg_few_kernel<4>, dim3(few), dim3(256), 0, st, p);
    else hipLaunchKernelGGL(pg_fwd_kernel, dim3((unsigned)workers), dim3(kThreads), 0, st, p);
    if (const int rc = mica_err(hipGetLastError())) return rc;
    if (pl.states == 0) return 0;
    const bool units = pl.units < pl.runs;
    const unsigned joins = (unsigned)((units ? pl.units : pl.runs - 1) * HK * pl.nb);
    // Many parts a unit, and few workgroups with four pairs a thread: four waves share the parts.  Without / with, us: 16 rows
    // after 30000 tokens 77 / 39, 32 after 30000 70 / 51, 64 after 30000 80 / 68, 4 x 16 after 7000 45 / 37, but 8 x 16 57 / 58,
    // 4 x 64 63 / 73.
    if (units && pl.runs >= 8 * pl.units && (pl.nb <= 8 || joins < 4 * kCus / 2))
        hipLaunchKernelGGL((pg_merge_kernel<4, 1, true>), dim3(joins * 4), dim3(256), 0, st, p);
    else if (units && pl.nb < 4) hipLaunchKernelGGL((pg_merge_kernel<1, 1, true>), dim3(joins), dim3(256), 0, st, p);
    else if (units) hipLaunchKernelGGL((pg_merge_kernel<1, 4, true>), dim3(joins / 4), dim3(256), 0, st, p);
    else if (pl.nb < 4) hipLaunchKernelGGL((pg_merge_kernel<1, 1, false>), dim3(joins), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((pg_merge_kernel<1, 4, false>), dim3(joins / 4), dim3(256), 0, st, p);
    return mica_err(hipGetLastError());
}

extern "C" long long mica_attention_paged_workspace_bytes(int B, int T, int HK, int width, int longest) {
    if (B < 0 || T < 0 || HK <= 0 || HK > (1 << 16) || width < 0 || width > (1 << 24)) return -1;
    return state_bytes(plan(B, T, HK, width, longest));
}
