// Causal grouped-query attention over prompts of different lengths packed one behind the other (mica_attention_packed), head
// dim 256, 4 query heads per key/value head.
//
//   o[t, h] = sum_{u in seq(t), u <= t} softmax_u(scale q[t, h] . k[u, h / 4]) v[u, h / 4]
//
// Work split: a workgroup takes one key/value head and a block of 32 rows of one sequence; wave w takes query head 4 hk + w, so
// that every tile of 32 keys brought into LDS serves four heads.  It computes S^T = K Q^T (32 keys x 32 rows,
// v_mfma_f32_32x32x16_bf16), the online softmax of its rows (a lane holds 16 of a row's 32 scores, lane l ^ 32 the others) and
// O^T += V^T P^T.  Blocks are found on the device from the sequences' starts, so that nothing is padded.  Where a few long
// prompts do not fill the chip, a block's keys are divided over workgroups, whose partial states (fp32) pk_merge_kernel joins.
//
// Data movement: K and V tiles come by LDS DMA into two stages in turn, 16-byte chunks XOR-swizzled by row, rows past the
// sequence's end as zeros (the buffer's range check); V is kept as it lies in memory and its V^T fragments are transposing
// reads (ds_read_b64_tr_b16: 16 lanes fetch 4 keys x 16 dims and each gets the 4 keys of one dim).
//
// Bound: the matrix cores beside the softmax, two waves a SIMD (10922 + 5461 tokens 1029 to 1094 us, 1115 to 1190 TFLOP/s, busy 68 %
// of the cycles; the library's 8192^3 product reaches 1400); of shorter prompts a block's queries and output as well, 16 us beside
// 1.65 us a tile, which two workgroups a CU hide poorly (13 of up to 2047 tokens 188 to 205 us, 810 to 880 TFLOP/s); of a short one
// its tiles one after the other (77 tokens 9 us).  The queries come straight from memory, a lane a row (by whole rows through LDS:
// 198.5 -> 196 us, not kept).  Rounding: the weights become bf16 for the matrix cores, their sum does not, and the result is
// rounded once.
#include "attn_common.h"
#include "ragged.h"

namespace {

constexpr int kD = 256;             // head dim
constexpr int kGroup = 4;           // query heads per key/value head, a wave each
constexpr int kB = 32;              // rows of a block, keys of a tile
constexpr int kThreads = 64 * kGroup;
constexpr int kRows = kGroup * kB;  // (head, row) pairs of a block
constexpr int kTile = kB * kD * 2;  // 16 KB of K or V
constexpr int kStage = 2 * kTile;

struct PackedParams {
    const uint16_t *q; long long shq, ldq; // head h of row t: q + h shq + t ldq
    const uint16_t *k; long long shk, ldk;
    const uint16_t *v; long long shv, ldv;
    uint16_t *o; long long sho, ldo;
    Ragged rows;
    int HK, fill;                          // fill: rows of no sequence become zeros
    float scale_log2;                      // softmax scale x log2(e)
    int chunk, chunks;                     // a block's tiles are divided into chunks of about `chunk`, at most `chunks` of them
    float4 *part_o;                        // partial O: [block][chunk][HK][64 fours of dims][128 rows x heads]
    float2 *part_ml;                       // partial (m, l): [block][chunk][HK][128]
    MICA_DEVICE int parts(int tiles) const { return min((tiles + chunk - 1) / chunk, chunks); }
};

// zeros for rows i0 .. i0 + 31 of those that no sequence has (the rows before the first and behind the last sequence)
MICA_DEVICE void fill_rows(const PackedParams &p, int hk, int i0) {
    const int before = p.rows.at(0), behind = p.rows.at(p.rows.B);
    for (int x = threadIdx.x; x < kB * kGroup * (kD / 8); x += kThreads) {
        const int i = i0 + x / (kGroup * (kD / 8)), c = x % (kGroup * (kD / 8));
        const long long t = i < before ? i : (long long)behind + i - before;
        if (t < p.rows.T) *(u32x4 *)(p.o + (hk * kGroup + c / (kD / 8)) * p.sho + t * p.ldo + c % (kD / 8) * 8) = u32x4{0u, 0u, 0u, 0u};
    }
}

// The id-th block of all, the longest first (a block has as many tiles as its place in its sequence, and one): with one sequence
// after the other the last ones keep a few CUs busy alone (13 prompts of up to 2047 tokens: 202 -> 196 us).  Up to 64 sequences, a
// lane each; a lane for each of 64 candidate places.  False where there are fewer blocks (b is then their number).
MICA_DEVICE bool longest_first(const Ragged &rows, int id, int &b, int &qb) {
    const int lane = threadIdx.x & 63;
    const int nb = lane < rows.B ? (rows.rows(lane) + kB - 1) / kB : 0;
    int most = nb;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) most = max(most, __shfl_xor(most, m, 64));
    most = __builtin_amdgcn_readfirstlane(most);
    auto from = [&](int place) { // blocks at that place or later
        int n = 0;
        for (int i = 0; i < rows.B; ++i) n += max(__builtin_amdgcn_readlane(nb, i) - place, 0);
        return n;
    };
    int step = 1, place = 0; // the last place from which on there are more than id blocks, by strides
    while (step * 64 <= most) step *= 64;
    for (;; step /= 64) {
        const int n = from(place + lane * step);
        const unsigned long long more = __builtin_amdgcn_ballot_w64(n > id);
        if (!more) {
            b = __builtin_amdgcn_readfirstlane(n);
            return false;
        }
        place += (63 - __builtin_clzll(more)) * step;
        if (step == 1) break;
    }
    const unsigned long long has = __builtin_amdgcn_ballot_w64(nb > place);
    const int rank = __builtin_popcountll(has & ((1ull << lane) - 1));
    b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(nb > place && rank == id - from(place + 1)));
    qb = place;
    return true;
}

// The id-th block: its sequence and its place in it; false where there are fewer (b is then their number)
MICA_DEVICE bool find_block(const Ragged &rows, int id, int &b, int &qb) {
    bool any;
    if (rows.B == 1) { // (no search for one prompt)
        const int nb = (rows.rows(0) + kB - 1) / kB;
        any = id < nb, b = any ? 0 : nb, qb = nb - 1 - id;
    } else if (rows.B <= 64) {
        any = longest_first(rows, id, b, qb);
    } else {
        any = find_unit(rows.B, [&](int i) { return (rows.rows(i) + kB - 1) / kB; }, id, b, qb);
        if (any) qb = (rows.rows(b) + kB - 1) / kB - 1 - qb; // a sequence's longest first
    }
    b = __builtin_amdgcn_readfirstlane(b), qb = __builtin_amdgcn_readfirstlane(qb);
    return any;
}

__global__ __launch_bounds__(kThreads, 2) void pk_fwd_kernel(PackedParams p) {
    constexpr int kSmem = kGroup * kB * kD * 2 > 2 * kStage ? kGroup * kB * kD * 2 : 2 * kStage; // the stages; the output, in the end
    __shared__ __attribute__((aligned(1024))) int8_t smem[kSmem + 16];
    int *const odd_tile = (int *)(smem + kSmem); // whether the diagonal tile holds a value that is not finite

    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
    const int hk = blockIdx.x % p.HK, chunk = blockIdx.x / p.HK % p.chunks, id = blockIdx.x / p.HK / p.chunks;
    int b, qb;
    if (!find_block(p.rows, id, b, qb)) {
        if (p.fill && chunk == 0) fill_rows(p, hk, (id - b) * kB);
        return;
    }
    const int first = p.rows.at(b), n = p.rows.rows(b), q0 = qb * kB;
    const int parts = p.parts(qb + 1); // this workgroup's tiles, i0 .. i1 - 1 of the block's
    if (chunk >= parts) return;
    const int i0 = (int)((long long)(qb + 1) * chunk / parts), i1 = (int)((long long)(qb + 1) * (chunk + 1) / parts);

    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void *)smem;
    const uint16_t *const kb = p.k + hk * p.shk + (long long)first * p.ldk;
    const uint16_t *const vb = p.v + hk * p.shv + (long long)first * p.ldv;
    // DMA of tile i into stage st; past the last from a zero-sized buffer
    auto issue = [&](int i, int st) {
        const int rows = i < i1 ? min(n - i * kB, kB) : 0;
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
            (void *)(kb + (long long)i * kB * p.ldk), 0, rows > 0 ? (int)((rows - 1) * p.ldk * 2) + kD * 2 : 0, kBufferFlags);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
            (void *)(vb + (long long)i * kB * p.ldv), 0, rows > 0 ? (int)((rows - 1) * p.ldv * 2) + kD * 2 : 0, kBufferFlags);
        // 1 KB block x = key rows 2 x + hi; chunk c of row r lies at c ^ (r % 16) (K), c ^ 4 (r % 4) (V).  The offsets come from
        // an opaque copy of the lane id at every tile: hoisted out of the loop they take registers that the tiles need.
        int ln = lane;
        __asm__ volatile("" : "+v"(ln));
        const int r0 = 8 * wave + (ln >> 5), k2 = (int)(p.ldk * 2), v2 = (int)(p.ldv * 2);
        const int rk0 = r0 * k2, rv0 = r0 * v2;
        int8_t *s = smem + st * kStage + 4 * wave * 1024;
#pragma unroll
        for (int x = 0; x < 4; ++x)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void *)(s + x * 1024), 16,
                                                     rk0 + 2 * x * k2 + (((ln & 31) ^ ((r0 + 2 * x) & 15)) << 4), 0, 0, 0);
#pragma unroll
        for (int x = 0; x < 4; ++x)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void *)(s + kTile + x * 1024), 16,
                                                     rv0 + 2 * x * v2 + (((ln & 31) ^ (((r0 + 2 * x) & 3) << 2)) << 4), 0, 0, 0);
    };
    // Q fragments (B operand of S^T: dims 16 s + 8 hi .. + 7 of row q0 + l % 32); rows past the sequence repeat its last
    bf16x8 qf[kD / 16];
    {
        const uint16_t *qr = p.q + (hk * kGroup + wave) * p.shq + (long long)(first + min(q0 + l32, n - 1)) * p.ldq + hi * 8;
#pragma unroll
        for (int s = 0; s < kD / 16; ++s) qf[s] = __builtin_bit_cast(bf16x8, *(const u32x4 *)(qr + s * 16));
    }
    __builtin_amdgcn_sched_barrier(0);
    issue(i0, 0);
    if (tid == 0) *odd_tile = 0;
    wait_lgkmcnt0(); // seen by every wave after the first tile's barrier
    f32x16 O[kD / 32];
#pragma unroll
    for (int dt = 0; dt < kD / 32; ++dt) O[dt] = f32x16{};
    float m = -__builtin_inff(), lsum = 0.0f;

    // V^T fragment of 32-dim tile dt, step s: keys 16 s + 4 hi .. + 3 and 16 s + 8 + 4 hi .. + 3 (the keys of P^T's accumulator
    // rows 8 s .. 8 s + 7) of dim 32 dt + l % 32
    const int vrow = 4 * hi + ((l32 & 15) >> 2);
    const int vchunk = (2 * (l32 >> 4) + ((l32 & 3) >> 1)) ^ ((vrow & 3) << 2);
    const uint32_t vbase = lds0 + kTile + vrow * (kD * 2) + (vchunk << 4) + (l32 & 1) * 8;
    // K fragment s: chunk 2 s + hi of key row l % 32, at chunk ^ (l % 16)
    const uint32_t kbase = lds0 + l32 * (kD * 2) + ((hi ^ (l32 & 15)) << 4);
    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    auto kfrag = [](uint32_t stage, int s) { return __builtin_bit_cast(bf16x8, *(lds_u32x4 *)(uintptr_t)((stage ^ (s << 5)))); };
    // (opaque: as a constant it would be put into tr_read itself, which then says nothing)
    lds_void *none = (lds_void *)smem;
    __asm__ volatile("" : "+s"(none));
    auto vfrag = [none](uint32_t stage, int s, int dt) {
        const uint32_t a = (stage ^ (dt << 6)) + s * 16 * (kD * 2);
        const s16x4 x = tr_read((lds_s16x4 *)(uintptr_t)a, none);
        const s16x4 y = tr_read((lds_s16x4 *)(uintptr_t)(a + 8 * (kD * 2)), none);
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    constexpr int kPf = 3; // operand fragments read ahead
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
        const int st = (i - i0) & 1;
        // this wave's DMA of tile i landed; after the barrier every wave's has, and nobody reads tile i - 1 any more
        wait_vmcnt<0>();
        meet();
        __builtin_amdgcn_sched_barrier(0);
        issue(i + 1, 1 - st);
        const int8_t *stage = smem + st * kStage;
        const uint32_t ks = kbase + st * kStage, vs = vbase + st * kStage;
        // ---- S^T = K Q^T: rows = keys of the tile, column = this lane's row ----
        f32x16 sc = {};
        __builtin_amdgcn_s_setprio(1);
        bf16x8 kf[kPf];
#pragma unroll
        for (int s = 0; s < kPf; ++s) kf[s] = kfrag(ks, s);
#pragma unroll
        for (int s = 0; s < kD / 16; ++s) {
            const bf16x8 a = kf[s % kPf];
            if (s + kPf < kD / 16) kf[s % kPf] = kfrag(ks, s + kPf);
            __builtin_amdgcn_sched_barrier(0);
            sc = mfma_bf16(a, qf[s], sc);
        }
        __builtin_amdgcn_s_setprio(0);
        // ---- the diagonal tile: score r of a lane is key 8 (r / 4) + 4 hi + r % 4, seen by rows from it on ----
        if (i == qb) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = 8 * (r >> 2) + 4 * hi + (r & 3) <= l32 ? sc[r] : -__builtin_inff();
        }
        // ---- online softmax in log2 units; the reference moves only when the maximum exceeds it by more than 8 ----
        float mx = -__builtin_inff();
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = __builtin_fmaxf(mx, sc[r]);
        mx = half_swap_max(mx) * p.scale_log2;
        const bool grow = mx > m + 8.0f;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
        if (grow) m = mx;
        if (__builtin_amdgcn_ballot_w64(grow)) {
#pragma unroll
            for (int dt = 0; dt < kD / 32; ++dt) O[dt] *= alpha;
            lsum *= alpha;
        }
        const float ref = m == -__builtin_inff() ? 0.0f : m; // nothing but scores of -inf yet: exp2(-inf - 0) = 0
        bf16x8 pb[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * s + 2 * e], p.scale_log2, -ref));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * s + 2 * e + 1], p.scale_log2, -ref));
                lsum += p0 + p1;
                w[e] = pack_bf16x2(p0, p1); // the matrix cores' operand type; the sum keeps the unrounded weights
            }
            pb[s] = __builtin_bit_cast(bf16x8, w);
        }
        // A value that is not finite must not reach the rows before its own (0 x inf = NaN): looked for in the diagonal tile
        // by all waves, each in its part.
        if (i == qb) {
            uint32_t odd = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const u32x4 w = *(const u32x4 *)(stage + kTile + (4 * wave + x) * 1024 + lane * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) odd |= (w[e] & 0x7f807f80u) + 0x00800080u;
            }
            if (__builtin_amdgcn_ballot_w64((odd & 0x80008000u) != 0) && lane == 0) *odd_tile = 1;
            wait_lgkmcnt0();
            meet();
            if (*odd_tile) { // the same for every wave: into the rows that give their keys a weight, then zeros in their place
                bf16x8 ind[2];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    u32x4 w = __builtin_bit_cast(u32x4, pb[s]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = ((w[e] & 0xffffu) ? 0x7f00u : 0u) | ((w[e] >> 16) ? 0x7f000000u : 0u);
                    ind[s] = __builtin_bit_cast(bf16x8, w);
                }
#pragma unroll
                for (int x = 0; x < 4 * (kD / 32); ++x) {
                    const int s = x & 1, dt = x >> 2;
                    const uint32_t sign = x & 2 ? 0x8000u : 0u;
                    u32x4 w = __builtin_bit_cast(u32x4, vfrag(vs, s, dt));
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = odd_value(w[e] & 0xffffu, sign) | (odd_value(w[e] >> 16, sign) << 16);
                    O[dt] = mfma_bf16(__builtin_bit_cast(bf16x8, w), ind[s], O[dt]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                __syncthreads();
#pragma unroll 1
                for (int x = tid; x < kTile / 4; x += kThreads) {
                    uint32_t *w = (uint32_t *)(smem + st * kStage + kTile) + x;
                    *w &= (odd_value(*w & 0xffffu, 0) ? 0u : 0xffffu) | (odd_value(*w >> 16, 0) ? 0u : 0xffff0000u);
                }
                __syncthreads();
            }
        }
        // ---- O^T += V^T P^T ----
        __builtin_amdgcn_s_setprio(1);
        bf16x8 vf[kPf];
#pragma unroll
        for (int x = 0; x < kPf; ++x) vf[x] = vfrag(vs, x >> 3, x & 7);
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const bf16x8 a = vf[x % kPf];
            if (x + kPf < 16) vf[x % kPf] = vfrag(vs, (x + kPf) >> 3, (x + kPf) & 7);
            __builtin_amdgcn_sched_barrier(0);
            O[x & 7] = mfma_bf16(a, pb[x >> 3], O[x & 7]);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    wait_vmcnt<0>(); // the last (empty) loads have written before the stages are used again
    const float ltot = half_swap_sum(lsum);
    if (parts > 1) { // the state, left for pk_merge_kernel
        const long long part = ((long long)id * p.chunks + chunk) * p.HK + hk;
        const int row = wave * kB + l32;
#pragma unroll
        for (int dt = 0; dt < kD / 32; ++dt)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                p.part_o[(part * 64 + (dt * 4 + r4) * 2 + hi) * kRows + row] =
                    float4{O[dt][4 * r4], O[dt][4 * r4 + 1], O[dt][4 * r4 + 2], O[dt][4 * r4 + 3]};
        if (hi == 0) p.part_ml[part * kRows + row] = float2{m, ltot};
        return;
    }
    // ---- normalise (a row whose scores are all -inf has no softmax: 0 / 0), stage in LDS, write 16-byte row pieces ----
    const float inv = 1.0f / ltot;
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < kD / 32; ++dt)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = dt * 32 + 8 * r4 + 4 * hi;
            u32x2 w;
            w[0] = pack_bf16x2(O[dt][4 * r4] * inv, O[dt][4 * r4 + 1] * inv);
            w[1] = pack_bf16x2(O[dt][4 * r4 + 2] * inv, O[dt][4 * r4 + 3] * inv);
            *(u32x2 *)(smem + (wave * kB + l32) * (kD * 2) + (((d >> 3) ^ l32) << 4) + (d & 4) * 2) = w;
        }
    __syncthreads();
#pragma unroll 2
    for (int x = tid; x < kGroup * kB * 32; x += kThreads) {
        const int rr = x >> 5, ch = x & 31, t = q0 + rr % kB;
        if (t < n)
            *(u32x4 *)(p.o + (long long)(hk * kGroup + rr / kB) * p.sho + (long long)(first + t) * p.ldo + ch * 8) =
                *(const u32x4 *)(smem + rr * (kD * 2) + ((ch ^ (rr & 31)) << 4));
    }
}

// The partial states of a divided block joined: with M = max_c m_c, w_c = 2^(m_c - M), o = (sum w_c O_c) / (sum w_c l_c); a
// thread has four dims of a row, for four rows.
__global__ __launch_bounds__(256) void pk_merge_kernel(PackedParams p) {
    constexpr int K = 4, kBlocks = 64 * kRows / (256 * K); // workgroups of a block and head
    const int x0 = (blockIdx.x % kBlocks * 4 + (threadIdx.x >> 6)) * (64 * K) + (threadIdx.x & 63);
    const int hk = blockIdx.x / kBlocks % p.HK, id = blockIdx.x / kBlocks / p.HK;
    int b, qb;
    if (!find_block(p.rows, id, b, qb)) return;
    const int parts = p.parts(qb + 1);
    if (parts < 2) return; // its workgroup wrote it
    const int first = p.rows.at(b), n = p.rows.rows(b);
    float mx[K], l[K];
    float4 acc[K];
#pragma unroll
    for (int k = 0; k < K; ++k) mx[k] = -__builtin_inff(), l[k] = 0.0f, acc[k] = float4{0.0f, 0.0f, 0.0f, 0.0f};
    // no part has a score above -inf: weights 1 on zeros
    auto weight = [](float m, float top) { return top == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - top); };
    constexpr int kBatch = 2; // parts whose loads are in flight together
    for (int c0 = 0; c0 < parts; c0 += kBatch) {
        float2 ml[K][kBatch];
        float4 o[K][kBatch];
#pragma unroll
        for (int y = 0; y < kBatch; ++y) {
            const long long at = ((long long)id * p.chunks + min(c0 + y, parts - 1)) * p.HK + hk;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int x = x0 + k * 64;
                ml[k][y] = p.part_ml[at * kRows + x % kRows];
                o[k][y] = p.part_o[at * 64 * kRows + x];
                if (c0 + y >= parts) ml[k][y] = float2{-__builtin_inff(), 0.0f}, o[k][y] = float4{0.0f, 0.0f, 0.0f, 0.0f};
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
            for (int y = 0; y < kBatch; ++y) {
                const float v = weight(ml[k][y].x, top);
                l[k] += v * ml[k][y].y;
                acc[k].x += v * o[k][y].x;
                acc[k].y += v * o[k][y].y;
                acc[k].z += v * o[k][y].z;
                acc[k].w += v * o[k][y].w;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int x = x0 + k * 64, row = x % kRows, four = x / kRows, t = qb * kB + row % kB;
        if (t >= n) continue;
        const float inv = 1.0f / l[k];
        const u32x2 w = {pack_bf16x2(acc[k].x * inv, acc[k].y * inv), pack_bf16x2(acc[k].z * inv, acc[k].w * inv)};
        *(u32x2 *)(p.o + (long long)(hk * kGroup + row / kB) * p.sho + (long long)(first + t) * p.ldo + four * 4) = w;
    }
}

// ---- host side ----

constexpr int kCus = 256; // CUs of the chip

struct Plan {
    int chunk, chunks;
    long long units, states; // blocks (of all sequences and of the rows of none), partial rows
};

Plan plan(long long B, long long T, long long HK, int longest) {
    Plan pl{};
    // blocks: at most (n + 31) / 32 and n of each sequence, and of the rows of none
    const long long most = (T + 31 * B + 31) / 32;
    pl.units = most < T ? most : T;
    pl.chunk = 1 << 30, pl.chunks = 1;
    // Unknown: as if all had as many rows (4 heads: 4 x 400 25.7 / 22.1 us with T as the guess / so, 5 x 300 26.3 / 19.0, 3 x 600
    // 32.2 / 29.1; 1500 + 375 47.5 / 56.6, which the hint mends: 50).
    const long long guess = longest > 0 ? longest : B > 0 ? (T + B - 1) / B : T, hint = guess < T ? guess : T;
    const long long nb = (hint + kB - 1) / kB;
    // Too few blocks to fill the chip, and long ones: each is divided into up to three chunks, so that the longest does not
    // run alone in the end, against 64 KB of state a wave, written and read.  Undivided / divided, us:
    //   4 heads, 1 x 700 30 / 27, 1000 40 / 34, 1500 56 / 47, 2048 73.6 / 60.5, 2400 86 / 74, 2500 90 / 85, 2600 94 / 97, 3000
    //   110 / 118: as long as the divided blocks' workgroups are about two a CU (units x HK up to 320; 1 head, 10000 rows 328 / 249);
    //   2 x 768 33.9 / 36.2, 900 38.5 / 40.6, 1000 41.7 / 47.1, 1500 61 / 75, but 1 head 5 x 1000 40 / 36, 6 x 1000 40.5 / 38.3,
    //   6 x 1500 58 / 57, 8 x 1000 42 / 46, 3 heads 2 x 1000 40 / 38, 4 heads 1000 + 500 40.7 / 36.5, 1500 + 1125 59 / 64: where all
    //   rows and heads are those of up to six of the longest sequence.
    // Chunks of 16 / 24 / 32 tiles: 1 x 1000 33.8 / 39.9 / 40.3, 1 x 2048 82.0 / 61.1 / 69.8.
    if (pl.units * HK <= kCus + kCus / 4 && T * HK <= 6 * hint && nb >= 24) {
        pl.chunk = (int)((3 * nb / 8 + 7) / 8 * 8);
        pl.chunks = (int)((nb + pl.chunk - 1) / pl.chunk);
        pl.states = pl.units * pl.chunks * HK * kRows;
    }
    return pl;
}
long long state_bytes(const Plan &pl) { return pl.states * (kD * 4 + 8); }

}  // namespace

extern "C" int mica_attention_packed(const void *q, long long shq, long long ldq, const void *k, long long shk, long long ldk,
                                     const void *v, long long shv, long long ldv, void *o, long long sho, long long ldo,
                                     const int *starts, int B, int T, int HQ, int HK, int head_dim, float scale, int fill,
                                     int longest, void *workspace, long long workspace_bytes, mica_stream_t stream) {
    if (head_dim != kD || HK <= 0 || HK > (1 << 20) || HQ != HK * kGroup || B < 0 || T < 0) return MICA_MISS_SHAPE;
    if (!(scale > 0.0f) || !(scale * kLog2e < __builtin_inff())) return MICA_MISS_ARG;
    if (T == 0 || (B == 0 && !fill)) return 0;
    if (!q || !k || !v || !o || !starts) return MICA_MISS_ARG;
    if (T == 1) ldk = ldv = kD; // (never used; the range check of a tile counts on it)
    for (long long x : {shq, ldq, shk, ldk, shv, ldv, sho, ldo})
        if (x < 0 || x % 8) return MICA_MISS_STRIDE;
    for (long long x : {ldk, ldv}) {
        if (x < kD) return MICA_MISS_STRIDE;
        if (x * 2 * kB >= (1LL << 31)) return MICA_MISS_RANGE; // a tile's rows within a buffer's range
    }
    if (!mica_aligned16(q) || !mica_aligned16(k) || !mica_aligned16(v) || !mica_aligned16(o) || ((uintptr_t)starts & 3))
        return MICA_MISS_ALIGN;
    const Plan pl = plan(B, T, HK, longest);
    if (pl.units * HK * pl.chunks >= (1 << 24)) return MICA_MISS_RANGE; // (a grid of 2^32 work-items wraps round)
    if (pl.states && (!workspace || !mica_aligned16(workspace) || workspace_bytes < state_bytes(pl))) return MICA_MISS_ARG;
    PackedParams p{};
    p.q = (const uint16_t *)q; p.shq = shq; p.ldq = ldq;
    p.k = (const uint16_t *)k; p.shk = shk; p.ldk = ldk;
    p.v = (const uint16_t *)v; p.shv = shv; p.ldv = ldv;
    p.o = (uint16_t *)o; p.sho = sho; p.ldo = ldo;
    p.rows = Ragged{starts, B, T};
    p.HK = HK; p.fill = fill;
    p.scale_log2 = scale * kLog2e;
    p.chunk = pl.chunk, p.chunks = pl.chunks;
    p.part_o = (float4 *)workspace;
    p.part_ml = (float2 *)((char *)workspace + pl.states * kD * 4);
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(pk_fwd_kernel, dim3((unsigned)(pl.units * HK * pl.chunks)), dim3(kThreads), 0, st, p);
    if (const int rc = mica_err(hipGetLastError())) return rc;
    if (pl.states == 0) return 0;
    hipLaunchKernelGGL(pk_merge_kernel, dim3((unsigned)(pl.units * HK * (64 * kRows / 1024))), dim3(256), 0, st, p);
    return mica_err(hipGetLastError());
}

extern "C" long long mica_attention_packed_workspace_bytes(int B, int T, int HK, int longest) {
    if (B < 0 || T < 0 || HK <= 0 || HK > (1 << 20)) return -1;
    return state_bytes(plan(B, T, HK, longest));
}
