// Attention of each sequence's newest rows over the paged 8-bit cache (mica_attention_paged), head dim 256, 4 query heads per
// key/value head; paged.h has the cache's layout.
//
//   o[t, h] = sum_{u <= p} softmax_u(scale q[t, h] . key_u[h / 4]) value_u[h / 4],   p = len - n + i  for row i of n
//   key_u = s_K q_u for a block's scale s_K and int8 q_u, bf16 in the rest; values likewise; zeros where p < 0
//
// Work split: a workgroup takes one key/value head and a block of 8 R rows of one sequence, 32 R (row, head) pairs.  Each of
// its R x D waves holds 32 of them: it computes S^T = K Q^T (32 keys x 32 pairs, v_mfma_f32_32x32x16_bf16), the online softmax
// of its pairs (a lane holds 16 of a pair's 32 scores, lane l ^ 32 the others) and 256 / D dims of O^T += V^T P^T.
//
// The products are of whole numbers: int8 values are exact in bf16, so a block's key scale multiplies the scores and its value
// scale the weights, once each, and nothing is rounded that a bf16 cache would not round.
//
// Data movement: a page's 16 KB of a head are 16 pieces of 1 KB, 16 bytes a lane, in the order of the matrix cores' operands.
// Every wave loads its share of the next page into registers while this one is computed, widens it to bf16 once for all waves
// and writes it to one of two LDS stages, from which every operand is one contiguous 16-byte read a lane.
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
};

// four int8 as two packed bf16 pairs
MICA_DEVICE u32x2 widen4(uint32_t w) {
    u32x2 x;
    x[0] = pack_bf16x2((float)(int8_t)w, (float)(int8_t)(w >> 8));
    x[1] = pack_bf16x2((float)(int8_t)(w >> 16), (float)((int32_t)w >> 24));
    return x;
}

template <int R, int D>
__global__ __launch_bounds__(64 * R * D, 2) void pg_fwd_kernel(PagedParams p) {
    constexpr int kWaves = R * D, kThreads = 64 * kWaves;
    constexpr int NB = 8 * R;               // rows of the workgroup
    constexpr int NDT = kD / 32 / D;        // 32-dim tiles of O a wave holds
    constexpr int kOwn = 16 / kWaves;       // pieces of a page a wave brings
    constexpr int kSmem = R * 32 * kD * 2 > 2 * kStage ? R * 32 * kD * 2 : 2 * kStage; // the stages; the output, in the end
    __shared__ __attribute__((aligned(1024))) int8_t smem[kSmem + 16];
    int *const odd_rest = (int *)(smem + kSmem); // whether the rest holds a value that is not finite

    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rb = wave / D, dt0 = (wave % D) * NDT;
    const int hk = blockIdx.x % p.c.HK, id = blockIdx.x / p.c.HK;
    int b, qb;
    if (!find_unit(p.rows.B, [&](int i) { return (p.rows.rows(i) + NB - 1) / NB; }, id, b, qb)) {
        if (p.fill) {
            const int i0 = (id - b) * NB, before = p.rows.at(0), behind = p.rows.at(p.rows.B);
            for (int x = tid; x < NB * kGroup * (kD / 8); x += kThreads) {
                const int i = i0 + x / (kGroup * (kD / 8)), c = x % (kGroup * (kD / 8));
                const long long t = i < before ? i : (long long)behind + i - before;
                if (t < p.rows.T)
                    *(u32x4 *)(p.o + (hk * kGroup + c / (kD / 8)) * p.sho + t * p.ldo + c % (kD / 8) * 8) = u32x4{0u, 0u, 0u, 0u};
            }
        }
        return;
    }
    b = __builtin_amdgcn_readfirstlane(b), qb = __builtin_amdgcn_readfirstlane(qb);
    const int first = p.rows.at(b), n = p.rows.rows(b), len = p.c.len(b), slot = p.c.slot(b);
    const int q0 = qb * NB, from = len - n;                  // the block's first row; the position of the sequence's
    const int last = from + min(n, q0 + NB) - 1;             // position of the block's last row
    const int tiles = last < 0 ? 0 : last / kBK + 1, whole = len / kBK;

    // this lane's pair: a row and a query head
    const int pair = rb * 32 + l32, head = hk * kGroup + pair / NB, t = q0 + pair % NB, pos = from + t;
    // Q fragments (B operand of S^T): step 2 c + e takes dims 32 c + 16 hi + 8 e .. + 7, as a page's bytes lie; rows past the
    // last repeat it
    bf16x8 qf[kD / 16];
    {
        const uint16_t *qr = p.q + head * p.shq + (long long)(first + min(t, n - 1)) * p.ldq + hi * 16;
#pragma unroll
        for (int s = 0; s < kD / 16; ++s) qf[s] = __builtin_bit_cast(bf16x8, *(const u32x4 *)(qr + (s >> 1) * 32 + (s & 1) * 8));
    }
    // Pieces 0 .. 7 of a page are keys (32 dims of each token), 8 .. 15 values (32 dims' rows); this wave brings kOwn of them.
    u32x4 raw[kOwn];
    float sk = 0.0f, sv = 0.0f, sk_next = 0.0f, sv_next = 0.0f;  // the tile's scales
    auto fetch = [&](int i) { // tile i's pieces into registers, and its scales
        if (i >= tiles) return;
        if (i >= whole) { // (the rest: see below)
            const bool bad = slot < 0;
            sk_next = sv_next = bad ? __builtin_nanf("") : 1.0f;
            return;
        }
        const int page = p.c.page(b, i);
        // (a block without a page: NaN, for the rows that see it)
        sk_next = page >= 0 ? p.c.scales[p.c.index(page, 0, hk)] : __builtin_nanf("");
        sv_next = page >= 0 ? p.c.scales[p.c.index(page, 1, hk)] : __builtin_nanf("");
#pragma unroll
        for (int x = 0; x < kOwn; ++x) {
            const int piece = wave * kOwn + x;
            raw[x] = page >= 0 ? *(const u32x4 *)(p.c.block(page, piece >> 3, hk) + (piece & 7) * 1024 + l32 * 32 + hi * 16)
                               : u32x4{0u, 0u, 0u, 0u};
        }
    };
    // Tile i into LDS stage st: piece x becomes two operands of 64 lanes x 16 bytes.  Keys: bytes 8 e .. 8 e + 7 are step
    // 2 c + e's; values: fours s and s + 2 are step s's (tokens 16 s + 4 hi .. + 3 and 8 more on: P^T's accumulator rows).
    auto stage_in = [&](int i, int st) {
        int8_t *s = smem + st * kStage + lane * 16;
        if (i < whole) {
#pragma unroll
            for (int x = 0; x < kOwn; ++x) {
                const int piece = wave * kOwn + x;
                const u32x2 w0 = widen4(raw[x][0]), w1 = widen4(raw[x][1]), w2 = widen4(raw[x][2]), w3 = widen4(raw[x][3]);
                const bool value = piece >= 8;
                u32x4 a = {w0[0], w0[1], w1[0], w1[1]}, c = {w2[0], w2[1], w3[0], w3[1]};
                if (value) a = u32x4{w0[0], w0[1], w2[0], w2[1]}, c = u32x4{w1[0], w1[1], w3[0], w3[1]};
                *(u32x4 *)(s + piece * 2048) = a;
                *(u32x4 *)(s + piece * 2048 + 1024) = c;
            }
            return;
        }
        // The rest: bf16 rows, the same operands; zeros past its last token.
        const int have = slot < 0 ? 0 : len - whole * kBK;
        const uint16_t *kr = p.c.rest(max(slot, 0), 0, hk), *vr = p.c.rest(max(slot, 0), 1, hk);
        uint32_t odd = 0;
#pragma unroll 1
        for (int x = 0; x < kOwn; ++x) {
            const int piece = wave * kOwn + x;
            u32x4 a = {}, c = {};
            if (piece < 8) {
                if (l32 < have) {
                    const u32x4 *src = (const u32x4 *)(kr + l32 * kD + piece * 32 + hi * 16);
                    a = src[0], c = src[1];
                }
            } else {
                const uint16_t *src = vr + (piece - 8) * 32 + l32;
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) { // step e / 8, its token e % 8
                    const int token = 16 * (e >> 3) + 8 * ((e >> 2) & 1) + 4 * hi + (e & 3);
                    w[e] = token < have ? src[token * kD] : 0u;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = w[2 * e] | w[2 * e + 1] << 16, c[e] = w[8 + 2 * e] | w[9 + 2 * e] << 16;
#pragma unroll
                for (int e = 0; e < 4; ++e) odd |= ((a[e] & 0x7f807f80u) + 0x00800080u) | ((c[e] & 0x7f807f80u) + 0x00800080u);
            }
            *(u32x4 *)(s + piece * 2048) = a;
            *(u32x4 *)(s + piece * 2048 + 1024) = c;
        }
        if (__builtin_amdgcn_ballot_w64((odd & 0x80008000u) != 0) && lane == 0) *odd_rest = 1;
    };
    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    const uint32_t base = (uint32_t)(uintptr_t)(lds_void *)smem + lane * 16;
    auto kfrag = [](uint32_t a, int s) { return __builtin_bit_cast(bf16x8, *(lds_u32x4 *)(uintptr_t)(a + s * 1024)); };
    auto vfrag = [&](uint32_t a, int s, int dt) {
        return __builtin_bit_cast(bf16x8, *(lds_u32x4 *)(uintptr_t)(a + kTile + (dt0 + dt) * 2048 + s * 1024));
    };

    f32x16 O[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) O[dt] = f32x16{};
    float m = -__builtin_inff(), lsum = 0.0f;
    if (tid == 0) *odd_rest = 0;
    __syncthreads();
    fetch(0);
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
        const int st = i & 1;
        stage_in(i, st);
        sk = sk_next, sv = sv_next;
        fetch(i + 1);
        // every wave's pieces are there; nobody reads the other stage (tile i - 1) any more when tile i + 1 is written to it
        wait_lgkmcnt0();
        meet();
        const uint32_t at = base + st * kStage;
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
        const float scale = p.scale_log2 * sk;
        // ---- keys past a row's position: score -inf (score r of a lane is key 8 (r / 4) + 4 hi + r % 4) ----
        const bool masked = (i + 1) * kBK - 1 > from + q0;
        if (masked) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = i * kBK + 8 * (r >> 2) + 4 * hi + (r & 3) <= pos ? sc[r] : -__builtin_inff();
        }
        // ---- online softmax in log2 units; the reference moves only when the maximum exceeds it by more than 8 ----
        float mx = -__builtin_inff();
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = __builtin_fmaxf(mx, sc[r]);
        mx = half_swap_max(mx) * scale;
        const bool grow = mx > m + 8.0f;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
        if (grow) m = mx;
        if (__builtin_amdgcn_ballot_w64(grow)) {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) O[dt] *= alpha;
            lsum *= alpha;
        }
        const float ref = m == -__builtin_inff() ? 0.0f : m; // a row that has seen nothing yet: exp2(-inf - 0) = 0
        float pr[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            pr[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], scale, -ref));
            if (masked) pr[r] = i * kBK + 8 * (r >> 2) + 4 * hi + (r & 3) <= pos ? pr[r] : 0.0f; // (a scale may be NaN)
        }
        bf16x8 pb[2];
        const bool odd_scale = !(sv < __builtin_inff());
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p0 = pr[8 * s + 2 * e], p1 = pr[8 * s + 2 * e + 1];
                lsum += p0 + p1;
                float v0 = p0 * sv, v1 = p1 * sv;
                if (odd_scale) v0 = p0 == 0.0f ? 0.0f : v0, v1 = p1 == 0.0f ? 0.0f : v1;
                w[e] = pack_bf16x2(v0, v1); // the matrix cores' operand type; the sum keeps the unrounded weights
            }
            pb[s] = __builtin_bit_cast(bf16x8, w);
        }
        // A value of the rest that is not finite must not reach the rows before its own (0 x inf = NaN): into the rows that give
        // its key a weight, then zeros in its place.
        if (i >= whole && *odd_rest) {
            bf16x8 ind[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                u32x4 w = __builtin_bit_cast(u32x4, pb[s]);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = ((w[e] & 0xffffu) ? 0x7f00u : 0u) | ((w[e] >> 16) ? 0x7f000000u : 0u);
                ind[s] = __builtin_bit_cast(bf16x8, w);
            }
#pragma unroll
            for (int x = 0; x < 4 * NDT; ++x) {
                const int s = x & 1, dt = x >> 2;
                const uint32_t sign = x & 2 ? 0x8000u : 0u;
                u32x4 w = __builtin_bit_cast(u32x4, vfrag(at, s, dt));
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
        // ---- O^T += V^T P^T ----
        constexpr int kPv = kPf < 2 * NDT ? kPf : 2 * NDT;
        __builtin_amdgcn_s_setprio(1);
        bf16x8 vf[kPv];
#pragma unroll
        for (int x = 0; x < kPv; ++x) vf[x] = vfrag(at, x / NDT, x % NDT);
#pragma unroll
        for (int x = 0; x < 2 * NDT; ++x) {
            const bf16x8 a = vf[x % kPv];
            if (x + kPv < 2 * NDT) vf[x % kPv] = vfrag(at, (x + kPv) / NDT, (x + kPv) % NDT);
            __builtin_amdgcn_sched_barrier(0);
            O[x % NDT] = mfma_bf16(a, pb[x / NDT], O[x % NDT]);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    // ---- normalise (a row whose scores are all -inf has no softmax: 0 / 0; one that sees no key: zeros), stage, write ----
    const float inv = pos < 0 ? 0.0f : 1.0f / half_swap_sum(lsum);
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = (dt0 + dt) * 32 + 8 * r4 + 4 * hi;
            const f32x16 x = O[dt];
            u32x2 w;
            w[0] = pack_bf16x2(x[4 * r4] * inv, x[4 * r4 + 1] * inv);
            w[1] = pack_bf16x2(x[4 * r4 + 2] * inv, x[4 * r4 + 3] * inv);
            *(u32x2 *)(smem + pair * (kD * 2) + (((d >> 3) ^ l32) << 4) + (d & 4) * 2) = w;
        }
    __syncthreads();
#pragma unroll 2
    for (int x = tid; x < 32 * R * 32; x += kThreads) {
        const int rr = x >> 5, ch = x & 31, tt = q0 + rr % NB;
        if (tt < n)
            *(u32x4 *)(p.o + (long long)(hk * kGroup + rr / NB) * p.sho + (long long)(first + tt) * p.ldo + ch * 8) =
                *(const u32x4 *)(smem + rr * (kD * 2) + ((ch ^ (rr & 31)) << 4));
    }
}

}  // namespace

extern "C" int mica_attention_paged(const void *q, long long shq, long long ldq, void *o, long long sho, long long ldo,
                                    const int *starts, int B, int T, int HQ, const void *data, const float *scales,
                                    const void *recent, int pages, int n_slots, int HK, int head_dim, const int *table,
                                    long long ldt, int width, const int *lens, const int *slots, float scale, int fill,
                                    int longest, void *workspace, long long workspace_bytes, mica_stream_t stream) {
    if (B < 0 || T < 0) return MICA_MISS_SHAPE;
    if (!(scale > 0.0f) || !(scale < __builtin_inff())) return MICA_MISS_ARG;
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
    p.q = (const uint16_t *)q; p.shq = shq; p.ldq = ldq;
    p.o = (uint16_t *)o; p.sho = sho; p.ldo = ldo;
    p.rows = Ragged{starts, B, T};
    p.fill = fill;
    p.scale_log2 = scale * 1.44269504088896341f;
    const int hint = longest > 0 && longest < T ? longest : T;
    const int R = hint <= 8 ? 1 : hint <= 16 ? 2 : 4, nb = 8 * R;
    const long long most = ((long long)T + (nb - 1ll) * B + nb - 1) / nb, units = most < T ? most : T, wgs = units * HK;
    if (wgs >= (1 << 24)) return MICA_MISS_RANGE; // (a grid of 2^32 work-items wraps round)
    hipStream_t st = (hipStream_t)stream;
    if (R == 1) hipLaunchKernelGGL((pg_fwd_kernel<1, 4>), dim3((unsigned)wgs), dim3(256), 0, st, p);
    else if (R == 2) hipLaunchKernelGGL((pg_fwd_kernel<2, 2>), dim3((unsigned)wgs), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((pg_fwd_kernel<4, 1>), dim3((unsigned)wgs), dim3(256), 0, st, p);
    return mica_err(hipGetLastError());
}

extern "C" long long mica_attention_paged_workspace_bytes(int B, int T, int HK, int width, int longest) {
    if (B < 0 || T < 0 || HK <= 0 || width < 0) return -1;
    return 0;
}
