// Attention of new tokens over kept keys on gfx950, head dim 256, 4 query heads per key/value head: a tree of
// candidate tokens over a cache (mica_attention_tree) and causal attention within a sliding window and over a few
// first tokens (mica_attention_window).
//
//   o[i, h] = sum_{u in S(i)} softmax_u(scale q[i, h] . k[u, h / 4]) v[u, h / 4];   zeros where S(i) is empty, NaN where
//   all its scores are -inf
//   tree:    S(i) = the sequence's first cache_len cached keys and the new keys j whose bit is set in node i's words
//            (a node without any bit is absent and sees nothing)
//   window:  S(i) = { u : u <= p and (u > p - window or u < sinks) },  p = position of query i
//
// Work split: a workgroup takes one (sequence, key/value head), a block of 8 R query positions, i.e. 32 R rows (position,
// head), and a run of 32-key tiles.  Each of its R x D waves holds 32 rows: it computes S^T = K Q^T (32 keys x 32 rows,
// v_mfma_f32_32x32x16_bf16), the online softmax of its rows (a lane holds 16 of a row's 32 scores, its partner l ^ 32
// the others) and 256 / D dims of O^T += V^T P^T.  With few rows, D > 1 waves share a row block: they repeat its scores
// (cheap beside the tile's memory time) and divide the dims of O.
//
// Data movement: K and V tiles of 32 rows come by LDS DMA into two stages in turn, 16-byte chunks XOR-swizzled by row,
// rows past the last key as zeros (the buffer's range check).  K fragments are 16-byte reads; V is kept as it lies in
// memory and its V^T fragments are transposing reads (ds_read_b64_tr_b16: 16 lanes fetch 4 keys x 16 dims and each gets
// the 4 keys of one dim), so no pass over V comes before.
//
// Up to 64 query positions, one row block takes them all, and the key tiles of all sequences, one after the other, are
// divided evenly over the chip's workgroups (STREAM): a workgroup may end one sequence and begin the next, so
// key counts that differ, or sequences that do not divide the chip, leave no CU idle.  In that row of tiles each sequence
// has a few empty ones before its own, for the time its beginning takes.  Many or short sequences are not divided: a
// workgroup each.  More positions take a workgroup for each block, their tiles divided into chunks where that leaves too
// few.  ca_merge_kernel joins the partial softmax states (fp32) of what was divided.
#include "attn_common.h"

#include <algorithm>

namespace {

constexpr int kD = 256;                    // head dim
constexpr int kGroup = 4;                  // query heads per key/value head
constexpr int kBK = 32;                    // keys per tile
constexpr int kTile = kBK * kD * 2;        // 16 KB of K or V
constexpr int kStage = 2 * kTile;
constexpr int kMaxNodes = 512;             // nodes of a tree
constexpr int kCus = 256;                  // CUs of the chip

struct CaParams {
    const uint16_t *q; long long sbq, shq, ldq;     // head h of row t of sequence b: q + b sbq + h shq + t ldq
    const uint16_t *k; long long sbk, shk, ldk;     // the new keys (tree), all keys (window)
    const uint16_t *v; long long sbv, shv, ldv;
    const uint16_t *kc; long long sbkc, shkc, ldkc; // the cache (tree)
    const uint16_t *vc; long long sbvc, shvc, ldvc;
    uint16_t *o; long long sbo, sho, ldo;
    const int *len;                                 // [B] cached keys (tree) or keys (window), or null: cap
    const uint32_t *tree; long long sbt;            // words [N][tw] of a sequence, sbt words apart (0: one tree for all)
    int tw;
    int B, Sq, cap, HK;
    int window, sinks;
    float scale_log2;                               // softmax scale x log2(e)
    int nqb, gq, chunk, nchunk;                     // query blocks, in groups of gq; tiles a workgroup, chunks a sequence
    int runs, dense, least, begin;                  // STREAM: see Plan
    float *part_o;                                  // partial O, a wave's accumulators 64 lanes x 16 bytes at a time
    float2 *part_ml;                                // partial (m, l) of each row
};

// a sequence's key count
MICA_DEVICE int key_count(const CaParams &p, int b) { return p.len ? min(max(p.len[b], 0), p.cap) : p.cap; }

// The key tiles of a query block, in the order they are walked.  tree: the cache's, then the new keys'.  window: the
// sinks' tiles below the window, then the window's.
template <bool TREE>
struct Tiles {
    int n, n0, skip; // tiles; of them cached (tree) or before the window (window); tiles skipped after those (window)
    int end;         // the new keys (tree); the keys up to the block's last position (window)
    MICA_DEVICE Tiles(const CaParams &p, int keys, int q0, int rows) {
        if constexpr (TREE) {
            n0 = (keys + kBK - 1) / kBK;
            n = n0 + (p.Sq + kBK - 1) / kBK;
            skip = 0, end = p.Sq;
        } else {
            const int first = keys - p.Sq + q0, last = first + rows - 1; // positions of the block's queries
            end = max(last + 1, 0);
            if (last < 0) { // no key: one tile that nothing is read for, so that the zeros are written
                n = 1, n0 = skip = 0;
                return;
            }
            const int w0 = max(max(first, 0) - (p.window - 1), 0) / kBK;
            n0 = min((min(p.sinks, last + 1) + kBK - 1) / kBK, w0);
            skip = w0 - n0;
            n = n0 + last / kBK - w0 + 1;
        }
    }
    MICA_DEVICE int tile(int i) const { return i < n0 ? i : i + skip; } // window: the key tile's index
};

// How STREAM divides the tiles: those of all sequences, one after the other, into runs, and a workgroup for each run and
// head.  Workgroups next to each other take the heads of one run: their rows lie side by side in memory (with the heads
// one after the other instead, 64 single tokens with a window of 4096 took 201 us and not 194).  All lanes of a wave call
// and get the same; a lane reads every 64th sequence's count.
template <bool TREE>
struct Stream {
    int total, per; // tiles of a head, tiles of a run, p.begin for each sequence's beginning among them
    int x, sum;     // this lane's sequence of 64 (the first 64 at the end): its tiles, those up to and with it
    int count;      // and its keys
    MICA_DEVICE static int of(const CaParams &p, int keys) { return Tiles<TREE>(p, keys, 0, p.Sq).n + p.begin; }
    // a wave's running sums
    MICA_DEVICE static int scan(int x) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(x, d, 64);
            x += (int)(threadIdx.x & 63) >= d ? y : 0;
        }
        return x;
    }
    MICA_DEVICE void take(const CaParams &p, int base) {
        const int b = base + (int)(threadIdx.x & 63);
        count = b < p.B ? key_count(p, b) : 0;
        x = b < p.B ? of(p, count) : 0;
        sum = scan(x);
    }
    MICA_DEVICE Stream(const CaParams &p) {
        if (p.len == nullptr) {
            count = p.cap;
            x = of(p, count);
            total = p.B * x;
        } else {
            total = 0;
            for (int base = (p.B - 1) & ~63; base >= 0; base -= 64) { // (the first 64 last: they are kept)
                take(p, base);
                total += __builtin_amdgcn_readlane(sum, 63);
            }
        }
        per = (total + p.runs - 1) / p.runs;
        const int half = max(p.runs / 2, 1);
        if (per < p.dense) per = (total + half - 1) / half;
        per = max(per, (long long)total * p.HK <= kCus ? p.least : 4);
    }
    // the sequence, its keys and its tile at `at` (below total)
    MICA_DEVICE void find(const CaParams &p, int at, int &b, int &keys, int &tile) {
        if (p.len == nullptr) {
            b = at / x, tile = at % x, keys = count;
            return;
        }
        for (int base = 0, before = 0;; base += 64) {
            if (base) take(p, base);
            const unsigned long long past = __builtin_amdgcn_ballot_w64(before + sum > at);
            if (past) {
                const int l = __builtin_ctzll(past);
                b = base + l, keys = __builtin_amdgcn_readlane(count, l);
                tile = at - before - __builtin_amdgcn_readlane(sum - x, l);
                return;
            }
            before += __builtin_amdgcn_readlane(sum, 63);
        }
    }
    // the first of sequence b's tiles
    MICA_DEVICE int first(const CaParams &p, int b) {
        if (p.len == nullptr) return b * x;
        int before = 0;
        for (int base = 0; base < b / 64 * 64; base += 64) {
            if (base) take(p, base);
            before += __builtin_amdgcn_readlane(sum, 63);
        }
        if (b >= 64) take(p, b / 64 * 64);
        return before + __builtin_amdgcn_readlane(sum - x, b % 64);
    }
};

// A V value (bf16 code) that is not finite as the largest finite value of its sign, NaN with the given sign (0 or 0x8000);
// 0 for a finite one.  Times 2^127 and summed by the matrix cores these give +-inf, and, with both signs, NaN.
MICA_DEVICE uint32_t odd_value(uint32_t h, uint32_t nan_sign) {
    if ((h & 0x7f80u) != 0x7f80u) return 0u;
    return 0x7f7fu | ((h & 0x7fu) ? nan_sign : (h & 0x8000u));
}

// A workgroup barrier that waits for nothing else; no access to memory moves across it.
MICA_DEVICE void meet() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
// A transposing read.  The compiler knows nothing of what the DMA in flight writes, and would let every one of these reads
// wait for all of it, the next tile's too.  `w`, which nothing is accessed through, says that the read meets no unknown
// store; the waits are the loop's own.  (16 x 64 nodes after 4000 keys 97.9 -> 94.5 us, 2 x 32 nodes after 10000 38.3 -> 36.)
MICA_DEVICE s16x4 tr_read(lds_s16x4 *p, lds_void *__restrict w) {
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
    __builtin_assume(w != nullptr);
    return x;
}

// What bounds it, and the whole call's time (at the rates of a large copy, 4.87 TB/s, and a large matrix product, 1401
// TFLOP/s): few rows, the cache's bytes: 64 single tokens with a window of 4096 take 190 us, 5.7 TB/s; 32 x 16 nodes over up
// to 4096 keys 97 us of 86.  Many rows, the matrix cores beside the softmax, with two waves a SIMD: 16384 tokens with a
// window of 2048 469 us of 368 (548 in a long run of nothing else); 64 nodes after 32768 keys 63 us of 28, of them 8 for the
// first tile and 20 for writing and joining 64 MB of partial states; 4 x 255 nodes after 2048 shared keys 59 us of 24.5.  A
// short call is two launches: 8 nodes after 500 keys 12.5 us.  (Four stages with one workgroup a CU 1 to 5 us slower, with
// eight waves 1 us; fragments read further ahead, 64 rows a wave, two chains for S^T: no faster, or slower for the registers that they spill.)
template <int R, int D, bool TREE, bool STREAM>
__global__ __launch_bounds__(64 * R * D, 2) void ca_fwd_kernel(CaParams p) {
    constexpr int kWaves = R * D, kThreads = 64 * kWaves;
    constexpr int NB = 8 * R;                 // query positions of the workgroup
    constexpr int NDT = kD / 32 / D;          // 32-dim tiles of O a wave holds
    constexpr int kBlk = 16 / kWaves;         // 1 KB DMA blocks of K, and of V, a wave issues for a tile
    constexpr int kPf = D > 1 ? 8 : 3;        // operand fragments read ahead (D = 1: more would spill)
    constexpr int kWords = TREE ? NB * (STREAM ? 2 : kMaxNodes / 32) : 0; // (STREAM: up to 64 nodes)
    constexpr int kSmem = R * 32 * kD * 2 > 2 * kStage ? R * 32 * kD * 2 : 2 * kStage; // the tiles; the output, in the end
    __shared__ __attribute__((aligned(1024))) int8_t smem[kSmem + 16 + kWords * 4];
    int *const odd_tile = (int *)(smem + kSmem); // the last tile that held a value that is not finite
    uint32_t *const words = (uint32_t *)(smem + kSmem + 16);

    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void *)smem;
    const int rb = wave / D, dt0 = (wave % D) * NDT;
    int b, hk, qb = 0, i0, keys, left = 0; // the sequence, head, query block, first tile here, keys; tiles left (STREAM)
    int blk;                         // where its partial state goes
    if (STREAM && p.runs == 0) { // a whole sequence
        hk = blockIdx.x % p.HK, b = blockIdx.x / p.HK, i0 = 0, blk = 0;
        keys = key_count(p, b);
        left = Tiles<TREE>(p, keys, 0, p.Sq).n;
    } else if constexpr (STREAM) {
        Stream<TREE> all(p);
        hk = blockIdx.x % p.HK;
        const int at = blockIdx.x / p.HK * all.per;
        if (at >= all.total) return;
        all.find(p, at, b, keys, i0);
        b = __builtin_amdgcn_readfirstlane(b), i0 = __builtin_amdgcn_readfirstlane(i0);
        keys = __builtin_amdgcn_readfirstlane(keys);
        left = __builtin_amdgcn_readfirstlane(min(all.per, all.total - at));
        const int unused = max(p.begin - i0, 0); // of the sequence's beginning
        left -= unused, i0 += unused - p.begin;
        if (left <= 0) return;
        blk = 2 * blockIdx.x;
    } else {
        // Consecutive workgroups go to the 8 XCDs in turn; the gq query blocks of a group, which read the same keys, stay
        // on one XCD, one after the other.
        // The last positions, whose windows are the fullest, come first.
        const int id = blockIdx.x, units = p.B * p.nchunk * p.HK;
        const int grp = id / (8 * p.gq) * 8 + id % 8, unit = grp % units;
        qb = p.nqb - 1 - (grp / units * p.gq + id / 8 % p.gq);
        if (qb < 0) return;
        hk = unit % p.HK, b = unit / p.HK / p.nchunk, i0 = unit / p.HK % p.nchunk * p.chunk;
        blk = unit * p.nqb + qb;
        keys = key_count(p, b);
    }
    for (;;) {
        // what depends on the lane alone is made here, from an opaque copy of its id: the compiler would make it before the
        // loop and hold it in registers that the tiles need (45 of them spilled)
        int tid = threadIdx.x;
        __asm__ volatile("" : "+v"(tid));
        const int lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
        const int q0 = qb * NB;
        const Tiles<TREE> tl(p, keys, q0, min(NB, p.Sq - q0));
        const int i1 = min(STREAM ? i0 + left : i0 + p.chunk, tl.n);
        if (!STREAM && i0 >= tl.n) return;
        const bool whole = STREAM ? i0 == 0 && i1 == tl.n : p.nchunk == 1;

        // this lane's row: a position and a query head
        const int row = rb * 32 + l32, head = hk * kGroup + row / NB, t = q0 + row % NB;
        // DMA of tile i into stage st; past i1 from a zero-sized buffer, so that every step issues as many instructions
        auto issue = [&](int i, int st) {
            const uint16_t *kb, *vb;
            long long ldk = p.ldk, ldv = p.ldv;
            int rows;
            if (TREE && i < tl.n0) {
                ldk = p.ldkc, ldv = p.ldvc;
                kb = p.kc + b * p.sbkc + hk * p.shkc + (long long)i * kBK * ldk;
                vb = p.vc + b * p.sbvc + hk * p.shvc + (long long)i * kBK * ldv;
                rows = keys - i * kBK;
            } else {
                const int j = TREE ? i - tl.n0 : tl.tile(i);
                kb = p.k + b * p.sbk + hk * p.shk + (long long)j * kBK * ldk;
                vb = p.v + b * p.sbv + hk * p.shv + (long long)j * kBK * ldv;
                rows = tl.end - j * kBK;
            }
            rows = i < i1 ? min(rows, kBK) : 0;
            const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
                (void *)kb, 0, rows > 0 ? (int)((rows - 1) * ldk * 2) + kD * 2 : 0, kBufferFlags);
            const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
                (void *)vb, 0, rows > 0 ? (int)((rows - 1) * ldv * 2) + kD * 2 : 0, kBufferFlags);
            // 1 KB block x = key rows 2 x + hi; chunk c of row r lies at c ^ (r % 16) (K), c ^ 4 (r % 4) (V).  The offsets
            // come from an opaque copy of the lane id at every tile: hoisted out of the loop they take 16 registers, and
            // what these push into scratch is then loaded back behind the DMA, which every such load waits for.
            int ln = lane;
            __asm__ volatile("" : "+v"(ln));
            const int r0 = 2 * kBlk * wave + (ln >> 5), k2 = (int)(ldk * 2), v2 = (int)(ldv * 2);
            const int rk0 = r0 * k2, rv0 = r0 * v2;
            int8_t *s = smem + st * kStage + kBlk * wave * 1024;
#pragma unroll
            for (int x = 0; x < kBlk; ++x)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void *)(s + x * 1024), 16,
                                                         rk0 + 2 * x * k2 + (((ln & 31) ^ ((r0 + 2 * x) & 15)) << 4), 0, 0, 0);
#pragma unroll
            for (int x = 0; x < kBlk; ++x)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void *)(s + kTile + x * 1024), 16,
                                                         rv0 + 2 * x * v2 + (((ln & 31) ^ (((r0 + 2 * x) & 3) << 2)) << 4), 0,
                                                         0, 0);
        };
        // The block's words and this lane's Q fragments (B operand of S^T: dims 16 s + 8 hi .. + 7 of the row) come before the
        // first tile: loads end in order.
        constexpr int kMine = (kWords + kThreads - 1) / kThreads;
        uint32_t mine[TREE ? kMine : 1];
        if constexpr (TREE) {
#pragma unroll
            for (int x = 0; x < kMine; ++x) {
                const int i = tid + x * kThreads, node = q0 + i / p.tw;
                mine[x] = i < NB * p.tw && node < p.Sq ? p.tree[b * p.sbt + (long long)node * p.tw + i % p.tw] : 0u;
            }
        }
        bf16x8 qf[kD / 16];
        {
            // (rows past the last position repeat it: they are not stored)
            const uint16_t *qr = p.q + b * p.sbq + head * p.shq + (long long)min(t, p.Sq - 1) * p.ldq + hi * 8;
#pragma unroll
            for (int s = 0; s < kD / 16; ++s) qf[s] = __builtin_bit_cast(bf16x8, *(const u32x4 *)(qr + s * 16));
        }
        __builtin_amdgcn_sched_barrier(0);
        issue(i0, 0);
        if constexpr (TREE) {
#pragma unroll
            for (int x = 0; x < kMine; ++x) {
                const int i = tid + x * kThreads, left = p.Sq - 32 * (i % p.tw); // bits past the last node do not count
                if (i < NB * p.tw) words[i] = left >= 32 ? mine[x] : left <= 0 ? 0u : mine[x] & ((1u << left) - 1u);
            }
        }
        if (tid == 0) *odd_tile = -1;
        wait_lgkmcnt0(); // seen by every wave after the first tile's barrier
        f32x16 O[NDT];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) O[dt] = f32x16{};
        float m = -__builtin_inff(), lsum = 0.0f;
        const int pos = keys - p.Sq + t; // window: this row's position

        // V^T fragment of 32-dim tile dt, step s: keys 16 s + 4 hi .. + 3 and 16 s + 8 + 4 hi .. + 3 (the keys of P^T's
        // accumulator rows 8 s .. 8 s + 7) of dim 32 dt + l % 32.  The lane's address: key row 4 hi + (l % 16) / 4, dims
        // 16 ((l / 16) % 2) + 4 (l % 4); chunk c of row r lies at c ^ 4 (r % 4), which spreads the 4 rows x 64 bytes of
        // each half of a read over all banks (c ^ 2 (r % 8) spreads all 8 rows, but a half over half of the banks: it cost 1.3
        // conflict cycles an LDS instruction, 1% of the time).
        const int vrow = 4 * hi + ((l32 & 15) >> 2);
        const int vchunk = (2 * (l32 >> 4) + ((l32 & 3) >> 1)) ^ ((vrow & 3) << 2) ^ (4 * dt0);
        const uint32_t vbase = lds0 + kTile + vrow * (kD * 2) + (vchunk << 4) + (l32 & 1) * 8;
        // K fragment s: chunk 2 s + hi of key row l % 32, at chunk ^ (l % 16).  The chunk's five bits are address bits of
        // their own in both tiles, so a fragment's address is one exclusive or away from its stage's.
        const uint32_t kbase = lds0 + l32 * (kD * 2) + ((hi ^ (l32 & 15)) << 4);
        typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
        auto kfrag = [](uint32_t stage, int s) { // stage: kbase + the stage's offset
            return __builtin_bit_cast(bf16x8, *(lds_u32x4 *)(uintptr_t)((stage ^ (s << 5))));
        };
        auto vfrag = [](uint32_t stage, int s, int dt) { // stage: vbase + the stage's offset
            const uint32_t a = (stage ^ (dt << 6)) + s * 16 * (kD * 2);
            const s16x4 x = tr_read((lds_s16x4 *)(uintptr_t)a, (lds_void *)smem);
            const s16x4 y = tr_read((lds_s16x4 *)(uintptr_t)(a + 8 * (kD * 2)), (lds_void *)smem);
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        };

#pragma unroll 1
        for (int i = i0; i < i1; ++i) {
            const int st = (i - i0) & 1;
            // this wave's DMA of tile i landed; after the barrier every wave's has, and nobody reads tile i - 1 any more
            wait_vmcnt<0>();
            meet();
            __builtin_amdgcn_sched_barrier(0);
            issue(i + 1, 1 - st);
            if constexpr (TREE && !STREAM) { // new keys that none of the block's nodes sees, as those after them (2 x 500 nodes
                                             // after 500 keys 58.4 -> 45.8 us; up to 64 nodes there are hardly any)
                if (i >= tl.n0 && !__builtin_amdgcn_ballot_w64(words[lane % NB * p.tw + (i - tl.n0)])) continue;
            }
            const int8_t *stage = smem + st * kStage;
            const uint32_t ks = kbase + st * kStage, vs = vbase + st * kStage;
            // ---- S^T = K Q^T: rows = keys of the tile, column = this lane's row; fragments read kPf steps ahead ----
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
            // ---- keys that a row does not see: score -inf, weight 0 (score r of a lane is key 8 (r / 4) + 4 hi + r % 4) ----
            bool masked = false, own = false;
            if constexpr (TREE) {
                own = i >= tl.n0;
                masked = own || (i + 1) * kBK > keys;
                if (own) {
                    const uint32_t w = words[row % NB * p.tw + (i - tl.n0)] >> (4 * hi);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        sc[r] = (w >> (8 * (r >> 2) + (r & 3))) & 1u ? sc[r] : -__builtin_inff();
                } else if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        sc[r] = i * kBK + 8 * (r >> 2) + 4 * hi + (r & 3) < keys ? sc[r] : -__builtin_inff();
                }
            } else {
                const int k0 = tl.tile(i) * kBK, first = keys - p.Sq + q0;
                // (differences of positions, which are small: a window up to the largest int would overflow taken from one)
                masked = k0 + kBK - 1 > first || (first + NB - 1 - k0 >= p.window && k0 + kBK > p.sinks);
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int key = k0 + 8 * (r >> 2) + 4 * hi + (r & 3);
                        const bool sees = key <= pos && (pos - key < p.window || key < p.sinks);
                        sc[r] = sees ? sc[r] : -__builtin_inff();
                    }
                }
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
                for (int dt = 0; dt < NDT; ++dt) O[dt] *= alpha;
                lsum *= alpha;
            }
            const float ref = m == -__builtin_inff() ? 0.0f : m; // a row that has seen nothing yet: exp2(-inf - 0) = 0
            bf16x8 pb[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * s + 2 * e], p.scale_log2, -ref));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * s + 2 * e + 1], p.scale_log2, -ref));
                    lsum += p0 + p1;
                    // the matrix cores' operand type; the sum keeps the unrounded weights.  The result is then 0.0022 of its
                    // norm off, where its own rounding to bf16 alone makes 0.0017 (as causal_gqa_attention's)
                    w[e] = pack_bf16x2(p0, p1);
                }
                pb[s] = __builtin_bit_cast(bf16x8, w);
            }
            // A value that is not finite must not reach the rows that do not see its key (0 x inf = NaN): looked for in
            // the tiles where rows see different keys, by every wave in its part of the tile (by each in all of it, 3 x 1111
            // tokens with a window of 200 took 32.1 us and not 30.5, and 2000 with one of 100 21.4 and not 19.4).  (Rows past
            // the last key are zeros, and where all rows see all keys there is no such row.)
            if (masked) {
                uint32_t odd = 0;
#pragma unroll
                for (int x = 0; x < kBlk; ++x) {
                    const u32x4 w = *(const u32x4 *)(stage + kTile + (kBlk * wave + x) * 1024 + lane * 16);
#pragma unroll
                    for (int e = 0; e < 4; ++e) odd |= (w[e] & 0x7f807f80u) + 0x00800080u;
                }
                if (__builtin_amdgcn_ballot_w64((odd & 0x80008000u) != 0) && lane == 0) *odd_tile = i;
                wait_lgkmcnt0();
                meet(); // (not __syncthreads, which waits for the DMA too)
                if (*odd_tile == i) { // the same for every wave
                    // into the rows that give their keys a weight, then zeros in their place
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
                        u32x4 w = __builtin_bit_cast(u32x4, vfrag(vs, s, dt));
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = odd_value(w[e] & 0xffffu, sign) | (odd_value(w[e] >> 16, sign) << 16);
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
            constexpr int kPv = kPf < 2 * NDT ? kPf : 2 * NDT;
            __builtin_amdgcn_s_setprio(1);
            bf16x8 vf[kPv];
#pragma unroll
            for (int x = 0; x < kPv; ++x) vf[x] = vfrag(vs, x / NDT, x % NDT);
#pragma unroll
            for (int x = 0; x < 2 * NDT; ++x) {
                const bf16x8 a = vf[x % kPv];
                if (x + kPv < 2 * NDT) vf[x % kPv] = vfrag(vs, (x + kPv) / NDT, (x + kPv) % NDT);
                __builtin_amdgcn_sched_barrier(0);
                O[x % NDT] = mfma_bf16(a, pb[x / NDT], O[x % NDT]);
            }
            __builtin_amdgcn_s_setprio(0);
        }
        wait_vmcnt<0>();  // the last (empty) loads have written before the stages are used again or given up
        float ltot = half_swap_sum(lsum);
        // A row that sees no key (a tree node without a bit, a position before the first key) has zeros, and -1 in the place of
        // its sum.  One that sees keys has a sum of 0 only where all their scores are -inf: no softmax, 0 / 0.
        uint32_t sees = pos >= 0;
        if constexpr (TREE) {
            sees = 0;
#pragma unroll 1
            for (int w = 0; w < p.tw; ++w) sees |= words[row % NB * p.tw + w];
        }
        if (sees == 0) { // (a node's cached keys were computed like the others': nothing of them leaves)
            m = -__builtin_inff(), ltot = -1.0f;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) O[dt] = f32x16{};
        }
        if (!whole) {
            float *po = p.part_o + (((long long)blk * kWaves + wave) * (NDT * 4) * 64 + lane) * 4;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4)
                    *(float4 *)(po + (dt * 4 + r4) * 256) =
                        float4{O[dt][4 * r4], O[dt][4 * r4 + 1], O[dt][4 * r4 + 2], O[dt][4 * r4 + 3]};
            if (dt0 == 0 && hi == 0) p.part_ml[(long long)blk * (32 * R) + row] = float2{m, ltot};
        } else {
            // ---- normalise, stage in LDS (32 R rows x 512 B), write 16-byte row pieces ----
            const float inv = ltot < 0.0f ? 0.0f : 1.0f / ltot;
            __syncthreads();
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const int d = (dt0 + dt) * 32 + 8 * r4 + 4 * hi;
                    u32x2 w;
                    w[0] = pack_bf16x2(O[dt][4 * r4] * inv, O[dt][4 * r4 + 1] * inv);
                    w[1] = pack_bf16x2(O[dt][4 * r4 + 2] * inv, O[dt][4 * r4 + 3] * inv);
                    *(u32x2 *)(smem + row * (kD * 2) + (((d >> 3) ^ l32) << 4) + (d & 4) * 2) = w;
                }
            __syncthreads();
#pragma unroll 2
            for (int x = tid; x < 32 * R * 32; x += kThreads) {
                const int rr = x >> 5, ch = x & 31, tt = q0 + rr % NB;
                if (tt < p.Sq)
                    *(u32x4 *)(p.o + b * p.sbo + (long long)(hk * kGroup + rr / NB) * p.sho + (long long)tt * p.ldo + ch * 8) =
                        *(const u32x4 *)(smem + rr * (kD * 2) + ((ch ^ (rr & 31)) << 4));
            }
        }
        if (!STREAM) return;
        left -= i1 - i0 + p.begin;
        if (left <= 0) return;
        i0 = 0, blk = 2 * blockIdx.x + 1; // (what lies between a workgroup's first and last is whole)
        ++b;
        keys = key_count(p, b);
        __syncthreads(); // everybody is done with the stages and the words
    }
}

// The partial states of a block's parts joined: with M = max_c m_c, w_c = 2^(m_c - M), o = (sum w_c O_c) / (sum w_c l_c).
// A part's accumulators are taken 64 lanes x 16 bytes at a time (4 dims of 32 rows x 2), by W waves that share the parts.
// Bound by reading the states that were just written: 64 MB take 15 us, 4.3 TB/s (more waves, more loads in flight or
// nontemporal ones: no faster); 1 MB takes 4 us.
template <int R, int D, bool TREE, bool STREAM, int W>
__global__ __launch_bounds__(256) void ca_merge_kernel(CaParams p) {
    constexpr int NB = 8 * R, NDT = kD / 32 / D, kFrags = 32 * R, kPer = 4 / W;
    __shared__ float4 accs[W > 1 ? 4 : 1][64];
    __shared__ float2 mls[W > 1 ? 4 : 1][64];
    const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int f = (blockIdx.x % (kFrags / kPer)) * kPer + wave / W, u = blockIdx.x / (kFrags / kPer);
    const int qb = u % p.nqb, hk = u / p.nqb % p.HK;
    int b = u / p.nqb / p.HK;
    const int q0 = qb * NB, row = f / (NDT * 4 * D) * 32 + l32;
    int n, g0 = 0, per = 0, s = 0; // parts; STREAM: the run of the first, the runs' tiles, the sequence's first tile
    if constexpr (STREAM) {
        Stream<TREE> all(p);
        per = all.per;
        int keys;
        if (p.B > p.runs) { // the sequence in which run b + 1 begins, if no run before begins in it
            const int at = (b + 1) * per;
            if (at >= all.total) return;
            int tile;
            all.find(p, at, b, keys, tile);
            s = at - tile;
            if (tile <= p.begin || (s + p.begin) / per < at / per - 1) return;
        } else {
            keys = key_count(p, b);
            s = all.first(p, b);
        }
        const int tiles = Tiles<TREE>(p, keys, q0, min(NB, p.Sq - q0)).n;
        g0 = (s + p.begin) / per;
        n = (s + p.begin + tiles - 1) / per - g0 + 1;
        if (n == 1) return; // its workgroup wrote it
    } else {
        n = (Tiles<TREE>(p, key_count(p, b), q0, min(NB, p.Sq - q0)).n + p.chunk - 1) / p.chunk;
    }
    auto part = [&](int c) -> long long {
        if constexpr (STREAM) return 2 * ((long long)(g0 + c) * p.HK + hk) + ((g0 + c) * per < s);
        return ((long long)(b * p.nchunk + c) * p.HK + hk) * p.nqb + qb;
    };
    float mx = -__builtin_inff(), l = 0.0f;
    float4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    // no part has a key that counts: weights 1 on zeros (a sum that is NaN or -1 stays so)
    auto weight = [](float m, float top) { return top == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - top); };
    auto add = [&](float w, float2 ml, float4 o) {
        l += w * ml.y;
        acc.x += w * o.x;
        acc.y += w * o.y;
        acc.z += w * o.z;
        acc.w += w * o.w;
    };
    constexpr int kBatch = W > 1 ? 8 : 4; // parts whose loads are in flight together
    for (int c0 = wave % W; c0 < n; c0 += W * kBatch) {
        float2 ml[kBatch];
        float4 o[kBatch];
#pragma unroll
        for (int x = 0; x < kBatch; ++x) {
            const int c = c0 + x * W;
            const long long at = part(c < n ? c : c0);
            ml[x] = p.part_ml[at * (32 * R) + row];
            o[x] = *(const float4 *)(p.part_o + ((at * kFrags + f) * 64 + lane) * 4);
            if (c >= n) ml[x] = float2{-__builtin_inff(), 0.0f}, o[x] = float4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        float top = mx;
#pragma unroll
        for (int x = 0; x < kBatch; ++x) top = __builtin_fmaxf(top, ml[x].x);
        const float w = weight(mx, top);
        l *= w, acc.x *= w, acc.y *= w, acc.z *= w, acc.w *= w;
        mx = top;
#pragma unroll
        for (int x = 0; x < kBatch; ++x) add(weight(ml[x].x, mx), ml[x], o[x]);
    }
    if constexpr (W > 1) {
        accs[wave][lane] = acc, mls[wave][lane] = float2{mx, l};
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 1; w < W; ++w) mx = __builtin_fmaxf(mx, mls[w][lane].x);
        l = 0.0f, acc = float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; ++w) add(weight(mls[w][lane].x, mx), mls[w][lane], accs[w][lane]);
    }
    const int t = q0 + row % NB;
    if (t >= p.Sq) return;
    const float inv = l < 0.0f ? 0.0f : 1.0f / l; // (a row that sees no key: the parts' -1)
    const int fr = f % (NDT * 4), dt = f / (NDT * 4) % D * NDT + fr / 4, d = dt * 32 + 8 * (fr % 4) + 4 * hi;
    u32x2 w;
    w[0] = pack_bf16x2(acc.x * inv, acc.y * inv);
    w[1] = pack_bf16x2(acc.z * inv, acc.w * inv);
    *(u32x2 *)(p.o + b * p.sbo + (long long)(hk * kGroup + row / NB) * p.sho + (long long)t * p.ldo + d) = w;
}

// ---- host side ----

// How a call is divided: row blocks (R) and dim parts (D) of a workgroup, and the work.
struct Plan {
    int R, D, nqb, gq, chunk, nchunk;
    int runs, dense;  // STREAM: most runs of tiles (0: every sequence whole); the tiles of a run below which half as many are made
    int least, begin; // a run's fewest tiles; the tiles that a sequence's beginning counts for
    bool stream, wide;
    long long tiles, wgs, states; // STREAM: a head's tiles; workgroups; partial rows
};

Plan plan(int B, int Sq, int HK, int max_tiles) {
    Plan pl{};
    pl.stream = Sq <= 64;
    pl.R = Sq <= 8 ? 1 : Sq <= 16 ? 2 : Sq <= 32 || !pl.stream ? 4 : 8;
    pl.D = pl.R < 4 ? 4 / pl.R : 1;
    pl.nqb = (Sq + 8 * pl.R - 1) / (8 * pl.R);
    pl.gq = pl.nqb < 8 ? pl.nqb : 8;
    pl.chunk = max_tiles, pl.nchunk = 1;
    const int slots = kCus * (pl.R < 8 ? 2 : 1);
    const long long units = (long long)B * HK;
    // A workgroup a sequence and head, undivided, where those are many or short: no state to write and join, no sequence
    // begun behind another's end.  The longest of a batch is then waited for, alone in the end, so only up to a length that
    // grows with how full the chip is: 10 tiles, or 10 max(R, 2) for every 128 sequences x heads.  (These workgroups, evenly
    // divided, would have a quarter of a sequence's tiles each at 128 sequences x heads, or half with R = 8, and states to
    // write and join.)  Divided / whole, us (nodes, sequences x keys): 4, 1 x 60 13.2 /
    // 8.9, 32 x 1000 31.9 / 42.4, 64 x 500 43.7 / 32.0, 200 x 3500 394 / 362; 16, 32 x 1000 40.8 / 45.0, 64 x 500 43.0 / 35.0;
    // 32, 32 x 1000 51.5 / 47.7, 600 x 800 554 / 423; 64, 8 x 250 30.4 / 26.1, 64 x 2000 179 / 139.
    if (pl.stream && max_tiles <= std::max(10ll, 10ll * std::max(pl.R, 2) * (units / 128))) {
        pl.wgs = units;
        return pl;
    }
    if (pl.stream) {
        // Two workgroups a CU, while each gets enough tiles to repay the partial state that it writes (32 R KB) and the merge
        // reads (R = 1: 8, else 12); else one, of 4 tiles at least, and of fewer only where even so the chip would be nearly
        // empty.  Measured, us, two / one a CU (nodes, sequences x keys): 4, 8 x 5000 44.3 / 46.5, 2 x 10000 27.1 / 24.1;
        // 16, 32 x 4096 102 / 110, 1 x 32768 45.6 / 41.3; 32, 16 x 2000 56.8 / 50.1, 16 x 4000 84 / 85.  Tiles a workgroup
        // 2 / 4 in a nearly empty chip: 8, 1 x 500 14.1 / 15.9; 64, 1 x 500 23.5 / 22.8.
        pl.dense = pl.R == 8 ? 0 : pl.R == 1 ? 8 : 12;
        pl.least = pl.R == 8 ? 4 : 2;
        // A sequence's beginning (its words, queries and first tile are waited for) takes a workgroup as long as a few tiles:
        // counted for none / 4 tiles, 16 x 32 nodes after 4000 keys 89.4 / 83.9 us, 2 x 10000 42.8 / 36.4; 64 nodes, none / 4 /
        // 6: 2 x 10000 62.7 / 51.9 / 52.5, 16 x 4000 105 / 102 / 96.
        pl.begin = B == 1 ? 0 : pl.R == 8 ? 6 : 4;
        pl.tiles = (long long)B * (max_tiles + pl.begin);
        const long long most = (pl.tiles + pl.least - 1) / pl.least;
        pl.runs = HK < slots ? slots / HK : 1;
        pl.wgs = (most < pl.runs ? most : pl.runs) * HK;
        pl.states = pl.wgs * 2 * 32 * pl.R;
        // (few waves, then, of many parts each; 8 nodes, 1 x 32768 keys 54.6 -> 40.2 us, but 16 x 4000 64.2 -> 68.9 if waves
        // share there)
        pl.wide = units * pl.R <= 16;
        return pl;
    }
    // The chunks that take the least time, in 1/20 us: a tile of a workgroup alone on its CU 30, beside another 44; with
    // several chunks the partial states (128 KB a workgroup) written and joined.  Counted as rounds of tiles, and 10 tiles
    // for the states, instead: 8 x 255 nodes after 300 keys 60.1 us, now 42.6; 2000 tokens with a window of 1000 60.6, now
    // 50.5; 3 x 130 nodes after 3500 keys 53.9, now 53.1.  Up to 64 chunks (65 nodes after 32768 keys: with 16 94
    // us, with 24 88, now 78).  Never so many workgroups that a grid, here or of the join (8 R workgroups a block), would reach
    // 2^32 work-items: it would wrap round without an error.
    const long long base = units * pl.nqb;
    long long best = -1;
    for (int n = 1; n <= 64 && base > 0 && (n == 1 || base * n < (1 << 20)); ++n) {
        const long long tiles = (max_tiles + n - 1) / n, wgs = base * n, full = wgs / slots, rest = wgs % slots;
        const long long cost = tiles * (full * 44 + (rest > kCus ? 44 : rest ? 30 : 0)) + (n > 1 ? 180 + wgs * 17 / 20 : 0);
        if (best < 0 || cost < best) best = cost, pl.chunk = (int)tiles;
    }
    pl.nchunk = pl.chunk > 0 ? (max_tiles + pl.chunk - 1) / pl.chunk : 1;
    const long long groups = units * pl.nchunk * ((pl.nqb + pl.gq - 1) / pl.gq);
    pl.wgs = (groups + 7) / 8 * 8 * pl.gq;
    pl.states = pl.nchunk > 1 ? base * pl.nchunk * 32 * pl.R : 0;
    return pl;
}

int tree_tiles(int N, int cap) { return (int)((cap + (kBK - 1ll)) / kBK) + (N + kBK - 1) / kBK; }
// most tiles of a block of Sq <= 64 or 32 queries: the sinks', the window's and the block's own, never more than the keys'
int window_tiles(int Sq, int Sk, int window, int sinks) {
    const long long all = Sk > 0 ? ((long long)Sk + kBK - 1) / kBK : 1;
    const long long span = ((long long)window + (Sq <= 64 ? Sq : 32) + 2 * kBK - 3) / kBK + 1;
    const long long n = (sinks + kBK - 1ll) / kBK + span;
    return (int)(n < all ? n : all);
}
long long state_bytes(const Plan &pl) { return pl.states * (kD * 4 + 8); }

template <int R, int D, bool TREE, bool STREAM>
int launch_as(const CaParams &p, const Plan &pl, hipStream_t st) {
    hipLaunchKernelGGL((ca_fwd_kernel<R, D, TREE, STREAM>), dim3((unsigned)pl.wgs), dim3(64 * R * D), 0, st, p);
    if (const int rc = mica_err(hipGetLastError())) return rc;
    if (pl.states == 0) return 0;
    // STREAM: a sequence is divided where a run begins in it, so that there are no more of these than runs (every workgroup
    // walks all the key counts: with workgroups for all sequences, 3000 tokens of up to 200 keys each took 2052 us and not 498)
    const long long blocks = (long long)(STREAM && p.B > pl.runs ? pl.runs - 1 : p.B) * p.HK * pl.nqb;
    if (blocks == 0) return 0;
    const dim3 one((unsigned)(blocks * 8 * R)), four((unsigned)(blocks * 32 * R));
    if (STREAM && pl.wide) hipLaunchKernelGGL((ca_merge_kernel<R, D, TREE, STREAM, STREAM ? 4 : 1>), four, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((ca_merge_kernel<R, D, TREE, STREAM, 1>), one, dim3(256), 0, st, p);
    return mica_err(hipGetLastError());
}

template <bool TREE>
int launch(CaParams &p, const Plan &pl, void *workspace, hipStream_t st) {
    p.nqb = pl.nqb, p.gq = pl.gq, p.chunk = pl.chunk, p.nchunk = pl.nchunk;
    p.runs = pl.runs, p.dense = pl.dense, p.least = pl.least, p.begin = pl.begin;
    p.part_o = (float *)workspace;
    p.part_ml = (float2 *)((char *)workspace + pl.states * kD * 4);
    if (pl.wgs >= (1LL << 31) || pl.tiles >= (1LL << 30)) return MICA_MISS_RANGE;
    if (!pl.stream) return launch_as<4, 1, TREE, false>(p, pl, st);
    if (pl.R == 1) return launch_as<1, 4, TREE, true>(p, pl, st);
    if (pl.R == 2) return launch_as<2, 2, TREE, true>(p, pl, st);
    if (pl.R == 4) return launch_as<4, 1, TREE, true>(p, pl, st);
    return launch_as<8, 1, TREE, true>(p, pl, st);
}

// a row stride of `rows` rows that are read by DMA: 32 rows within a buffer's 31-bit range, none overlapping
int row_stride(long long &ld, long long rows) {
    if (rows <= 1) ld = kD; // (never used; the range check of a tile counts on it)
    if (ld < kD || ld % 8) return MICA_MISS_STRIDE;
    return ld * 2 * kBK >= (1LL << 31) ? MICA_MISS_RANGE : 0;
}
bool strides_ok(std::initializer_list<long long> v) {
    for (long long x : v)
        if (x < 0 || x % 8) return false;
    return true;
}
// common checks of sizes; 0 when the call goes on
int check_sizes(int B, int Sq, int HQ, int HK, int head_dim, float scale) {
    if (head_dim != kD || HK <= 0 || HK > (1 << 20) || HQ != HK * kGroup || B < 0 || Sq < 0) return MICA_MISS_SHAPE;
    if (!(scale > 0.0f) || !(scale < __builtin_inff())) return MICA_MISS_ARG;
    if ((long long)B * HK * ((Sq + 7) / 8) >= (1LL << 24)) return MICA_MISS_RANGE;
    return 0;
}

}  // namespace

extern "C" long long mica_attention_tree_workspace_bytes(int B, int N, int HK, int cache_cap) {
    if (B < 0 || N < 0 || N > kMaxNodes || HK <= 0 || cache_cap < 0) return -1;
    return state_bytes(plan(B, N, HK, tree_tiles(N, cache_cap)));
}

extern "C" int mica_attention_tree(const void *q, long long sbq, long long shq, long long ldq, const void *k, long long sbk,
                                   long long shk, long long ldk, const void *v, long long sbv, long long shv,
                                   long long ldv, const void *k_cache, long long sbkc, long long shkc, long long ldkc,
                                   const void *v_cache, long long sbvc, long long shvc, long long ldvc, int cache_cap,
                                   const int *cache_len, const unsigned long long *tree, long long sbt, void *o,
                                   long long sbo, long long sho, long long ldo, int B, int N, int HQ, int HK, int head_dim,
                                   float scale, void *workspace, long long workspace_bytes, mica_stream_t stream) {
    if (const int rc = check_sizes(B, N, HQ, HK, head_dim, scale)) return rc;
    if (N > kMaxNodes || cache_cap < 0) return MICA_MISS_SHAPE;
    if (B == 0 || N == 0) return 0;
    if (!q || !k || !v || !o || !tree || (cache_cap > 0 && (!k_cache || !v_cache))) return MICA_MISS_ARG;
    if (!strides_ok({sbq, shq, ldq, sbk, shk, sbv, shv, sbo, sho, ldo}) || sbt < 0) return MICA_MISS_STRIDE;
    if (cache_cap > 0 && !strides_ok({sbkc, shkc, sbvc, shvc})) return MICA_MISS_STRIDE;
    if (cache_cap == 0) ldkc = ldvc = kD;
    const struct { long long *ld; long long rows; } ch[4] = {{&ldk, N}, {&ldv, N}, {&ldkc, cache_cap}, {&ldvc, cache_cap}};
    for (const auto &x : ch)
        if (const int rc = row_stride(*x.ld, x.rows)) return rc;
    if (!mica_aligned16(q) || !mica_aligned16(k) || !mica_aligned16(v) || !mica_aligned16(o) || ((uintptr_t)tree & 7) ||
        (cache_cap > 0 && (!mica_aligned16(k_cache) || !mica_aligned16(v_cache))))
        return MICA_MISS_ALIGN;
    const Plan pl = plan(B, N, HK, tree_tiles(N, cache_cap));
    if (pl.states && (!workspace || !mica_aligned16(workspace) || workspace_bytes < state_bytes(pl))) return MICA_MISS_ARG;
    CaParams p{};
    p.q = (const uint16_t *)q; p.sbq = sbq; p.shq = shq; p.ldq = ldq;
    p.k = (const uint16_t *)k; p.sbk = sbk; p.shk = shk; p.ldk = ldk;
    p.v = (const uint16_t *)v; p.sbv = sbv; p.shv = shv; p.ldv = ldv;
    p.kc = (const uint16_t *)k_cache; p.sbkc = sbkc; p.shkc = shkc; p.ldkc = ldkc;
    p.vc = (const uint16_t *)v_cache; p.sbvc = sbvc; p.shvc = shvc; p.ldvc = ldvc;
    p.o = (uint16_t *)o; p.sbo = sbo; p.sho = sho; p.ldo = ldo;
    p.len = cache_len; p.cap = cache_cap;
    p.tree = (const uint32_t *)tree; p.sbt = 2 * sbt; p.tw = 2 * ((N + 63) / 64);
    p.B = B; p.Sq = N; p.HK = HK;
    p.scale_log2 = scale * 1.44269504088896341f;
    return launch<true>(p, pl, workspace, (hipStream_t)stream);
}

extern "C" long long mica_attention_window_workspace_bytes(int B, int Sq, int Sk, int HK, int window, int sinks) {
    if (B < 0 || Sq < 0 || Sk < 0 || HK <= 0 || window < 1 || sinks < 0) return -1;
    return state_bytes(plan(B, Sq, HK, window_tiles(Sq, Sk, window, sinks)));
}

extern "C" int mica_attention_window(const void *q, long long sbq, long long shq, long long ldq, const void *k,
                                     long long sbk, long long shk, long long ldk, const void *v, long long sbv,
                                     long long shv, long long ldv, void *o, long long sbo, long long sho, long long ldo,
                                     int B, int Sq, int Sk, int HQ, int HK, int head_dim, float scale, int window, int sinks,
                                     const int *kv_len, void *workspace, long long workspace_bytes, mica_stream_t stream) {
    if (const int rc = check_sizes(B, Sq, HQ, HK, head_dim, scale)) return rc;
    if (Sk < 0 || window < 1 || sinks < 0) return MICA_MISS_SHAPE;
    if (B == 0 || Sq == 0) return 0;
    if (!q || !o || (Sk > 0 && (!k || !v))) return MICA_MISS_ARG;
    if (!strides_ok({sbq, shq, ldq, sbk, shk, sbv, shv, sbo, sho, ldo})) return MICA_MISS_STRIDE;
    if (const int rc = row_stride(ldk, Sk)) return rc;
    if (const int rc = row_stride(ldv, Sk)) return rc;
    if (!mica_aligned16(q) || !mica_aligned16(o) || (Sk > 0 && (!mica_aligned16(k) || !mica_aligned16(v))))
        return MICA_MISS_ALIGN;
    const Plan pl = plan(B, Sq, HK, window_tiles(Sq, Sk, window, sinks));
    if (pl.states && (!workspace || !mica_aligned16(workspace) || workspace_bytes < state_bytes(pl))) return MICA_MISS_ARG;
    CaParams p{};
    p.q = (const uint16_t *)q; p.sbq = sbq; p.shq = shq; p.ldq = ldq;
    p.k = (const uint16_t *)k; p.sbk = sbk; p.shk = shk; p.ldk = ldk;
    p.v = (const uint16_t *)v; p.sbv = sbv; p.shv = shv; p.ldv = ldv;
    p.o = (uint16_t *)o; p.sbo = sbo; p.sho = sho; p.ldo = ldo;
    p.len = kv_len; p.cap = Sk;
    p.B = B; p.Sq = Sq; p.HK = HK; p.window = window; p.sinks = sinks;
    p.scale_log2 = scale * 1.44269504088896341f;
    return launch<false>(p, pl, workspace, (hipStream_t)stream);
}
