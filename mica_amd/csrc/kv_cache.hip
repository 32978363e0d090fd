// Keys and values into the paged 8-bit cache (mica_kv_append), and back out of it in bf16 (mica_kv_read); paged.h has the
// layout.
//
// append: a row's key head is normed and rotated where asked for, in fp32 and rounded to bf16 once; then
//   block full:      s = max(max |x|, 1e-8) / 127 over the block's 32 x 256 values of a head,  q = rint(x / s)
//   block not full:  the bf16 rows wait in the sequence's slot
// so a block's values are those of its bf16 rows whichever call brought them.
//
// Work split: a workgroup takes one block of 32 tokens of one head and side, 8 threads a token (thread `sub` holds the 16-byte
// chunks sub, sub + 8, sub + 16, sub + 24 of the row, so a load instruction reads whole 128-byte lines).  A sequence's first
// workgroup also writes its rest: the rows that it replaces are those that the same threads have read.
//
// Bound: append by HBM and, before it, the waves' phases (load, norm and rotation, the block's largest, store): 15 prompts of up to
// 2047 tokens, 16 K rows of 4 heads, 31 us, 67 MB read and 34 written, 3.2 TB/s.  More waves a SIMD than the registers allow (5 / 6
// / 8) spill: 52 -> 59 / 69 / 84 us with the read of the same rows.  Read by HBM: 40005 rows of 4 heads 38 to 52 us, 4.7 to 6.4 TB/s.
// Single tokens cost their launch: 64 x 1 appended 5 us, 320 rows read 5.
//
// Rounding: a bf16 value goes to the nearest of 255 steps of its block's scale once; read, scale x int8 goes to bf16 once.
#include "paged.h"

namespace {

constexpr int kThreads = 256;

struct AppendParams {
    Pages c;
    Ragged rows;
    const uint16_t *k; long long shk, ldk;  // head h of row t: k + h shk + t ldk
    const uint16_t *v; long long shv, ldv;
    const uint16_t *w;                      // bf16 [256] head norm weight, or null
    float off, eps;
    int rot_dim, n_pos;
    const void *cos_tab, *sin_tab;          // [n_pos][rot_dim / 2], bf16 or fp32
    int wide;                               // fp32 tables
    const int *pos;                         // [T] or null: the row's place in its sequence
    int each;                               // workgroups a sequence; 0: one for each unit
};

// 8 table entries from entry i on
MICA_DEVICE void table8(const void *t, int wide, long long i, float (&x)[8]) {
    if (wide) {
        const float4 a = *(const float4 *)((const float *)t + i), b = *(const float4 *)((const float *)t + i + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const u32x4 a = *(const u32x4 *)((const uint16_t *)t + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[2 * e] = bf16_lo(a[e]), x[2 * e + 1] = bf16_hi(a[e]);
    }
}

// A key row (this thread's chunks of it) normed and rotated.  The 8 threads of a row call together; `live`: it is one.
MICA_DEVICE void treat(const AppendParams &p, u32x4 (&x)[4], int sub, bool live, int pos) {
    float f[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) f[i][2 * e] = bf16_lo(x[i][e]), f[i][2 * e + 1] = bf16_hi(x[i][e]);
    if (p.w != nullptr) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(f[i][e], f[i][e], ss);
#pragma unroll
        for (int m = 1; m < 8; m <<= 1) ss += __shfl_xor(ss, m, 64);
        const float rstd = 1.0f / __builtin_sqrtf(ss / (float)kPagedDim + p.eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u32x4 w = *(const u32x4 *)(p.w + 8 * (sub + 8 * i));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[i][2 * e] = (f[i][2 * e] * rstd) * (p.off + bf16_lo(w[e]));
                f[i][2 * e + 1] = (f[i][2 * e + 1] * rstd) * (p.off + bf16_hi(w[e]));
            }
        }
    }
    // dim d of the first half of the rotated ones pairs with d + rot_dim / 2: h chunks on, which is h / 8 of this thread's
    // own, or another thread's
    const int h = p.rot_dim >> 4;
    if (h > 0) {
        const bool turn = live && pos >= 0 && pos < p.n_pos; // out-of-table positions are left as they are
        const long long row = (long long)(turn ? pos : 0) * (p.rot_dim >> 1);
        auto pair = [&](float (&a)[8], float (&b)[8], int chunk) {
            float c[8], s[8];
            table8(p.cos_tab, p.wide, row + 8 * chunk, c);
            table8(p.sin_tab, p.wide, row + 8 * chunk, s);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float lo = a[e] * c[e] - b[e] * s[e], hi = b[e] * c[e] + a[e] * s[e];
                if (turn) a[e] = lo, b[e] = hi;
            }
        };
        if (h == 16) {
            pair(f[0], f[2], sub);
            pair(f[1], f[3], sub + 8);
        } else if (h == 8) {
            pair(f[0], f[1], sub);
        } else { // chunks 0 .. 2 h - 1 are the threads' first ones
            float a[8], b[8];
            const bool upper = (sub & h) != 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float o = __shfl_xor(f[0][e], h, 64);
                a[e] = upper ? o : f[0][e], b[e] = upper ? f[0][e] : o;
            }
            pair(a, b, sub & (h - 1));
            if (sub < 2 * h)
#pragma unroll
                for (int e = 0; e < 8; ++e) f[0][e] = upper ? b[e] : a[e];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = pack_bf16x2(f[i][2 * e], f[i][2 * e + 1]);
}

__global__ __launch_bounds__(kThreads) void kv_append_kernel(AppendParams p) {
    __shared__ int tops[4];
    __shared__ __attribute__((aligned(16))) int8_t tile[kPage][kPagedDim];
    const int tid = threadIdx.x, token = tid >> 3, sub = tid & 7;
    const int side = blockIdx.x % 2, hk = blockIdx.x / 2 % p.c.HK, id = blockIdx.x / 2 / p.c.HK;
    // a sequence's units: the blocks that it finishes, or one for the rest alone
    auto units = [&](int b) {
        const int n = p.rows.rows(b);
        return n ? max((p.c.len(b) % kPage + n) / kPage, 1) : 0;
    };
    int b, u;
    if (p.each) b = id / p.each, u = id % p.each;
    else if (!find_unit(p.rows.B, units, id, b, u)) return;
    b = __builtin_amdgcn_readfirstlane(b), u = __builtin_amdgcn_readfirstlane(u);
    const int first = p.rows.at(b), n = p.rows.rows(b), p0 = p.c.len(b), slot = p.c.slot(b);
    if (n == 0 || slot < 0) return;
    const int r = p0 % kPage, full = (r + n) / kPage, left = (r + n) % kPage;
    const bool keys = side == 0, any = p.w != nullptr || p.rot_dim > 0;
    uint16_t *rest = p.c.rest(slot, side, hk);
    const uint16_t *src = keys ? p.k + hk * p.shk : p.v + hk * p.shv;
    const long long ld = keys ? p.ldk : p.ldv;
    // this thread's chunks of new row i (0 .. n - 1)
    auto fetch = [&](int i, bool live, u32x4 (&x)[4]) {
        const uint16_t *row = src + (long long)(first + (live ? i : 0)) * ld + 8 * sub;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = live ? *(const u32x4 *)(row + 64 * j) : u32x4{0u, 0u, 0u, 0u};
        if (keys && any) treat(p, x, sub, live, !live ? -1 : p.pos ? p.pos[first + i] : p0 + i);
    };
    for (; u < max(full, 1); u += p.each ? p.each : (1 << 30)) {
        if (u < full) {
            const int i = u * kPage + token - r; // the token's new row; below 0 one that waits already
            u32x4 x[4];
            fetch(i, i >= 0, x);
            if (i < 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = *(const u32x4 *)(rest + token * kPagedDim + 8 * (sub + 8 * j));
            }
            // the largest magnitude, as bf16 bits: ordered like the values, with infinities and NaN above all of them
            int top = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, max((int)(x[j][e] & 0x7fffu), (int)((x[j][e] >> 16) & 0x7fffu)));
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) top = max(top, __shfl_xor(top, m, 64));
            if ((tid & 63) == 0) tops[tid >> 6] = top;
            __syncthreads();
            top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
            const bool fine = top < 0x7f80;
            const float amax = fine ? bf16_to_f32((uint16_t)top) : 0.0f, s = row_scale(amax);
            const float mul = fma_quant_recip(amax, s, 1.0f / s);
            const int block = p0 / kPage + u, page = p.c.page(b, block);
            u32x2 q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[2 * e] = bf16_lo(x[j][e]), f[2 * e + 1] = bf16_hi(x[j][e]);
                q[j] = fine ? fma_quant8(f, mul) : u32x2{0u, 0u};
            }
            if (page >= 0 && tid == 0) // (a value that is not finite: every value of the block is NaN)
                p.c.scales[p.c.index(page, side, hk)] = fine ? s : __builtin_nanf("");
            if (keys) {
                if (page >= 0) {
                    int8_t *out = p.c.block(page, 0, hk) + token * 32 + (sub & 3) * 8;
#pragma unroll
                    for (int j = 0; j < 4; ++j) *(u32x2 *)(out + (2 * j + (sub >> 2)) * 1024) = q[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) *(u32x2 *)(&tile[token][8 * (sub + 8 * j)]) = q[j];
                __syncthreads();
                u32x4 o[2]; // dim tid's 32 tokens
#pragma unroll
                for (int w = 0; w < 8; ++w) {
                    const int t = 4 * page_four(w);
                    o[w >> 2][w & 3] = pack_i8x4(tile[t][tid], tile[t + 1][tid], tile[t + 2][tid], tile[t + 3][tid]);
                }
                if (page >= 0) {
                    u32x4 *out = (u32x4 *)(p.c.block(page, 1, hk) + tid * 32);
                    out[0] = o[0], out[1] = o[1];
                }
            }
            __syncthreads(); // tops and the tile are free again
        }
        if (u == 0) {
            // the rest: new rows behind those that wait, or the last `left` rows
            const int i = full ? n - left + token : token - r;
            const bool live = full ? token < left : token >= r && i < n;
            if (full && left == 0) continue;
            u32x4 x[4];
            fetch(i, live, x);
            if (live) {
#pragma unroll
                for (int j = 0; j < 4; ++j) *(u32x4 *)(rest + token * kPagedDim + 8 * (sub + 8 * j)) = x[j];
            }
        }
    }
}

struct ReadParams {
    Pages c;
    Ragged rows;
    uint16_t *k, *v;   // [T][HK][256]
    int each, wgs;     // workgroups a sequence (0: one for each unit); of a head and side
};

__global__ __launch_bounds__(kThreads) void kv_read_kernel(ReadParams p) {
    __shared__ __attribute__((aligned(16))) uint16_t tile[kPage][kPagedDim];
    const int tid = threadIdx.x, token = tid >> 3, sub = tid & 7;
    const int side = blockIdx.x % 2, hk = blockIdx.x / 2 % p.c.HK, id = blockIdx.x / 2 / p.c.HK;
    uint16_t *out = (side ? p.v : p.k) + hk * kPagedDim;
    const long long ld = (long long)p.c.HK * kPagedDim;
    auto store = [&](long long row, const u32x4 (&x)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) *(u32x4 *)(out + row * ld + 8 * (sub + 8 * j)) = x[j];
    };
    const u32x4 zeros[4] = {};
    // rows of no sequence, before the first and behind the last
    const int before = p.rows.at(0), none = before + p.rows.T - p.rows.at(p.rows.B);
    for (int i = id * kPage + token; i < none; i += p.wgs * kPage) store(i < before ? i : p.rows.T - none + (long long)i, zeros);
    // a sequence's units: the blocks that its rows lie in (places before the sequence's beginning too: they are zeros)
    auto units = [&](int b) {
        const int n = p.rows.rows(b), last = p.c.len(b) - 1;
        return n ? (last >> 5) - ((last - n + 1) >> 5) + 1 : 0;
    };
    int b, u;
    if (p.each) b = id / p.each, u = id % p.each;
    else if (!find_unit(p.rows.B, units, id, b, u)) return;
    b = __builtin_amdgcn_readfirstlane(b), u = __builtin_amdgcn_readfirstlane(u);
    const int n = p.rows.rows(b), len = p.c.len(b), from = len - n, first = p.rows.at(b), slot = p.c.slot(b);
    for (const int all = units(b); u < all; u += p.each ? p.each : all) {
        const int block = (from >> 5) + u, at = block * kPage + token;
        const bool live = at >= from && at < len;
        const long long row = first + (long long)at - from;
        if (block < 0) {
            if (live) store(row, zeros);
            continue;
        }
        u32x4 x[4];
        if (block < len / kPage) {
            const int page = p.c.page(b, block);
            const float s = p.c.scale(page, side, hk);
            const int8_t *src = p.c.block(max(page, 0), side, hk);
            if (side == 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const u32x2 q = page >= 0 ? *(const u32x2 *)(src + (2 * j + (sub >> 2)) * 1024 + token * 32 + (sub & 3) * 8)
                                              : u32x2{0u, 0u};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t w = q[e >> 1] >> (16 * (e & 1));
                        x[j][e] = pack_bf16x2((float)(int8_t)w * s, (float)(int8_t)(w >> 8) * s);
                    }
                }
            } else {
                u32x4 q[2] = {};
                if (page >= 0) q[0] = ((const u32x4 *)(src + tid * 32))[0], q[1] = ((const u32x4 *)(src + tid * 32))[1];
#pragma unroll
                for (int w = 0; w < 8; ++w)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        tile[4 * page_four(w) + e][tid] = f32_to_bf16((float)(int8_t)(q[w >> 2][w & 3] >> (8 * e)) * s);
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = *(const u32x4 *)&tile[token][8 * (sub + 8 * j)];
                __syncthreads(); // the tile is free again
            }
        } else {
            const uint16_t *rest = p.c.rest(max(slot, 0), side, hk);
            const uint32_t nan = 0x7fc07fc0u;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[j] = slot >= 0 && live ? *(const u32x4 *)(rest + token * kPagedDim + 8 * (sub + 8 * j)) : u32x4{nan, nan, nan, nan};
        }
        if (live) store(row, x);
    }
}

}  // namespace

extern "C" int mica_kv_append(const void *k, long long shk, long long ldk, const void *v, long long shv, long long ldv,
                              const int *starts, int B, int T, void *data, float *scales, void *recent, int pages, int n_slots,
                              int HK, int head_dim, const int *table, long long ldt, int width, const int *lens,
                              const int *slots, const void *norm_w, float norm_offset, float norm_eps, int rot_dim,
                              const void *cos_tab, const void *sin_tab, int tab_dtype, int n_pos, const int *pos, int longest,
                              mica_stream_t stream) {
    if (B < 0 || T < 0) return MICA_MISS_SHAPE;
    if (rot_dim != 0 && rot_dim != 16 && rot_dim != 32 && rot_dim != 64 && rot_dim != 128 && rot_dim != 256) return MICA_MISS_SHAPE;
    if (tab_dtype != MICA_BF16 && tab_dtype != MICA_FP32) return MICA_MISS_DTYPE;
    if (B == 0 || T == 0) return 0;
    AppendParams p{};
    if (const int rc = mica_paged_check(p.c, data, scales, recent, pages, n_slots, HK, head_dim, table, ldt, width, lens, slots, B))
        return rc;
    if (!k || !v || !starts || (rot_dim && (!cos_tab || !sin_tab || n_pos < 0))) return MICA_MISS_ARG;
    for (long long x : {shk, ldk, shv, ldv})
        if (x < 0 || x % 8) return MICA_MISS_STRIDE;
    if (!mica_aligned16(k) || !mica_aligned16(v) || !mica_aligned16(norm_w) || !mica_aligned16(cos_tab) ||
        !mica_aligned16(sin_tab) || ((uintptr_t)starts & 3) || ((uintptr_t)pos & 3))
        return MICA_MISS_ALIGN;
    if (rot_dim && n_pos == 0) return MICA_MISS_ARG; // (a row outside the tables takes their first row's place, unused)
    p.rows = Ragged{starts, B, T};
    p.k = (const uint16_t *)k; p.shk = shk; p.ldk = ldk;
    p.v = (const uint16_t *)v; p.shv = shv; p.ldv = ldv;
    p.w = (const uint16_t *)norm_w; p.off = norm_offset; p.eps = norm_eps;
    p.rot_dim = rot_dim; p.cos_tab = cos_tab; p.sin_tab = sin_tab; p.wide = tab_dtype == MICA_FP32; p.n_pos = n_pos; p.pos = pos;
    // units of all sequences: every block that n rows finish, or one; at most (n + 31) / 32 and n of each
    const long long most = ((long long)T + 31ll * B) / 32, units = most < T ? most : T;
    // Where no sequence has many (`longest` rows: a hint, a workgroup takes more than one if it has to), a workgroup for each,
    // without the search.
    const long long hint = longest > 0 && longest < T ? longest : T, each = (hint + 31) / 32;
    p.each = each * B <= 2 * units ? (int)each : 0;
    const long long wgs = (p.each ? each * B : units) * HK * 2;
    if (wgs >= (1 << 24)) return MICA_MISS_RANGE; // (a grid of 2^32 work-items wraps round)
    hipLaunchKernelGGL(kv_append_kernel, dim3((unsigned)wgs), dim3(kThreads), 0, (hipStream_t)stream, p);
    return mica_err(hipGetLastError());
}

extern "C" int mica_kv_read(void *k, void *v, const int *starts, int B, int T, const void *data, const float *scales,
                            const void *recent, int pages, int n_slots, int HK, int head_dim, const int *table, long long ldt,
                            int width, const int *lens, const int *slots, int longest, mica_stream_t stream) {
    if (B < 0 || T < 0) return MICA_MISS_SHAPE;
    if (T == 0) return 0;
    ReadParams p{};
    if (const int rc = mica_paged_check(p.c, (void *)data, (void *)scales, (void *)recent, pages, n_slots, HK, head_dim, table, ldt,
                                   width, lens, slots, B))
        return rc;
    if (!k || !v || !starts) return MICA_MISS_ARG;
    if (!mica_aligned16(k) || !mica_aligned16(v) || ((uintptr_t)starts & 3)) return MICA_MISS_ALIGN;
    p.rows = Ragged{starts, B, T};
    p.k = (uint16_t *)k; p.v = (uint16_t *)v;
    // blocks that n rows lie in: at most (n + 62) / 32 and n; each sequence's without the search as for an append
    const long long most = ((long long)T + 62ll * B) / 32, units = B == 0 ? 1 : most < T ? most : T;
    const long long hint = longest > 0 && longest < T ? longest : T, each = hint < 2 ? 1 : (hint + 62) / 32;
    p.each = B > 0 && each * B <= 2 * units ? (int)each : 0;
    const long long per = p.each ? each * B : units, wgs = per * HK * 2;
    p.wgs = (int)(per < (1 << 30) ? per : 1);
    if (wgs >= (1 << 24)) return MICA_MISS_RANGE;
    hipLaunchKernelGGL(kv_read_kernel, dim3((unsigned)wgs), dim3(kThreads), 0, (hipStream_t)stream, p);
    return mica_err(hipGetLastError());
}
