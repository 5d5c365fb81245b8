// Dense bf16 linear with bias, activation and residual in its epilogue, and its backward: the unquantised linears of a
// transformer (primus/backends/megatron/core/extensions/primus_turbo.py:1180-1188 is the route without a recipe), whose bias, activation
// and residual are passes of their own over the output otherwise.
//
//   y = act(z) + residual,  z = a . b^T + bias     a [m, k], b [n, k];  fp32 from the products to y, one rounding
//   backward: dz = dy act'(z) in bf16,  da = dz . b,  db = dz^T . a,  dbias = column sums of dz before its rounding
//
// A product with enough tiles of 256 x 256 runs on the grouped kernels' (mx_gemm_bf16.hip) with one group.  This
// file holds the tiles of 256 x 128 and 64 x 64 for the others, the kernel for a few rows, which is bound by reading b, and
// the elementwise part of the backward.
#include "mx_gemm_bf16.h"
#include "mx_gemm_common.h"

namespace mxl {

typedef __bf16 d8bf __attribute__((ext_vector_type(8)));
typedef short d4s __attribute__((ext_vector_type(4)));

struct DenseArgs {
    const uint8_t* a;       // [m, k], or [k, m] (A_T)
    const uint8_t* b;       // [n, k], or [k, n] (B_T)
    uint16_t* c;            // [m, n]
    int64_t m, n, k;
    EpilogueArgs epi;
    float* partial;         // SPLIT: [splits, m, n]
    int splits, split_slots;
    float* sum;             // the join adds to this float [m, n] (the weight gradient into main_grad) instead of writing c
};

constexpr int DT_KS = 64;       // contraction elements per slot: 128 bytes of a row, four MFMA steps

template <int TM, int TN, int ST, bool SPLIT> constexpr int dense_lds_bytes() {
    const int loop = ST * (TM + TN) * DT_KS * 2, out = TM * (TN * (SPLIT ? 4 : 2) + 16);
    return loop > out ? loop : out;
}

// ---- tiles: WM x 2 waves, LDS-direct loads into three stages.  64 x 64: 4 waves, up to three workgroups on a CU, so that one's epilogue and
// waits run under another's MFMAs.  256 x 128: 8 waves of 64 x 64, two on a SIMD; a wave reads 1 KiB of LDS per MFMA, which with the
// fills makes 1375 clocks of LDS for 1024 of MFMAs in a slot.  A_T, B_T: the operand is [k, m], [k, n], read with the transposing LDS read.
// SPLIT: the contraction is cut into `splits` runs of slots, a workgroup each, whose fp32 sums dense_join_kernel adds up. ----
template <int TM, int TN, int WM, int ST, bool A_T, bool B_T, int ACT, bool SPLIT>
__global__ __launch_bounds__(WM * 128, 2) void dense_tile_kernel(DenseArgs p) {
    constexpr int THREADS = WM * 128, WROWS = TM / WM;     // waves WM x 2; rows of a wave
    constexpr int FM = WROWS / 32, FN = TN / 64;           // 32 x 32 fragments per wave
    constexpr int ROUND = THREADS * 16;                    // bytes of a load round
    constexpr int AR = TM * 128 / ROUND, BR = TN * 128 / ROUND, R = AR + BR;
    constexpr int A_BYTES = TM * DT_KS * 2, STAGE = A_BYTES + TN * DT_KS * 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int t = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int l = t & 63, lr = l & 31, g = l >> 5;
    const int wm = WM == 4 ? w & 3 : w >> 1, wn = WM == 4 ? w >> 2 : w & 1;      // the two waves of a SIMD hold the same rows

    // the tile: each XCD takes one contiguous run of the order, super-rows of 1024 rows
    const int tiles_m = (int)((p.m + TM - 1) / TM), tiles_n = (int)((p.n + TN - 1) / TN);
    const int total = tiles_m * tiles_n * (SPLIT ? p.splits : 1), per_xcd = (total + 7) >> 3;
    const int in_xcd = (int)(blockIdx.x >> 3);
    int tile = (int)(blockIdx.x & 7) * per_xcd + in_xcd;
    if (in_xcd >= per_xcd || tile >= total) return;
    int split = 0;
    if (SPLIT) {            // the runs of one split follow each other: their tiles share operands
        split = tile / (tiles_m * tiles_n);
        tile -= split * (tiles_m * tiles_n);
    }
    int pid_m, pid_n;
    {
        constexpr int SUPER = 1024 / TM;
        const int width = SUPER * tiles_n, first = tile / width * SUPER;
        const int gsz = (tiles_m - first) < SUPER ? (tiles_m - first) : SUPER;
        pid_m = first + (tile % width) % gsz;
        pid_n = (tile % width) / gsz;
    }
    const int64_t m0 = (int64_t)pid_m * TM, n0 = (int64_t)pid_n * TN;
    const int m_valid = (int)((p.m - m0) < TM ? p.m - m0 : TM), n_valid = (int)((p.n - n0) < TN ? p.n - n0 : TN);
    const int all_slots = (int)((p.k + DT_KS - 1) / DT_KS), s_first = SPLIT ? split * p.split_slots : 0;
    const int slots = SPLIT && s_first + p.split_slots < all_slots ? s_first + p.split_slots : all_slots;      // the run's end
    // the last slot's second half may be past the contraction, in the next row: not multiplied.  (Contraction rows past the end are zeros.)
    const bool odd = !A_T && (p.k & 32) != 0;

    const int64_t lda = A_T ? p.m * 2 : p.k * 2, ldb = B_T ? p.n * 2 : p.k * 2;
    // the descriptors end with the operands; what is requested past them arrives as zeros
    const addr::Desc da = A_T ? addr::tall_cols_desc(0, p.k, lda, m0 * 2) : addr::tall_rows_desc(p.m, m0, lda);
    const addr::Desc db = B_T ? addr::tall_cols_desc(0, p.k, ldb, n0 * 2) : addr::tall_rows_desc(p.n, n0, ldb);
    const v4i ra = make_rsrc(p.a + da.base, da.records), rb = make_rsrc(p.b + db.base, db.records);
    const uint32_t a_step = (uint32_t)__builtin_amdgcn_readfirstlane(A_T ? (int)(DT_KS * lda) : DT_KS * 2);
    const uint32_t b_step = (uint32_t)__builtin_amdgcn_readfirstlane(B_T ? (int)(DT_KS * ldb) : DT_KS * 2);
    uint32_t va[AR], vb[BR];
#pragma unroll
    for (int e = 0; e < AR; ++e) va[e] = A_T ? addr::dense_cols_lane(t, e, THREADS, TM, lda) : addr::dense_rows_lane(t, e, THREADS, lda);
#pragma unroll
    for (int e = 0; e < BR; ++e) vb[e] = B_T ? addr::dense_cols_lane(t, e, THREADS, TN, ldb) : addr::dense_rows_lane(t, e, THREADS, ldb);
    const uint32_t wave_base = (uint32_t)(uintptr_t)smem + (uint32_t)(w * 1024);
    // requests of slot s into a stage; past the range they are dropped, but counted
    struct In {
        uint32_t base, sa, sb;
    };
    auto in_begin = [&](int s, int stage) __attribute__((always_inline)) {
        const bool in = s < slots;
        return In{wave_base + (uint32_t)(stage * STAGE), in ? (uint32_t)s * a_step : addr::kDropped, in ? (uint32_t)s * b_step : addr::kDropped};
    };
    auto request = [&](auto e_tag, const In& r) __attribute__((always_inline)) {
        constexpr int e = decltype(e_tag)::value;
        if constexpr (e < AR) dma16_at<e * ROUND>(ra, r.base, va[e], r.sa);
        else dma16_at<A_BYTES + (e - AR) * ROUND>(rb, r.base, vb[e - AR], r.sb);
    };

    // fragment reads: contiguous, row lr, piece 2 ks + g XOR (row / 2) % 8; transposed, this lane addresses row tj of a 4-row
    // group, 8-byte piece ta4 of its 16-lane block's 16 columns
    const int lane_c = lr * 128 + 16 * (g ^ ((lr >> 1) & 7));
    const int tj = (l & 15) >> 2, ta4 = l & 3, tblk = (l >> 4) & 1;
    struct Frag {
        d8bf a[FM], b[FN];
    };
    // 8 contraction elements of 32 columns from col0 on, of an operand staged as [contraction row][columns] with `pitch` bytes a row
    auto read_trans = [&](uint8_t* base, int pitch, int col0, int ks) __attribute__((always_inline)) {
        const int shift = pitch >= 256 ? 2 : 1;
        d8bf out;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = 16 * ks + 8 * g + 4 * h + tj, byte = 2 * col0 + 32 * tblk + 8 * ta4;
            uint8_t* ptr = base + row * pitch + 16 * ((byte >> 4) ^ ((row & 3) << shift)) + (byte & 15);
            const d4s v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) d4s*)ptr);
            const v4bf q = __builtin_bit_cast(v4bf, v);
            out[4 * h] = q[0]; out[4 * h + 1] = q[1]; out[4 * h + 2] = q[2]; out[4 * h + 3] = q[3];
        }
        return out;
    };
    auto read_a = [&](uint8_t* st, int i, int ks) __attribute__((always_inline)) {
        if constexpr (A_T) return read_trans(st, TM * 2, wm * WROWS + 32 * i, ks);
        else return *(const d8bf*)(st + ((lane_c + wm * WROWS * 128) ^ (32 * ks)) + i * 4096);
    };
    auto read_b = [&](uint8_t* st, int j, int ks) __attribute__((always_inline)) {
        if constexpr (B_T) return read_trans(st + A_BYTES, TN * 2, wn * (TN / 2) + 32 * j, ks);
        else return *(const d8bf*)(st + A_BYTES + ((lane_c + wn * (TN / 2) * 128) ^ (32 * ks)) + j * 4096);
    };

    v16f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const bool live = __builtin_amdgcn_readfirstlane(wm * WROWS < m_valid);

    static_for<0, ST - 1>([&](auto s) {
        const In r = in_begin(s_first + decltype(s)::value, decltype(s)::value);
        static_for<0, R>([&](auto e) { request(e, r); });
    });
    // A step's fragments are read behind the MFMAs of the step before (pinned: on its own the compiler reads them in front of their
    // MFMAs and waits).  A slot's barrier stands one MFMA into its last step: by then every wave holds all its fragments of the
    // slot, so its stage is free, and the next slot's first fragments and the requests of slot s + ST go out behind the MFMAs
    // that are left and those of the next step.  (Barrier in front of the slot, its first fragments behind it: 71 us instead of 58 for
    // [2048, 4096] x 4096, 48 instead of 41 for [2051, 2880] x 2880.)
    constexpr int NM = FM * FN, NX = FM + FN, NL = NM - 1;      // MFMAs and reads of a step; MFMAs behind the barrier
    constexpr int Q = NL + NM, E3 = NM == 1 ? R : NL * R / Q;   // places for requests; of them in the last step
    const int full = slots - s_first - (odd && slots == all_slots ? 1 : 0);      // slots of four steps
    int stage = 0;
    In in = in_begin(s_first + ST - 1, ST - 1);
    if (live) {
        static_for<0, E3>([&](auto e) { request(e, in); });
        wait_vm<(ST - 2) * R + E3>();       // the first slot has landed
        __syncthreads();
        Frag f[2];
        auto read = [&](auto x_tag, auto ks_tag, uint8_t* st) __attribute__((always_inline)) {
            constexpr int x = decltype(x_tag)::value, ks = decltype(ks_tag)::value;
            if constexpr (x < FN) f[ks & 1].b[x] = read_b(st, x, ks);
            else f[ks & 1].a[x - FN] = read_a(st, x - FN, ks);
        };
        auto multiply = [&](auto m_tag, auto ks_tag) __attribute__((always_inline)) {
            constexpr int m = decltype(m_tag)::value, ks = decltype(ks_tag)::value, i = m % FM, j = m / FM;
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[ks & 1].b[j], f[ks & 1].a[i], acc[i][j], 0, 0, 0);
        };
        auto step = [&](auto ks_tag, uint8_t* st) __attribute__((always_inline)) {       // ks 0 .. 2
            constexpr int ks = decltype(ks_tag)::value;
            static_for<0, NM>([&](auto m_tag) {
                constexpr int m = decltype(m_tag)::value;
                multiply(m_tag, ks_tag);
                static_for<m * NX / NM, (m + 1) * NX / NM>([&](auto x) { read(x, std::integral_constant<int, ks + 1>{}, st); });
                if constexpr (ks == 0 && NM > 1) {
                    constexpr int q = NL + m;
                    static_for<q * R / Q, (q + 1) * R / Q>([&](auto e) { request(e, in); });
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        constexpr std::integral_constant<int, 0> k0{};
        constexpr std::integral_constant<int, 3> k3{};
        static_for<0, NX>([&](auto x) { read(x, k0, smem); });
        for (int s = 0; s < full; ++s) {
            uint8_t* st = smem + stage * STAGE;
            const int nstage = stage == ST - 1 ? 0 : stage + 1;
            step(k0, st);
            step(std::integral_constant<int, 1>{}, st);
            step(std::integral_constant<int, 2>{}, st);
            multiply(k0, k3);
            wait_vm<(ST - 2) * R>();        // slot s + 1 has landed
            __syncthreads();                // ... for every wave, and every wave holds its fragments of slot s
            in = in_begin(s_first + s + ST, stage);
            __builtin_amdgcn_sched_barrier(0);
            uint8_t* nx = smem + nstage * STAGE;
            if constexpr (NM == 1) {
                static_for<0, NX>([&](auto x) { read(x, k0, nx); });
                static_for<0, R>([&](auto e) { request(e, in); });
            } else {
                static_for<1, NM>([&](auto m_tag) {
                    constexpr int m = decltype(m_tag)::value, q = m - 1;
                    multiply(m_tag, k3);
                    static_for<(q * NX + NL - 1) / NL, ((q + 1) * NX + NL - 1) / NL>([&](auto x) { read(x, k0, nx); });
                    static_for<q * R / Q, (q + 1) * R / Q>([&](auto e) { request(e, in); });
                    __builtin_amdgcn_sched_barrier(0);
                });
            }
            stage = nstage;
        }
        if (full < slots - s_first) {       // the contraction's last slot of two steps
            uint8_t* st = smem + stage * STAGE;
            step(k0, st);
            static_for<0, NM>([&](auto m_tag) { multiply(m_tag, std::integral_constant<int, 1>{}); });
        }
    } else {
        // none of the tile's rows are this wave's: it only keeps its share of the requests going
        static_for<0, R>([&](auto e) { request(e, in); });
        wait_vm<(ST - 1) * R>();
        __syncthreads();
        for (int s = 0; s < full; ++s) {
            wait_vm<(ST - 2) * R>();
            __syncthreads();
            in = in_begin(s_first + s + ST, stage);
            static_for<0, R>([&](auto e) { request(e, in); });
            stage = stage == ST - 1 ? 0 : stage + 1;
        }
    }
    wait_vm<0>();
    __syncthreads();                    // nothing reads or writes the stages any more

    if constexpr (SPLIT) {
        constexpr int FP = TN * 4 + 16, FL = TN / 4;        // the fp32 tile through LDS: bytes per row, lanes per row
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(v4f*)(smem + (wm * WROWS + i * 32 + lr) * FP + (wn * (TN / 2) + j * 32 + 8 * q + 4 * g) * 4) =
                        v4f{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        __syncthreads();
        const int fr = t / FL, fc = (t % FL) * 4;
        float* out = p.partial + ((int64_t)split * p.m + m0) * p.n + n0 + fc;
        if (fc < n_valid) {
#pragma unroll
            for (int u = 0; u < TM / (THREADS / FL); ++u) {
                const int row = u * (THREADS / FL) + fr;
                if (row < m_valid) *(v4f*)(out + (int64_t)row * p.n) = *(const v4f*)(smem + row * FP + fc * 4);
            }
        }
        return;
    }

    // ---- epilogue.  Lane (lr, g) of fragment (i, j) holds row 32 i + lr, columns 32 j + 8 q + 4 g .. + 3 in registers 4 q .. + 3.  The
    // tile passes through LDS as bf16 in rows of 16-byte pieces: z on its way out, the residual on its way in (each lane then
    // finds its own four columns' values where it puts its results), y on its way out. ----
    constexpr int PITCH = TN * 2 + 16, LPR = TN / 8, RPI = THREADS / LPR;
    const int rr0 = t / LPR, cc = (t % LPR) * 8;
    const int64_t c0 = m0 * p.n + n0;
    auto spot = [&](int i, int j, int q) __attribute__((always_inline)) {
        return (uint2*)(smem + (wm * WROWS + i * 32 + lr) * PITCH + (wn * (TN / 2) + j * 32 + 8 * q + 4 * g) * 2);
    };
    auto leave = [&](uint16_t* out) __attribute__((always_inline)) {
        if (cc < n_valid) {
#pragma unroll
            for (int u = 0; u < TM / RPI; ++u) {
                const int row = u * RPI + rr0;
                if (row < m_valid) store16_streaming((uint8_t*)(out + c0 + (int64_t)row * p.n + cc), *(const uint4*)(smem + row * PITCH + cc * 2));
            }
        }
    };
    uint4 rr[TM / RPI];             // the residual, asked for while z is on its way out
    if (p.epi.residual && cc < n_valid) {
#pragma unroll
        for (int u = 0; u < TM / RPI; ++u) {
            const int row = u * RPI + rr0;
            rr[u] = row < m_valid ? load16_streaming(p.epi.residual + c0 + (int64_t)row * p.n + cc) : make_uint4(0, 0, 0, 0);
        }
    }
    if (p.epi.bias) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = wn * (TN / 2) + j * 32 + 8 * q + 4 * g;
                if (col < n_valid) {        // n is a multiple of 32: four columns are in or out together
                    const v4f b4 = epi_bias4(p.epi, n0 + col);
#pragma unroll
                    for (int i = 0; i < FM; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += b4[e];
                }
            }
    }
    auto quad = [&](int i, int j, int q) __attribute__((always_inline)) {
        return v4f{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    };
    if (p.epi.z) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) *spot(i, j, q) = pack4(quad(i, j, q));
        __syncthreads();
        leave(p.epi.z);
        __syncthreads();
    }
    if (p.epi.residual) {
        if (cc < n_valid) {
#pragma unroll
            for (int u = 0; u < TM / RPI; ++u) {
                const int row = u * RPI + rr0;
                *(uint4*)(smem + row * PITCH + cc * 2) = rr[u];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                v4f y = quad(i, j, q);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = epi_act<ACT>(y[e]);
                if (p.epi.residual) {
                    const v4f r = unpack4(*spot(i, j, q));
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] += r[e];
                }
                *spot(i, j, q) = pack4(y);
            }
    __syncthreads();
    leave(p.c);
}

// The runs of a split contraction added up in their order, and the epilogue, or the addition to a float buffer: eight columns of a row per
// thread.
template <int ACT>
__global__ __launch_bounds__(256) void dense_join_kernel(DenseArgs p) {
    const int64_t mn = p.m * p.n, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (at >= mn) return;
    const int64_t col = at % p.n;
    v4f lo = *(const v4f*)(p.partial + at), hi = *(const v4f*)(p.partial + at + 4);
    for (int s = 1; s < p.splits; ++s) {
        lo += *(const v4f*)(p.partial + s * mn + at);
        hi += *(const v4f*)(p.partial + s * mn + at + 4);
    }
    if (p.sum) {
        *(v4f*)(p.sum + at) += lo;
        *(v4f*)(p.sum + at + 4) += hi;
        return;
    }
    lo += epi_bias4(p.epi, col);
    hi += epi_bias4(p.epi, col + 4);
    if (p.epi.z) {
        const uint2 a = pack4(lo), b = pack4(hi);
        *(uint4*)(p.epi.z + at) = make_uint4(a.x, a.y, b.x, b.y);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) lo[e] = epi_act<ACT>(lo[e]), hi[e] = epi_act<ACT>(hi[e]);
    if (p.epi.residual) {
        const uint4 r = *(const uint4*)(p.epi.residual + at);
        lo += unpack4(make_uint2(r.x, r.y));
        hi += unpack4(make_uint2(r.z, r.w));
    }
    const uint2 a = pack4(lo), b = pack4(hi);
    *(uint4*)(p.c + at) = make_uint4(a.x, a.y, b.x, b.y);
}

// ---- up to 16 rows: bound by reading b once.  A workgroup has 16 NT columns; its 8 waves split the contraction, load the fragments
// straight into registers (16 rows of 64 bytes per request, FEW_AHEAD steps on their way) and join their sums through LDS.  b
// through the caches, although it is read once: weights up to the memory-side cache's size stay there from one token to the next.
// us, weight cached / from memory: one row by [14336, 4096] 21.5 / 24.9, past the caches 25.4 / 27.4 (the weight alone is 24.6 at the rate of a
// large copy); [4096, 14336] 19.3 / 24.0, with 8 steps on their way 20.9 / 28.8.  32 columns to a workgroup where that still gives 256 of them, for
// the rows' sake: 16 rows by [14336, 4096] 31.5 / 39.0 -> 25.2 / 33.7. ----
constexpr int FEW_AHEAD = 4;
template <int NT, int ACT>
__global__ __launch_bounds__(8 * 64) void dense_few_rows_kernel(DenseArgs p) {
    constexpr int AHEAD = FEW_AHEAD, WAVES = 8;
    __shared__ v4f part[WAVES][NT][64];
    const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), l = t & 63;
    const int row = l & 15, q = l >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);       // n is a multiple of 32: the columns exist
    const int steps = (int)(p.k / 32), per = (steps + WAVES - 1) / WAVES;
    const int s0 = w * per, s1 = s0 + per < steps ? s0 + per : steps;
    const uint8_t* b = p.b + (n0 + row) * p.k * 2 + q * 16;
    const uint8_t* a = p.a + (row < p.m ? row : p.m - 1) * p.k * 2 + q * 16;      // (a row past the end is another one's copy, not stored)
    const int64_t b_tile = p.k * 32;
    v4f acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
    int s = s0;
    for (; s + AHEAD <= s1; s += AHEAD) {
        d8bf fb[AHEAD][NT], fa[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
            for (int j = 0; j < NT; ++j) fb[u][j] = *(const d8bf*)(b + (int64_t)(s + u) * 64 + j * b_tile);
            fa[u] = *(const d8bf*)(a + (int64_t)(s + u) * 64);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[u][j], fa[u], acc[j], 0, 0, 0);
    }
    for (; s < s1; ++s) {
        const d8bf fa = *(const d8bf*)(a + (int64_t)s * 64);
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const d8bf*)(b + (int64_t)s * 64 + j * b_tile), fa, acc[j], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) part[w][j][l] = acc[j];
    __syncthreads();
    // lane (row of a = l % 16, columns 4 (l / 16) .. + 3)
    if (t < NT * 64) {
        const int j = t >> 6;
        const int64_t r = l & 15, col = n0 + 16 * j + 4 * (l >> 4);
        v4f z = part[0][j][l];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) z += part[k][j][l];
        if (r >= p.m) return;
        z += epi_bias4(p.epi, col);
        if (p.epi.z) *(uint2*)(p.epi.z + r * p.n + col) = pack4(z);
        v4f y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = epi_act<ACT>(z[e]);
        if (p.epi.residual) y += unpack4(*(const uint2*)(p.epi.residual + r * p.n + col));
        *(uint2*)(p.c + r * p.n + col) = pack4(y);
    }
}

// ---- the elementwise part of the backward: dz = dy act'(z) (not written without an activation) and column sums of dz.
// A workgroup has 256 columns (8 a lane) and a run of rows, 8 at a time; its sums go to partial[run][n], which a second launch
// adds up in order.  dz is rounded to bf16, the type of both gradient products' operands (an fp32 dz would be split into several bf16
// products); the bias gradient's sums are of dz before that.  With z in bf16, the activation's slope is that of the rounded z: together the
// gradients of [2051, 2880] x 2880 with GELU are 2.4e-3 of their norm off the definition, one rounding to bf16 alone 1.7e-3. ----
struct DzArgs {
    const uint16_t* dy;
    const uint16_t* z;
    uint16_t* dz;
    float* partial;         // [runs, n]; null: no sums wanted, or one run, which writes dbias itself
    int64_t m, n, run;      // rows per workgroup
    void* dbias;
    int f32;
};
__device__ __forceinline__ void put_dbias(void* dbias, int f32, int64_t col, float s) {
    if (f32) ((float*)dbias)[col] = s;
    else ((__bf16*)dbias)[col] = (__bf16)s;
}
template <int ACT>
__global__ __launch_bounds__(256) void dense_dz_kernel(DzArgs p) {
    __shared__ float sums[8][32][9];
    const int lane = threadIdx.x & 31, r8 = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 256 + lane * 8;
    const int64_t lo = (int64_t)blockIdx.y * p.run, hi = lo + p.run < p.m ? lo + p.run : p.m;
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    if (col < p.n) {
        for (int64_t r = lo + r8; r < hi; r += 8) {
            const uint4 d = ACT == kActNone ? *(const uint4*)(p.dy + r * p.n + col) : load16_streaming(p.dy + r * p.n + col);
            const uint32_t dw[4] = {d.x, d.y, d.z, d.w};
            float x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[2 * e] = bf16_lo(dw[e]), x[2 * e + 1] = bf16_hi(dw[e]);
            if constexpr (ACT != kActNone) {
                const uint4 zz = load16_streaming(p.z + r * p.n + col);
                const uint32_t zw[4] = {zz.x, zz.y, zz.z, zz.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[2 * e] *= epi_slope<ACT>(bf16_lo(zw[e]));
                    x[2 * e + 1] *= epi_slope<ACT>(bf16_hi(zw[e]));
                }
                *(uint4*)(p.dz + r * p.n + col) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += x[e];
        }
    }
    if (!p.partial && !p.dbias) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[r8][lane][e] = acc[e];
    __syncthreads();
    const int c = threadIdx.x;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += sums[i][c >> 3][c & 7];
    const int64_t at = (int64_t)blockIdx.x * 256 + c;
    if (at >= p.n) return;
    if (p.partial) p.partial[(int64_t)blockIdx.y * p.n + at] = s;
    else put_dbias(p.dbias, p.f32, at, s);
}

// dbias[n] = sum of the runs: 32 columns by 32 groups of runs, four loads on their way
__global__ __launch_bounds__(1024) void dense_dbias_kernel(const float* partial, int runs, int64_t n, void* dbias, int f32) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + lane;       // n is a multiple of 32
    float s = 0.f;
    for (int r0 = w; r0 < runs; r0 += 32 * 4) {
        float x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = r0 + 32 * u < runs ? partial[(int64_t)(r0 + 32 * u) * n + col] : 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u) s += x[u];
    }
    part[w][lane] = s;
    __syncthreads();
    if (w == 0) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += part[i][lane];
        put_dbias(dbias, f32, col, s);
    }
}

// rows per workgroup of dense_dz_kernel: about 2048 workgroups, a multiple of 8 rows.  Up to 64 rows are one run, whose workgroups write the
// bias gradient themselves: eight rounds of loads instead of a second launch.
static int64_t dz_run(int64_t m, int64_t n) {
    if (m <= 64) return 64;
    const int64_t cols = (n + 255) / 256;
    int64_t runs = 2048 / cols;
    if (runs < 1) runs = 1;
    int64_t run = (m + runs - 1) / runs;
    return (run + 7) / 8 * 8 < 8 ? 8 : (run + 7) / 8 * 8;
}

template <int TM, int TN, int WM, int ST, bool A_T, bool B_T, int ACT, bool SPLIT = false>
static int launch_dense_tile(const DenseArgs& a, hipStream_t st) {
    constexpr int lds = dense_lds_bytes<TM, TN, ST, SPLIT>();
    static std::atomic<bool> attr_set[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return MXL_ELAUNCH;
    auto kern = dense_tile_kernel<TM, TN, WM, ST, A_T, B_T, ACT, SPLIT>;
    if (!attr_set[dev & 63].load(std::memory_order_acquire)) {
        if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return MXL_ELAUNCH;
        attr_set[dev & 63].store(true, std::memory_order_release);
    }
    const int64_t tiles = ((a.m + TM - 1) / TM) * ((a.n + TN - 1) / TN) * (SPLIT ? a.splits : 1), grid = (tiles + 7) / 8 * 8;
    if (grid > 0x7FFFFFFF) return MXL_EINVAL;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(WM * 128), lds, st, a);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}

// How a product runs: tiles of 256 x 256 where they fill the chip; below that whichever of the four tiles, with the contraction in one
// or several runs, these figures make the soonest done.  us of a slot of 64 elements, half with the weight cached and half with it from
// memory, by the workgroups there are (w, of 256 CUs):
//   256 x 256  1.12 + 0.42 w / 256                    one on a CU
//   256 x 128  0.54 + 0.28 (w / 256)^2                one on a CU; 0.52 (w / 256)^2 for the weight gradient, which reads both operands transposed
//   64 x 64    0.30 up to 256, 0.45 with two on every CU, 0.63 with three
// and a split costs 4 us for the second launch and its fp32 sums' way out and in at 7 TB/s.  The figures are from launch to launch of a replayed graph
// with a cached and no residual: [333, 14336] x 4096 in four runs, 50 / 53 there and 56 / 58 on another board, is 62 with a, residual and weight all from
// memory, and in a trace of single launches 60 + 7 for the join.  Forward, us, weight cached / from memory, 256 x 256,
// 256 x 128 and 64 x 64 unsplit: [2048, 4096] x 4096 88 / 82, 58 / 61, 108 / 118; [1500, 2880] x 2880 55 / 66, 31 / 37, 46 / 51;
// [4096, 2880] x 2880 77 / 69, 73 / 77, 118 / 121; [1000, 2048] x 2048 41 / 48, 23 / 27, 15 / 18.  256 x 128 in several runs: [333, 14336] x
// 4096 120 / 133, four 50 / 53 (64 x 64 unsplit 76 / 104); [700, 4096] x 4096 40 / 47, two 34 / 36; [2048, 8192] x 2048 82 / 85, two
// 68 / 70.  (128 x 128, two workgroups on a CU, is level with 256 x 128 where the weight is cached and behind where it is not: 62 / 70, 34 / 41, 75 / 92
// for the first three; [333, 14336] x 4096 in four 53 / 65.)
// Weight gradient [m, n]^T . [m, k], us, 256 x 256 (the grouped kernel with one group) / 256 x 128 / 64 x 64, unsplit, best split: 2051, 2880, 2880
// 50 / 54 / 60; 1000, 2048, 2048 23 / 15 / 17; 4096, 1024, 4096 70 / 44 / 65, two runs 43; 8192, 2048, 1024 137 / 75 / 59, four runs of
// 256 x 128 43; 8192, 256, 512 131 / 72 / 33, eight runs of 64 x 64 12; 300, 512, 1120 11 / - / 4.
struct DensePlan {
    int tm, tn;         // output tile
    int splits;         // runs of the contraction, 1: not split
    int slots;          // slots per run
};
static DensePlan dense_plan(int64_t m, int64_t n, int64_t k, bool a_by_columns = false) {
    auto tiles = [&](int tm, int tn) { return ((m + tm - 1) / tm) * ((n + tn - 1) / tn); };
    const int slots = (int)((k + DT_KS - 1) / DT_KS);
    DensePlan best{256, 256, 1, slots};
    const double tall = (double)tiles(256, 256);
    if (tall >= 256) return best;
    double least = slots * (1.12 + 0.42 * tall / 256);
    auto consider = [&](int tm, int tn, double held, auto us_of) {
        for (int s = 1; s <= 16; ++s) {
            const int per = (slots + s - 1) / s;
            if ((s > 1 && per < 4) || (slots + per - 1) / per != s) continue;
            const double wgs = (double)(tiles(tm, tn) * s), rounds = wgs / held;
            // workgroups beyond those the chip holds start as others end: between their share of a round and a whole one
            const double passes = rounds <= 1.0 ? 1.0 : 0.5 * (rounds + (double)(int64_t)(rounds + 0.999999));
            const double us = passes * per * us_of((rounds < 1.0 ? wgs : held) / 256) + (s > 1 ? 4.0 + (double)s * (double)m * (double)n * 8.0 / 7e6 : 0.0);
            if (us < least) least = us, best = {tm, tn, s, per};
        }
    };
    auto part = [](double x, double lo, double hi) { return x <= lo ? 0.0 : x >= hi ? 1.0 : (x - lo) / (hi - lo); };
    consider(256, 128, 256, [&](double w) { return 0.54 + (a_by_columns ? 0.52 : 0.28) * w * w; });
    consider(64, 64, 768, [&](double w) { return 0.30 + 0.15 * part(w, 1.0, 2.0) + 0.18 * part(w, 2.0, 3.0); });
    return best;
}

template <bool A_T, bool B_T, int ACT>
static int launch_dense(DenseArgs a, const DensePlan& plan, hipStream_t st) {
    if (plan.splits == 1 && !a.sum) {
        if (plan.tm == 256) return launch_dense_tile<256, 128, 4, 3, A_T, B_T, ACT>(a, st);
        return launch_dense_tile<64, 64, 2, 3, A_T, B_T, ACT>(a, st);
    }
    a.splits = plan.splits;
    a.split_slots = plan.slots;
    const int rc = plan.tm == 256 ? launch_dense_tile<256, 128, 4, 3, A_T, B_T, kActNone, true>(a, st)
                                  : launch_dense_tile<64, 64, 2, 3, A_T, B_T, kActNone, true>(a, st);
    if (rc != MXL_OK) return rc;
    hipLaunchKernelGGL(dense_join_kernel<ACT>, dim3((unsigned)((a.m * a.n / 8 + 255) / 256)), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}

constexpr int64_t FEW_ROWS = 16;
template <int ACT>
static int launch_dense_forward(const DenseArgs& a, const DensePlan& plan, hipStream_t st) {
    if (a.m <= FEW_ROWS) {
        if (a.n / 32 >= 256) hipLaunchKernelGGL((dense_few_rows_kernel<2, ACT>), dim3((unsigned)(a.n / 32)), dim3(8 * 64), 0, st, a);
        else hipLaunchKernelGGL((dense_few_rows_kernel<1, ACT>), dim3((unsigned)(a.n / 16)), dim3(8 * 64), 0, st, a);
        return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
    }
    if (plan.tn == 256) {
        const Bf16Args t{a.a, a.b, a.c, nullptr, 1, a.m, 0, a.n, a.k, a.epi};
        return launch_bf16_linear_tall(t, ACT, st);
    }
    return launch_dense<false, false, ACT>(a, plan, st);
}

// (offsets inside a tile's operand rows are 32-bit: 256 rows of k or n stay below 2^31 bytes)
static bool dense_sizes_ok(int64_t m, int64_t n, int64_t k) {
    return m >= 0 && m <= 0x7FFFFFFF && n > 0 && n % 32 == 0 && k > 0 && k % 32 == 0 && n <= (1 << 21) && k <= (1 << 21) && n * k * 2 < ((int64_t)1 << 32);
}
// the weight gradient contracts over the m rows, whose number is free; its operands end below 4 GiB
static bool dense_wgrad_ok(int64_t m, int64_t n, int64_t k) { return dense_sizes_ok(m, n, k) && m * (n > k ? n : k) * 2 < ((int64_t)1 << 32); }
// fp32 sums of a product's runs [m, n] (a product that is added to a float buffer goes through them with one run too)
static int64_t runs_bytes(const DensePlan& plan, int64_t m, int64_t n, bool accum = false) {
    return plan.splits > 1 || (accum && plan.tn != 256) ? plan.splits * m * n * 4 : 0;
}
// The weight gradient runs on this file's tiles unless it has enough large ones, or no rows, or offsets that pass 32 bits in the 63 rows
// behind the last one
static DensePlan wgrad_plan(int64_t m, int64_t n, int64_t k) {
    if (m == 0 || (m + 64) * (n > k ? n : k) * 2 >= ((int64_t)1 << 32)) return {256, 256, 1, 0};
    return dense_plan(n, k, m, true);
}
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace mxl

using namespace mxl;

extern "C" int64_t mxl_linear_bf16_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (!dense_sizes_ok(m, n, k)) return -1;
    return m == 0 ? 0 : runs_bytes(dense_plan(m, n, k), m, n);
}

extern "C" int64_t mxl_linear_bf16_forward_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (!dense_sizes_ok(m, n, k)) return -1;
    return m <= FEW_ROWS ? 0 : runs_bytes(dense_plan(m, n, k), m, n);
}

extern "C" int mxl_linear_bf16_plan(int64_t m, int64_t n, int64_t k, int a_by_columns, int* tile_rows, int* tile_cols, int* splits) {
    if (!dense_sizes_ok(m, n, 32) || m == 0 || k <= 0 || k > 0x7FFFFFFF || !tile_rows || !tile_cols || !splits) return MXL_EINVAL;
    const DensePlan plan = dense_plan(m, n, k, a_by_columns != 0);
    *tile_rows = plan.tm, *tile_cols = plan.tn, *splits = plan.splits;
    return MXL_OK;
}

extern "C" int mxl_linear_bf16(const void* a_bf16, const void* b_bf16, const void* bias, int bias_dtype, int act, const void* residual_bf16, int64_t m,
                               int64_t n, int64_t k, void* y_bf16, void* z_bf16, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!dense_sizes_ok(m, n, k) || act < MXL_ACT_SILU || act > MXL_ACT_NONE || (bias_dtype != MXL_DT_F32 && bias_dtype != MXL_DT_BF16)) return MXL_EINVAL;
    if (m == 0) return MXL_OK;
    if (!a_bf16 || !b_bf16 || !y_bf16) return MXL_EINVAL;
    if (!aligned16(a_bf16) || !aligned16(b_bf16) || !aligned16(bias) || !aligned16(residual_bf16) || !aligned16(y_bf16) || !aligned16(z_bf16)) return MXL_EINVAL;
    const DensePlan plan = m > FEW_ROWS ? dense_plan(m, n, k) : DensePlan{};
    const int64_t need = m > FEW_ROWS ? runs_bytes(plan, m, n) : 0;
    if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    DenseArgs d{(const uint8_t*)a_bf16, (const uint8_t*)b_bf16, (uint16_t*)y_bf16, m, n, k, {bias, (const uint16_t*)residual_bf16, (uint16_t*)z_bf16, bias_dtype == MXL_DT_F32}, (float*)workspace, 1, 0, nullptr};
    hipStream_t st = (hipStream_t)stream;
    switch (act) {
        case MXL_ACT_SILU: return launch_dense_forward<kActSilu>(d, plan, st);
        case MXL_ACT_GELU: return launch_dense_forward<kActGelu>(d, plan, st);
        case MXL_ACT_RELU: return launch_dense_forward<kActRelu>(d, plan, st);
        default: return launch_dense_forward<kActNone>(d, plan, st);
    }
}

namespace mxl {
// da [m, k] = dz [m, n] . b [n, k]: the contraction is over n, b's slow dim
static int run_dgrad(const DensePlan& plan, const void* dz, const void* b, int64_t m, int64_t n, int64_t k, void* da, void* workspace, int64_t workspace_bytes,
                     void* stream) {
    if (!dz || !b || !da || !aligned16(dz) || !aligned16(b) || !aligned16(da)) return MXL_EINVAL;
    const int64_t need = runs_bytes(plan, m, k);
    if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    if (plan.tn == 256) return mxl_grouped_gemm_bf16(dz, b, da, nullptr, 1, m, k, n, MXL_BF_B_KN | MXL_BF_TILE_256, stream);
    DenseArgs d{(const uint8_t*)dz, (const uint8_t*)b, (uint16_t*)da, m, k, n, {nullptr, nullptr, nullptr, 0}, (float*)workspace, 1, 0, nullptr};
    return launch_dense<false, true, kActNone>(d, plan, (hipStream_t)stream);
}
// db [n, k] = dz [m, n]^T . a [m, k]
static int run_wgrad(const DensePlan& plan, const void* dz, const void* a, int64_t m, int64_t n, int64_t k, void* db, uint32_t flags, void* workspace,
                     int64_t workspace_bytes, void* stream) {
    if (plan.tn == 256) return mxl_grouped_gemm_bf16_wgrad(dz, a, db, nullptr, 1, m, n, k, flags, stream);      // one group
    if (!dz || !a || !db || !aligned16(dz) || !aligned16(a) || !aligned16(db)) return MXL_EINVAL;
    const bool accum = (flags & MXL_BF_ACCUM_F32) != 0;
    const int64_t need = runs_bytes(plan, n, k, accum);
    if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    DenseArgs d{(const uint8_t*)dz, (const uint8_t*)a, accum ? nullptr : (uint16_t*)db, n, k, m, {nullptr, nullptr, nullptr, 0}, (float*)workspace, 1, 0, accum ? (float*)db : nullptr};
    return launch_dense<true, true, kActNone>(d, plan, (hipStream_t)stream);
}
}  // namespace mxl

extern "C" int mxl_linear_bf16_dgrad(const void* dz_bf16, const void* b_bf16, int64_t m, int64_t n, int64_t k, void* da_bf16, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
    if (!dense_sizes_ok(m, n, k)) return MXL_EINVAL;
    if (m == 0) return MXL_OK;
    return run_dgrad(dense_plan(m, k, n), dz_bf16, b_bf16, m, n, k, da_bf16, workspace, workspace_bytes, stream);
}

extern "C" int64_t mxl_linear_bf16_wgrad_workspace_bytes(int64_t m, int64_t n, int64_t k, uint32_t flags) {
    if (!dense_wgrad_ok(m, n, k) || (flags & ~(uint32_t)MXL_BF_ACCUM_F32)) return -1;
    return runs_bytes(wgrad_plan(m, n, k), n, k, (flags & MXL_BF_ACCUM_F32) != 0);
}

extern "C" int mxl_linear_bf16_wgrad(const void* dz_bf16, const void* a_bf16, int64_t m, int64_t n, int64_t k, void* db, uint32_t flags, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
    if (!dense_wgrad_ok(m, n, k) || (flags & ~(uint32_t)MXL_BF_ACCUM_F32)) return MXL_EINVAL;
    return run_wgrad(wgrad_plan(m, n, k), dz_bf16, a_bf16, m, n, k, db, flags, workspace, workspace_bytes, stream);
}

extern "C" int64_t mxl_linear_bf16_dz_workspace_bytes(int64_t m, int64_t n) {
    if (m < 0 || n <= 0) return -1;
    const int64_t run = dz_run(m, n), runs = (m + run - 1) / run;
    return runs > 1 ? runs * n * 4 : 0;
}

extern "C" int mxl_linear_bf16_dz(const void* dy_bf16, const void* z_bf16, int act, int64_t m, int64_t n, void* dz_bf16, void* dbias, int dbias_dtype,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
    if (!dense_sizes_ok(m, n, 32) || act < MXL_ACT_SILU || act > MXL_ACT_NONE || (dbias_dtype != MXL_DT_F32 && dbias_dtype != MXL_DT_BF16)) return MXL_EINVAL;
    if (m > 0 && (!dy_bf16 || (act != MXL_ACT_NONE && (!z_bf16 || !dz_bf16)))) return MXL_EINVAL;
    if (!aligned16(dy_bf16) || !aligned16(z_bf16) || !aligned16(dz_bf16) || !aligned16(workspace)) return MXL_EINVAL;
    const int64_t need = dbias ? mxl_linear_bf16_dz_workspace_bytes(m, n) : 0;
    if (need > 0 && (!workspace || workspace_bytes < need)) return MXL_EINVAL;
    if (!dbias && (act == MXL_ACT_NONE || m == 0)) return MXL_OK;
    if (!device_is_gfx950()) return MXL_ENODEV;
    hipStream_t st = (hipStream_t)stream;
    const int64_t run = dz_run(m, n), runs = (m + run - 1) / run;
    DzArgs d{(const uint16_t*)dy_bf16, (const uint16_t*)z_bf16, (uint16_t*)dz_bf16, need > 0 ? (float*)workspace : nullptr, m, n, run, dbias, dbias_dtype == MXL_DT_F32};
    const dim3 grid((unsigned)((n + 255) / 256), (unsigned)runs);
    if (m > 0) {
        if (act == MXL_ACT_SILU) hipLaunchKernelGGL(dense_dz_kernel<kActSilu>, grid, dim3(256), 0, st, d);
        else if (act == MXL_ACT_GELU) hipLaunchKernelGGL(dense_dz_kernel<kActGelu>, grid, dim3(256), 0, st, d);
        else if (act == MXL_ACT_RELU) hipLaunchKernelGGL(dense_dz_kernel<kActRelu>, grid, dim3(256), 0, st, d);
        else hipLaunchKernelGGL(dense_dz_kernel<kActNone>, grid, dim3(256), 0, st, d);
    }
    if (dbias && runs != 1) hipLaunchKernelGGL(dense_dbias_kernel, dim3((unsigned)(n / 32)), dim3(1024), 0, st, (const float*)workspace, (int)runs, n, dbias, dbias_dtype == MXL_DT_F32);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}

// ---- the whole backward in one call ----
namespace mxl {
static int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }
struct BwdSpace {
    DensePlan dgrad, wgrad;
    int64_t dz, sums, runs, total;      // bytes: dz (with an activation), dbias's partial sums, the split sums of dgrad, then of the weight gradient
};
static BwdSpace bwd_space(int64_t m, int64_t n, int64_t k, int act, bool need_da, bool need_db, uint32_t db_flags, bool need_dbias) {
    BwdSpace s{};
    s.dz = act == MXL_ACT_NONE ? 0 : up256(m * n * 2);
    s.sums = need_dbias ? up256(mxl_linear_bf16_dz_workspace_bytes(m, n)) : 0;
    int64_t da = 0, db = 0;
    if (need_da && m > 0) s.dgrad = dense_plan(m, k, n), da = runs_bytes(s.dgrad, m, k);
    if (need_db) s.wgrad = wgrad_plan(m, n, k), db = runs_bytes(s.wgrad, n, k, (db_flags & MXL_BF_ACCUM_F32) != 0);
    s.runs = up256(da > db ? da : db);
    s.total = s.dz + s.sums + s.runs;
    return s;
}
}  // namespace mxl

extern "C" int64_t mxl_linear_bf16_bwd_workspace_bytes(int64_t m, int64_t n, int64_t k, int act, int need_da, int need_db, uint32_t db_flags,
                                                       int need_dbias) {
    if (!dense_sizes_ok(m, n, k) || act < MXL_ACT_SILU || act > MXL_ACT_NONE || (need_db && !dense_wgrad_ok(m, n, k)) ||
        (db_flags & ~(uint32_t)MXL_BF_ACCUM_F32))
        return -1;
    return bwd_space(m, n, k, act, need_da != 0, need_db != 0, db_flags, need_dbias != 0).total;
}

extern "C" int mxl_linear_bf16_bwd(const void* dy_bf16, const void* a_bf16, const void* b_bf16, const void* z_bf16, int act, int64_t m, int64_t n, int64_t k,
                                   void* da_bf16, void* db, uint32_t db_flags, void* dbias, int dbias_dtype, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
    if (!dense_sizes_ok(m, n, k) || act < MXL_ACT_SILU || act > MXL_ACT_NONE || (db_flags & ~(uint32_t)MXL_BF_ACCUM_F32) ||
        (db && !dense_wgrad_ok(m, n, k)))
        return MXL_EINVAL;
    const BwdSpace sp = bwd_space(m, n, k, act, da_bf16 != nullptr, db != nullptr, db_flags, dbias != nullptr);
    if (sp.total > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < sp.total)) return MXL_EINVAL;
    if (da_bf16 && m > 0 && !b_bf16) return MXL_EINVAL;
    uint8_t* at = (uint8_t*)workspace;
    void* dz = sp.dz ? at : nullptr;
    int rc = MXL_OK;
    if (da_bf16 || db || dbias)
        rc = mxl_linear_bf16_dz(dy_bf16, z_bf16, act, m, n, dz, dbias, dbias_dtype, at + sp.dz, sp.sums, stream);
    const void* d = sp.dz ? dz : dy_bf16;
    if (rc == MXL_OK && da_bf16 && m > 0) rc = run_dgrad(sp.dgrad, d, b_bf16, m, n, k, da_bf16, at + sp.dz + sp.sums, sp.runs, stream);
    if (rc == MXL_OK && db) rc = run_wgrad(sp.wgrad, d, a_bf16, m, n, k, db, db_flags, at + sp.dz + sp.sums, sp.runs, stream);
    return rc;
}
