// Root-mean-square norm with the residual's addition (dist_op_rmsnorm) and its backward (dist_op_rmsnorm_bwd).
//   h = x + res;  rstd = 1 / sqrt(mean_c h^2 + eps);  y = h rstd w
//   g = dy w, n = h rstd:  dh = rstd (g - n mean_c(g n)) + dres;  dw = sum_rows dy n
// HBM-bound: a row is read once and stays in the registers of its lanes between the statistics and the output, which is y in the input's type, y in e4m3 with one
// scale per row, or y in MXFP4 - the operands of dist_op_gemm_nt (DIST_EPI_FP8) and dist_op_gemm_mxfp4 - so that no separate quantisation pass reads y again.
// Everything between the loads and the one rounding of an output is fp32: y is formed from the unrounded x + res, not from the stored h.
#include "mx.h"

namespace {

constexpr int NT = 256;

// sum / maximum over the LPR lanes that own a row; every lane gets the result.  LPR = 256 or 512: the whole block, `red` = 4 or 8 words of LDS, fixed order
template <int LPR> DEV float row_sum(float v, float* red) {
    if constexpr (LPR <= 64) return wave_sum(v, LPR);
    v = wave_sum(v, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    const float s = (red[0] + red[1]) + (red[2] + red[3]);
    if constexpr (LPR == 512) return s + ((red[4] + red[5]) + (red[6] + red[7]));
    return s;
}
template <int LPR> DEV float row_max(float v, float* red) {
    if constexpr (LPR <= 64) return wave_max(v, LPR);
    v = wave_max(v, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// e4m3 factor and scale of a row whose largest |y| is a: those of dist_op_quant_rows_fp8 down to 2^-100; below that a counts as 2^-100 (448 / a would overflow)
DEV float e4m3_factor(float a, float& scale) {
    const float b = fmaxf(a, 7.8886090522101181e-31f);
    scale = a > 0.f ? b / 448.f : 1.f;
    return a > 0.f ? 448.f / b : 1.f;
}

// eight neighbouring values of a row from column c on -> the output of format FMT; the four lanes of a block of 32 are neighbours and all of them call
template <typename T, bool AL, int FMT>
DEV void put(const dist_rms_args& p, const float y[8], float inv, long row, long c, int Kp) {
    const long left = p.C - c;
    if constexpr (FMT == DIST_RMS_SAME) mx::store8<AL>(static_cast<T*>(p.y) + row * p.ldy + c, left, y);
    else if constexpr (FMT == DIST_RMS_E4M3) {
        int lo = 0, hi = 0;
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inv, y[1] * inv, lo, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inv, y[3] * inv, lo, true);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * inv, y[5] * inv, hi, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * inv, y[7] * inv, hi, true);
        unsigned char* q = static_cast<unsigned char*>(p.y) + row * p.ldy + c;
        if constexpr (AL) {
            const mx::i32x2_t w = {lo, hi};
            if (left > 0) __builtin_nontemporal_store(w, reinterpret_cast<mx::i32x2_t*>(q));
        } else {
            const unsigned long w = (unsigned)lo | (unsigned long)(unsigned)hi << 32;
            if (left >= 8) __builtin_memcpy(q, &w, 8);
            else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < left) q[e] = (unsigned char)(w >> (8 * e));
            }
        }
    } else {
        unsigned a = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) a = max(a, mx::abs_bits(y[e]));
        a = max(a, (unsigned)__shfl_xor((int)a, 1, 64));
        a = max(a, (unsigned)__shfl_xor((int)a, 2, 64));
        const int byte = mx::scale_byte(a);
        if (c < Kp) *reinterpret_cast<unsigned*>(static_cast<unsigned char*>(p.y) + row * (Kp / 2) + c / 2) = mx::pack8(y, byte);
        if (c % 32 == 0 && c < (long)(Kp + 255) / 256 * 256) static_cast<unsigned char*>(p.scale)[mx::scale_at(row, p.rows, (int)(c / 32))] = (unsigned char)(c < Kp ? byte : 0);
    }
}

// LPR lanes own a row and hold IT groups of eight elements each
template <typename T, bool AL, int LPR, int IT, int FMT>
__global__ __launch_bounds__(NT) void rms_fwd_kernel(const dist_rms_args p) {
    __shared__ float red[4];
    const int lr = threadIdx.x % LPR;
    const long row = (long)blockIdx.x * (NT / LPR) + threadIdx.x / LPR;
    if (row >= p.rows) return;
    const int C = p.C, Kp = (C + 31) / 32 * 32;
    const T* X = static_cast<const T*>(p.x) + row * p.ldx;
    const T* R = p.res ? static_cast<const T*>(p.res) + row * p.ldres : nullptr;
    float x[IT][8];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const int c = (lr + it * LPR) * 8;
        mx::load8<AL>(X + c, C - c, x[it]);
    }
    if (R) {
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const int c = (lr + it * LPR) * 8;
            float r[8];
            mx::load8<AL>(R + c, C - c, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[it][e] += r[e];
        }
    }
    float s = 0.f;
#pragma unroll
    for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += x[it][e] * x[it][e];
    const float rstd = 1.f / sqrtf(row_sum<LPR>(s, red) / (float)C + p.eps);
    if (p.rstd && lr == 0) p.rstd[row] = rstd;
    if (p.h) {
        T* H = static_cast<T*>(p.h) + row * p.ldh;
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const int c = (lr + it * LPR) * 8;
            mx::store8<AL>(H + c, C - c, x[it]);
        }
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const int c = (lr + it * LPR) * 8;
        float w[8];
        mx::load8<AL>(p.w + c, C - c, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[it][e] = AL || c + e < C ? x[it][e] * rstd * w[e] : 0.f;
    }
    float inv = 1.f;
    if constexpr (FMT == DIST_RMS_E4M3) {
        float a = 0.f, scale;
#pragma unroll
        for (int it = 0; it < IT; ++it)
#pragma unroll
            for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(x[it][e]));
        inv = e4m3_factor(row_max<LPR>(a, red), scale);
        if (lr == 0) static_cast<float*>(p.scale)[row] = scale;
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) put<T, AL, FMT>(p, x[it], inv, row, (long)(lr + it * LPR) * 8, Kp);
}

// rows too long for the registers: the block walks its row again for every step (the second and third walk find it in the L2).  h is stored last, so it may be x or res.
template <typename T, int FMT>
__global__ __launch_bounds__(NT) void rms_fwd_long_kernel(const dist_rms_args p) {
    __shared__ float red[4];
    const long row = blockIdx.x;
    const int C = p.C, Kp = (C + 31) / 32 * 32;
    const T* X = static_cast<const T*>(p.x) + row * p.ldx;
    const T* R = p.res ? static_cast<const T*>(p.res) + row * p.ldres : nullptr;
    T* H = p.h ? static_cast<T*>(p.h) + row * p.ldh : nullptr;
    auto group = [&](long c, float h[8]) __attribute__((always_inline)) {
        float r[8];
        mx::load8<false>(X + c, C - c, h);
        if (!R) return;
        mx::load8<false>(R + c, C - c, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] += r[e];
    };
    auto norm = [&](long c, float h[8], float rstd) __attribute__((always_inline)) {
        float w[8];
        mx::load8<false>(p.w + c, C - c, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = c + e < C ? h[e] * rstd * w[e] : 0.f;
    };
    float s = 0.f, h[8];
    for (long c = threadIdx.x * 8; c < C; c += NT * 8) {
        group(c, h);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += h[e] * h[e];
    }
    const float rstd = 1.f / sqrtf(row_sum<NT>(s, red) / (float)C + p.eps);
    if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
    float inv = 1.f;
    if constexpr (FMT == DIST_RMS_E4M3) {
        float a = 0.f, scale;
        for (long c = threadIdx.x * 8; c < C; c += NT * 8) {
            group(c, h);
            norm(c, h, rstd);
#pragma unroll
            for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(h[e]));
        }
        inv = e4m3_factor(row_max<NT>(a, red), scale);
        if (threadIdx.x == 0) static_cast<float*>(p.scale)[row] = scale;
    }
    for (long c = threadIdx.x * 8; c < ((long)C + NT * 8 - 1) / (NT * 8) * (NT * 8); c += NT * 8) {          // (every lane of a block of 32 takes part)
        group(c, h);
        if (H) mx::store8<false>(H + c, C - c, h);
        norm(c, h, rstd);
        put<T, false, FMT>(p, h, inv, row, c, Kp);
    }
}

// Backward.  A block keeps the sums of dw over its rows in registers and leaves one partial row; rms_dw_kernel adds the partial rows in a fixed order (no atomics:
// the same bits every time).
template <typename T, typename TD, bool AL, int LPR, int IT>
__global__ __launch_bounds__(LPR > NT ? LPR : NT, 2) void rms_bwd_kernel(const dist_rms_bwd_args p) {
    __shared__ float red[8];
    __shared__ float cols[LPR < NT ? LPR * IT * 8 : 1];
    const int lr = threadIdx.x % LPR, slot = threadIdx.x / LPR, C = p.C;
    constexpr int RPB = LPR < NT ? NT / LPR : 1;
    float w[IT][8], aw[IT][8];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const int c = (lr + it * LPR) * 8;
        mx::load8<AL>(p.w + c, C - c, w[it]);
#pragma unroll
        for (int e = 0; e < 8; ++e) aw[it][e] = 0.f;
    }
    // the next row is read while this one is worked on (50432 x 768 bf16 with dres: 77 us without, 62 with)
    const T* const A = static_cast<const T*>(p.dres);
    mx::Raw8<AL, T> hn[IT], rn[IT];
    mx::Raw8<AL, TD> dn[IT];
    float sn = 0.f;
    auto fetch = [&](long row) __attribute__((always_inline)) {
        row = min(row, p.rows - 1);
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const int c = (lr + it * LPR) * 8;
            hn[it].load(static_cast<const T*>(p.h) + row * p.ldh + c, C - c);
            dn[it].load(static_cast<const TD*>(p.dy) + row * p.lddy + c, C - c);
            if (A) rn[it].load(A + row * p.lddres + c, C - c);
        }
        sn = p.rstd[row];
    };
    const long stride = (long)gridDim.x * RPB;
    long row = (long)blockIdx.x * RPB + slot;
    if (row < p.rows) fetch(row);
    for (; row < p.rows; row += stride) {
        const float rstd = sn;
        float n[IT][8], g[IT][8], o[IT][8];
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const int c = (lr + it * LPR) * 8;
            hn[it].settle(C - c);
            dn[it].settle(C - c);
            if (A) rn[it].settle(C - c);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                n[it][e] = hn[it].get(e) * rstd;
                g[it][e] = dn[it].get(e);
                o[it][e] = A ? rn[it].get(e) : 0.f;
            }
        }
        if (row + stride < p.rows) fetch(row + stride);
        float s = 0.f;
#pragma unroll
        for (int it = 0; it < IT; ++it)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                aw[it][e] += g[it][e] * n[it][e];
                g[it][e] *= w[it][e];
                s += g[it][e] * n[it][e];
            }
        const float m = row_sum<LPR>(s, red) / (float)C;
        if (p.dh) {
            T* O = static_cast<T*>(p.dh) + row * p.lddh;
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                const int c = (lr + it * LPR) * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[it][e] = rstd * (g[it][e] - n[it][e] * m) + o[it][e];
                mx::store8<AL>(O + c, C - c, o[it]);
            }
        }
    }
    // the only workgroup (few rows) writes dw itself
    const bool only = gridDim.x == 1, add = only && p.accumulate;
    float* part = only ? p.dw : p.scratch + (long)blockIdx.x * C;
    if constexpr (LPR >= NT) {
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const int c = (lr + it * LPR) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < C) part[c + e] = add ? part[c + e] + aw[it][e] : aw[it][e];
        }
    } else {
        for (int k = 0; k < RPB; ++k) {                                       // the block's row slots, one after the other
            if (slot == k) {
#pragma unroll
                for (int it = 0; it < IT; ++it)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float& q = cols[(lr + it * LPR) * 8 + e];
                        q = k == 0 ? aw[it][e] : q + aw[it][e];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < C; c += NT) part[c] = add ? part[c] + cols[c] : cols[c];
    }
}

// long rows, and rows of less than a group: dh by a block per row (of many rows: the workgroups stride over them); dw by columns, one partial row per slice of rows
constexpr int64_t LONG_BLOCKS = 1 << 20;
template <typename T, typename TD>
__global__ __launch_bounds__(NT) void rms_bwd_long_kernel(const dist_rms_bwd_args p) {
    __shared__ float red[4];
    const int C = p.C;
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* H = static_cast<const T*>(p.h) + row * p.ldh;
        const TD* D = static_cast<const TD*>(p.dy) + row * p.lddy;
        const T* A = p.dres ? static_cast<const T*>(p.dres) + row * p.lddres : nullptr;
        T* O = static_cast<T*>(p.dh) + row * p.lddh;
        const float rstd = p.rstd[row];
        float s = 0.f;
        for (long c = threadIdx.x; c < C; c += NT) s += to_f(D[c]) * p.w[c] * (to_f(H[c]) * rstd);
        const float m = row_sum<NT>(s, red) / (float)C;
        for (long c = threadIdx.x; c < C; c += NT) O[c] = from_f<T>(rstd * (to_f(D[c]) * p.w[c] - to_f(H[c]) * rstd * m) + (A ? to_f(A[c]) : 0.f));
    }
}
template <typename T, typename TD>
__global__ __launch_bounds__(NT) void rms_dw_cols_kernel(const dist_rms_bwd_args p, const int slices, const int ctiles) {
    const int slice = blockIdx.x / ctiles;
    const long c = (long)(blockIdx.x % ctiles) * NT + threadIdx.x;
    if (c >= p.C) return;
    float s = 0.f;
    for (long row = slice; row < p.rows; row += slices)
        s += to_f(static_cast<const TD*>(p.dy)[row * p.lddy + c]) * (to_f(static_cast<const T*>(p.h)[row * p.ldh + c]) * p.rstd[row]);
    p.scratch[(long)slice * p.C + c] = s;
}

// dw[c] (+)= sum of the partial rows: 64 groups of 16 threads take every 64th row each, then the groups in order
__global__ __launch_bounds__(1024) void rms_dw_kernel(const float* __restrict__ part, const int G, const int C, float* __restrict__ dw, const int accumulate) {
    __shared__ float red[64][16];
    const int l = threadIdx.x & 15, c = blockIdx.x * 16 + l, g = threadIdx.x >> 4;
    float s = 0.f;
    if (c < C) {
#pragma unroll 8
        for (int k = g; k < G; k += 64) s += part[(long)k * C + c];
    }
    red[g][l] = s;
    __syncthreads();
    if (g == 0 && c < C) {
#pragma unroll 8
        for (int k = 1; k < 64; ++k) s += red[k][l];
        dw[c] = accumulate ? dw[c] + s : s;
    }
}

constexpr int FWD_MAX = 16384, BWD_MAX = 8192;                // widths whose rows stay in registers
// Workgroups of the backward kernel: two a CU of 256 threads each (50432 x 768: 384 67 us, 512 62, 640 77, 1024 66).  Of the 512 threads that rows over 4096 take a CU holds one
// (150 registers and more a lane), so that these run in two rounds of it (1831 x 8192 bf16 38.5 us for 92 MB; not tried with 256).
constexpr int PARTIALS = 512;

// lanes per row of the backward kernel (0: a long row, or one of less than a group).  At most three groups of eight a lane, else a CU holds one workgroup only (15 M elements in bf16: 2048 columns by 64 lanes
// of four groups 29.6 us, by 256 of one 27.6; 8192 by 256 of four 40.3, by 512 of two 38.6)
inline int bwd_lanes(int C) { return C < 8 ? 0 : C <= 384 ? 16 : C <= 768 ? 32 : C <= 1024 ? 64 : C <= 4096 ? 256 : C <= BWD_MAX ? 512 : 0; }
inline int64_t bwd_partials(int64_t rows, int C) {
    const int lanes = bwd_lanes(C);
    const int64_t per = lanes && lanes < NT ? NT / lanes : 1, need = (rows + per - 1) / per, most = lanes ? PARTIALS : 64;
    if (lanes && need <= 4) return 1;                         // (few rows: a second launch costs more than a workgroup's four steps)
    return need < 1 ? 1 : need > most ? most : need;
}
inline bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

template <typename T, bool AL, int FMT> int fwd(const dist_rms_args& p, hipStream_t s) {
    const int64_t Cr = FMT == DIST_RMS_MXFP4 ? ((int64_t)p.C + 255) / 256 * 256 : p.C;       // (the scale bytes of a whole chunk are written)
    const int64_t rows = p.rows;
#define DIST_RMS(LPR, IT) do { const int64_t b = (rows + NT / LPR - 1) / (NT / LPR); if (mx::too_many(b, NT)) return DIST_ERR_ARG; \
        hipLaunchKernelGGL((rms_fwd_kernel<T, AL, LPR, IT, FMT>), dim3((unsigned)b), dim3(NT), 0, s, p); } while (0)
    if (Cr <= 384) DIST_RMS(16, 3);
    else if (Cr <= 768) DIST_RMS(32, 3);
    else if (Cr <= 1024) DIST_RMS(64, 2);
    else if (Cr <= 2048) DIST_RMS(64, 4);
    else if (Cr <= 4096) DIST_RMS(256, 2);
    else if (Cr <= 8192) DIST_RMS(256, 4);
    else if (Cr <= FWD_MAX) DIST_RMS(256, 8);
    else {
        if (mx::too_many(rows, NT)) return DIST_ERR_ARG;
        hipLaunchKernelGGL((rms_fwd_long_kernel<T, FMT>), dim3((unsigned)rows), dim3(NT), 0, s, p);
    }
#undef DIST_RMS
    HIP_CHECK_RET(hipGetLastError());
    return DIST_OK;
}
template <typename T, int FMT> int fwd(const dist_rms_args& p, hipStream_t s) {
    const bool al = p.C % 8 == 0 && p.ldx % 8 == 0 && aligned16(p.x) && aligned16(p.w) && (!p.res || (p.ldres % 8 == 0 && aligned16(p.res))) &&
                    (!p.h || (p.ldh % 8 == 0 && aligned16(p.h))) && aligned16(p.y) && (FMT == DIST_RMS_MXFP4 || p.ldy % 8 == 0);
    return al ? fwd<T, true, FMT>(p, s) : fwd<T, false, FMT>(p, s);
}

template <typename T, typename TD, bool AL> int bwd(const dist_rms_bwd_args& p, hipStream_t s) {
    const int G = (int)bwd_partials(p.rows, p.C);
    const int lanes = bwd_lanes(p.C);
#define DIST_RMS(LPR, IT) hipLaunchKernelGGL((rms_bwd_kernel<T, TD, AL, LPR, IT>), dim3((unsigned)G), dim3(LPR > NT ? LPR : NT), 0, s, p)
    const int64_t sums = (p.C + 15) / 16;                     // workgroups of the last pass
    if (mx::too_many(sums, 1024)) return DIST_ERR_ARG;
    if (!lanes) {
        const int ctiles = (p.C + NT - 1) / NT;
        if (mx::too_many((int64_t)G * ctiles, NT)) return DIST_ERR_ARG;
        hipLaunchKernelGGL((rms_dw_cols_kernel<T, TD>), dim3((unsigned)(G * ctiles)), dim3(NT), 0, s, p, G, ctiles);       // (before dh, which may take h's or dy's place)
        if (p.dh && p.rows) hipLaunchKernelGGL((rms_bwd_long_kernel<T, TD>), dim3((unsigned)min(p.rows, LONG_BLOCKS)), dim3(NT), 0, s, p);
    } else if (lanes == 16) DIST_RMS(16, 3);
    else if (lanes == 32) DIST_RMS(32, 3);
    else if (lanes == 64) DIST_RMS(64, 2);
    else if (lanes == 256) { if (p.C <= 2048) DIST_RMS(256, 1); else DIST_RMS(256, 2); }
    else DIST_RMS(512, 2);
#undef DIST_RMS
    HIP_CHECK_RET(hipGetLastError());
    if (lanes && G == 1) return DIST_OK;
    hipLaunchKernelGGL(rms_dw_kernel, dim3((unsigned)sums), dim3(1024), 0, s, p.scratch, G, p.C, p.dw, p.accumulate);
    HIP_CHECK_RET(hipGetLastError());
    return DIST_OK;
}
template <typename T, typename TD> int bwd(const dist_rms_bwd_args& p, hipStream_t s) {
    const bool al = p.C % 8 == 0 && p.ldh % 8 == 0 && p.lddy % 8 == 0 && aligned16(p.h) && aligned16(p.dy) && aligned16(p.w) &&
                    (!p.dres || (p.lddres % 8 == 0 && aligned16(p.dres))) && (!p.dh || (p.lddh % 8 == 0 && aligned16(p.dh)));
    return al ? bwd<T, TD, true>(p, s) : bwd<T, TD, false>(p, s);
}

}  // namespace

extern "C" int dist_op_rmsnorm(const dist_rms_args* a, void* stream) {
    if (!a) return DIST_ERR_ARG;
    const dist_rms_args p = *a;
    if (p.dtype != DIST_BF16 && p.dtype != DIST_F32) return DIST_ERR_ARG;
    if (p.fmt != DIST_RMS_SAME && p.fmt != DIST_RMS_E4M3 && p.fmt != DIST_RMS_MXFP4) return DIST_ERR_ARG;
    if (p.rows < 0 || p.C <= 0 || p.C > (1 << 30) || !(p.eps >= 0.f)) return DIST_ERR_ARG;
    if (p.rows == 0) return DIST_OK;
    const uintptr_t es = p.dtype == DIST_BF16 ? 2 : 4;
    if (!p.x || !p.w || !p.y || (p.fmt != DIST_RMS_SAME && !p.scale) || p.ldx < p.C || (p.res && p.ldres < p.C) || (p.h && p.ldh < p.C)) return DIST_ERR_ARG;
    if (p.fmt != DIST_RMS_MXFP4 && p.ldy < p.C) return DIST_ERR_ARG;
    if ((uintptr_t)p.x % es || (uintptr_t)p.res % es || (uintptr_t)p.h % es || (p.fmt == DIST_RMS_SAME && (uintptr_t)p.y % es) || (p.fmt == DIST_RMS_MXFP4 && !aligned16(p.y))) return DIST_ERR_ARG;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.dtype == DIST_BF16)
        return p.fmt == DIST_RMS_SAME ? fwd<bf16_t, DIST_RMS_SAME>(p, s) : p.fmt == DIST_RMS_E4M3 ? fwd<bf16_t, DIST_RMS_E4M3>(p, s) : fwd<bf16_t, DIST_RMS_MXFP4>(p, s);
    return p.fmt == DIST_RMS_SAME ? fwd<float, DIST_RMS_SAME>(p, s) : p.fmt == DIST_RMS_E4M3 ? fwd<float, DIST_RMS_E4M3>(p, s) : fwd<float, DIST_RMS_MXFP4>(p, s);
}

extern "C" int64_t dist_op_rmsnorm_bwd_scratch(int64_t rows, int C) {
    if (rows < 0 || C <= 0) return -1;
    return bwd_partials(rows, C) * C;
}

extern "C" int dist_op_rmsnorm_bwd(const dist_rms_bwd_args* a, void* stream) {
    if (!a) return DIST_ERR_ARG;
    const dist_rms_bwd_args p = *a;
    if ((p.dtype != DIST_BF16 && p.dtype != DIST_F32) || (p.dy_dtype != DIST_BF16 && p.dy_dtype != DIST_F32)) return DIST_ERR_ARG;
    if (p.rows < 0 || p.C <= 0 || p.C > (1 << 30) || !p.w || !p.dw || !p.scratch) return DIST_ERR_ARG;
    if (p.scratch_elems < dist_op_rmsnorm_bwd_scratch(p.rows, p.C)) return DIST_ERR_WORKSPACE;
    if (p.rows > 0 && (!p.h || !p.rstd || !p.dy || p.ldh < p.C || p.lddy < p.C || (p.dres && p.lddres < p.C) || (p.dh && p.lddh < p.C))) return DIST_ERR_ARG;
    const uintptr_t es = p.dtype == DIST_BF16 ? 2 : 4, ed = p.dy_dtype == DIST_BF16 ? 2 : 4;
    if ((uintptr_t)p.h % es || (uintptr_t)p.dres % es || (uintptr_t)p.dh % es || (uintptr_t)p.dy % ed) return DIST_ERR_ARG;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.dtype == DIST_BF16) return p.dy_dtype == DIST_BF16 ? bwd<bf16_t, bf16_t>(p, s) : bwd<bf16_t, float>(p, s);
    return p.dy_dtype == DIST_BF16 ? bwd<float, bf16_t>(p, s) : bwd<float, float>(p, s);
}
