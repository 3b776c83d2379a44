// Products with an MXFP4 weight (dist_op_gemm_mxfp4): C[m][n] = a_scale[m] * sum_k A[m][k] B[n][k] + bias[n] + res[m][n], A in MXFP4 or in e4m3 with one scale per row.
//
// One v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 16 outputs over 128 elements, the block scales applied by the instruction.  A lane holds for its row (lane & 15)
// the 32 elements of block g = lane >> 4: 16 bytes of codes as they lie in memory.  An e4m3 operand has its 32 bytes in two runs of 16: elements 16 g .. and 64 + 16 g ..
// (measured with random operands; the scale of lane group g still belongs to block g, here 1 for all).
// The weight is the instruction's FIRST operand: the result has the outputs' n along the registers of a lane and m along the lanes, and with the weight's rows dealt to the
// NT fragments as n = (i >> 2) * 4 NT + 4 j + (i & 3) (fragment j, its row i) a lane owns 4 NT consecutive outputs of one row of C: 16-byte stores, whole 128-byte lines
// from four lanes at NT = 4, no exchange through LDS.
#include <type_traits>
#include "mx.h"

namespace {

typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef int v4i_t __attribute__((ext_vector_type(4)));
constexpr int NT_ = 256;

DEV v8i_t join(const v4i_t& lo, const v4i_t& hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
DEV v8i_t widen(const v4i_t& lo) { return join(lo, v4i_t{0, 0, 0, 0}); }

// acc (n x m) += B fragment x A fragment; S: which of the two scale bytes
template <bool A8, int S> DEV void mma(const v8i_t& b, const v8i_t& a, f32x4& acc, int bs, int as) {
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, acc, 4, A8 ? 0 : 4, S, bs, A8 ? 0 : S, as);
}

// 4 NT consecutive outputs of row m, from column n on
template <bool A8, typename TO, int NT>
DEV void store_row(const dist_gemm_mx_args& p, const f32x4 (&acc)[NT], long m, int n, bool vec) {
    if (m >= p.M || n >= p.N) return;
    float v[4 * NT];
    const float as = A8 ? static_cast<const float*>(p.a_scale)[m] : 1.f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[4 * j + r] = A8 ? acc[j][r] * as : acc[j][r];
    TO* C = static_cast<TO*>(p.C) + m * p.ldc + n;
    const TO* R = p.res ? static_cast<const TO*>(p.res) + m * p.ldres + n : nullptr;
    if (vec && n + 4 * NT <= p.N) {
        if constexpr (NT % 2 == 0) {
#pragma unroll
            for (int j = 0; j < NT / 2; ++j) {
                if (p.bias) { float b[8]; mx::load_v<8>(p.bias + n + 8 * j, b);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[8 * j + e] += b[e]; }
                if (R) { float b[8]; mx::load_v<8>(R + 8 * j, b);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[8 * j + e] += b[e]; }
                mx::store_v<8>(C + 8 * j, v + 8 * j);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (p.bias) { float b[4]; load4(p.bias + n + 4 * j, b);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * j + e] += b[e]; }
                if (R) { float b[4]; load4(R + 4 * j, b);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * j + e] += b[e]; }
                store4(C + 4 * j, v + 4 * j);
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4 * NT; ++e)
        if (n + e < p.N) C[e] = from_f<TO>(v[e] + (p.bias ? p.bias[n + e] : 0.f) + (R ? to_f(R[e]) : 0.f));
}

// Every wave a 16 MT x 16 NT tile of its own, fragments straight from global memory.
template <bool A8, typename TO, int MT, int NT>
__global__ __launch_bounds__(NT_) void gemm_mx_direct_kernel(const dist_gemm_mx_args p, const int vec, const int ntn) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const long m0 = ((long)(blockIdx.x / ntn) * 2 + (wave >> 1)) * (16 * MT);
    const int n0 = ((int)(blockIdx.x % ntn) * 2 + (wave & 1)) * (16 * NT);
    if (m0 >= p.M || n0 >= p.N) return;
    const unsigned char *A = static_cast<const unsigned char*>(p.A), *B = static_cast<const unsigned char*>(p.B);
    const unsigned char *SA = static_cast<const unsigned char*>(p.a_scale), *SB = static_cast<const unsigned char*>(p.b_scale);
    long am[MT], bn[NT];                                     // rows, clamped: what lies behind the last one is computed and not stored
#pragma unroll
    for (int t = 0; t < MT; ++t) am[t] = min(m0 + t * 16 + i, p.M - 1);
#pragma unroll
    for (int j = 0; j < NT; ++j) bn[j] = min((long)n0 + (i >> 2) * (4 * NT) + 4 * j + (i & 3), (long)p.N - 1);
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const v4i_t zero = {0, 0, 0, 0};
    for (int k0 = 0; k0 < p.K; k0 += mx::CHUNK) {
        int as[MT], bs[NT];
        const long chunk = k0 / mx::CHUNK;
#pragma unroll
        for (int t = 0; t < MT; ++t) as[t] = A8 ? 127 : *reinterpret_cast<const unsigned short*>(SA + (chunk * p.M + am[t]) * 8 + 2 * g);
#pragma unroll
        for (int j = 0; j < NT; ++j) bs[j] = *reinterpret_cast<const unsigned short*>(SB + (chunk * p.N + bn[j]) * 8 + 2 * g);
        auto step = [&](auto sc) {
            constexpr int S = decltype(sc)::value;
            const int k = k0 + S * 128;
            if (k >= p.K) return;
            v8i_t a[MT], b[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j] = widen(k + g * 32 < p.K ? *reinterpret_cast<const v4i_t*>(B + bn[j] * (p.K / 2) + k / 2 + g * 16) : zero);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if constexpr (A8) {
                    const unsigned char* q = A + am[t] * p.lda + k;
                    a[t] = join(k + g * 16 < p.K ? *reinterpret_cast<const v4i_t*>(q + g * 16) : zero, k + 64 + g * 16 < p.K ? *reinterpret_cast<const v4i_t*>(q + 64 + g * 16) : zero);
                } else a[t] = widen(k + g * 32 < p.K ? *reinterpret_cast<const v4i_t*>(A + am[t] * (p.K / 2) + k / 2 + g * 16) : zero);
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int j = 0; j < NT; ++j) mma<A8, S>(b[j], a[t], acc[t][j], bs[j], as[t]);
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) store_row<A8, TO, NT>(p, acc[t], m0 + t * 16 + i, n0 + g * (4 * NT), vec);
}

// ---- tiles through LDS ------------------------------------------------------------------------------------------------------------------------------------------
// WM x WN waves, each a 16 MT x 16 NT tile of outputs.  K advances by 128 elements a stage (one instruction deep): rows of 64 bytes of codes (e4m3: 128 bytes) go to LDS by
// LDS-DMA into a ring of S stages, S - 1 of them in flight; one barrier per stage, behind a counted wait: when it opens, stage t has landed for every wave and stage
// t - 1 is read by nobody, so its place receives stage t + S - 1.  Scale bytes follow per 256 elements into a ring of their own, with the stage that needs them first.
// A 16-byte chunk c of row r lies at chunk c ^ f(r), applied where the DMA reads (its LDS side is lane-linear): the 16 rows a fragment read touches fall on
// different banks.  Descriptors end behind the last row, and chunks behind K are sent past the end: all of these read as zeros.
typedef __attribute__((address_space(3))) void* lds_ptr;
DEV void regs_pin(unsigned& v) { asm volatile("" : "+v"(v)); }
template <int N> DEV void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
constexpr unsigned FAR_AWAY = 0x7ffffff0u;

// n of row i of fragment j inside a wave's columns.  16-bit outputs: two fragments share 32 columns, so that a lane's 8 outputs of the pair are 16 bytes and four lanes 64;
// 32-bit outputs: a lane's 4 outputs of one fragment are 16 bytes.
template <typename TO> DEV constexpr int frag_col(int j) { return sizeof(TO) == 2 ? (j >> 1) * 32 + (j & 1) * 4 : j * 16; }
template <typename TO> DEV int lane_col(int i) { return sizeof(TO) == 2 ? (i >> 2) * 8 + (i & 3) : i; }

template <bool A8> DEV int a_swz(int r) { return A8 ? (r >> 1) & 7 : ((r >> 2) & 1) | ((((r >> 1) ^ (r >> 3)) & 1) << 1); }
template <typename TO> DEV int b_swz(int r) {
    return sizeof(TO) == 2 ? ((r >> 3) & 1) | ((((r >> 1) ^ (r >> 4)) & 1) << 1) : a_swz<false>(r);
}

template <bool A8, typename TO, int WM, int WN, int MT, int NT, int S>
struct Tile {
    static constexpr int W = WM * WN, BM = WM * MT * 16, BN = WN * NT * 16;
    static constexpr int PA = A8 ? 128 : 64;                                       // bytes of a row of A in a stage
    static constexpr int A_BYTES = BM * PA, B_BYTES = BN * 64, STAGE = A_BYTES + B_BYTES;
    static constexpr int NA = A_BYTES / 1024, NB = B_BYTES / 1024, PER = (NA + NB) / W;     // DMA instructions of a stage, per wave
    static constexpr int SA_BYTES = A8 ? 0 : (BM * 8 + 1023) / 1024 * 1024, SB_BYTES = (BN * 8 + 1023) / 1024 * 1024, SC = SA_BYTES + SB_BYTES;
    static constexpr int NS = SC / 1024, PERS = (NS + W - 1) / W;                  // of the scales of 256 elements
    static constexpr int LDS = S * STAGE + 2 * SC;
    static_assert((NA + NB) % W == 0 && A_BYTES % 1024 == 0 && B_BYTES % 1024 == 0, "a stage is whole instructions for every wave");
};

template <bool A8, typename TO, int WM, int WN, int MT, int NT, int S, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void gemm_mx_tile_kernel(const dist_gemm_mx_args p, const int vec, const int ntm, const int ntn) {
    using T = Tile<A8, TO, WM, WN, MT, NT, S>;
    extern __shared__ char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    // block -> tile: block b runs on XCD b % 8; every XCD takes a contiguous run of tiles, ordered in groups of 8 row tiles, so that the tiles an XCD works on at a time
    // share row and column panels in its L2
    const int total = ntm * ntn, xcd = blockIdx.x & 7, each = total >> 3, more = total & 7;
    const int t0 = xcd * each + min(xcd, more) + (int)(blockIdx.x >> 3);
    const int grp = t0 / (8 * ntn), in = t0 - grp * 8 * ntn, gm = min(8, ntm - grp * 8);
    const long m0 = (long)(grp * 8 + in % gm) * T::BM;
    const int n0 = (in / gm) * T::BN;

    const long pitch_a = A8 ? p.lda : p.K / 2, pitch_b = p.K / 2;
    const int mrows = (int)min((long)T::BM, p.M - m0), nrows = min(T::BN, p.N - n0);
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(p.A) + m0 * pitch_a), 0, (int)(mrows * pitch_a), 0x00020000);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(p.B) + n0 * pitch_b), 0, (int)(nrows * pitch_b), 0x00020000);
    const int nk = (p.K + 127) / 128, tail = p.K - (nk - 1) * 128;                 // elements of the last stage

    // this wave's kilobytes of a stage: which operand, and the lane's offset in it
    unsigned voff[T::PER];
    int vchunk[T::PER];                                                            // first element of the lane's 16 bytes inside the stage
#pragma unroll
    for (int q = 0; q < T::PER; ++q) {
        const int k = wave * T::PER + q;
        constexpr int LPR = T::PA / 16;                                            // lanes per row of A
        const bool isa = k < T::NA;
        const int r = isa ? k * (64 / LPR) + lane / LPR : (k - T::NA) * 16 + (lane >> 2);
        const int c = isa ? (lane % LPR) ^ a_swz<A8>(r) : (lane & 3) ^ b_swz<TO>(r);
        voff[q] = (unsigned)(r * (isa ? pitch_a : pitch_b)) + c * 16;
        vchunk[q] = c * (isa && A8 ? 16 : 32);
    }
    auto issue = [&](const int kt) __attribute__((always_inline)) {
        char* base = smem + (kt % S) * T::STAGE;
        // (the offsets live in the same registers for the whole loop and change once, under a branch: hipcc waits for every load in flight before it reuses a register that
        // one of them takes its address from)
        if (kt == nk - 1 && tail < 128) {
#pragma unroll
            for (int q = 0; q < T::PER; ++q) {
                if (vchunk[q] >= tail) voff[q] = FAR_AWAY;
                regs_pin(voff[q]);
            }
        }
#pragma unroll
        for (int q = 0; q < T::PER; ++q) {
            const int k = wave * T::PER + q;                                       // wave-uniform
            const bool isa = k < T::NA;
            const unsigned v = voff[q];
            const int step = kt * (isa ? T::PA : 64);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(isa ? ra : rb, (lds_ptr)(base + k * 1024), 16, v, step, 0, 0);
        }
    };
    // the scales' kilobytes of this wave: source, what is there to read and the step to the next 256 elements (a wave without one of its own repeats the last: the
    // same bytes to the same place)
    const char* ssrc[T::PERS];
    long sstep[T::PERS];
    int sleft[T::PERS], sdst[T::PERS];
#pragma unroll
    for (int q = 0; q < T::PERS; ++q) {
        const int k = min(wave * T::PERS + q, T::NS - 1);
        sdst[q] = S * T::STAGE + k * 1024;
        if (k < T::SA_BYTES / 1024) {
            ssrc[q] = static_cast<const char*>(p.a_scale) + m0 * 8 + k * 1024;
            sstep[q] = p.M * 8;
            sleft[q] = max(mrows * 8 - k * 1024, 0);
        } else {
            ssrc[q] = static_cast<const char*>(p.b_scale) + (long)n0 * 8 + (k * 1024 - T::SA_BYTES);
            sstep[q] = (long)p.N * 8;
            sleft[q] = max(nrows * 8 - (k * 1024 - T::SA_BYTES), 0);
        }
    }
    auto issue_scales = [&](const int chunk) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < T::PERS; ++q) {
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(ssrc[q] + chunk * sstep[q]), 0, sleft[q], 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(smem + sdst[q] + (chunk & 1) * T::SC), 16, lane * 16, 0, 0, 0);
        }
    };

    // LDS addresses of this lane's fragments inside a stage
    const int arow = wm * MT * 16 + i, brow = wn * NT * 16 + lane_col<TO>(i);
    const int a_lo = arow * T::PA + ((g ^ a_swz<A8>(arow)) << 4), a_hi = arow * T::PA + (((4 + g) ^ a_swz<A8>(arow)) << 4);
    const int b_at = T::A_BYTES + brow * 64 + ((g ^ b_swz<TO>(brow)) << 4);

    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    int as[MT], bs[NT];
#pragma unroll
    for (int t = 0; t < MT; ++t) as[t] = 127;

    auto stage = [&](auto par, const int kt) __attribute__((always_inline)) {
        constexpr int P = decltype(par)::value;                                    // kt & 1: which byte of the scales
        // stages kt + 1 ... kt + S - 2 may stay in flight; of two neighbours one carries scales
        if (kt + S - 2 < nk) wait_vm<(S - 2) * T::PER + ((S - 2 + (P ? 1 : 0)) / 2) * T::PERS>();
        else wait_vm<0>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (kt + S - 1 < nk) {
            if (((kt + S - 1) & 1) == 0) issue_scales((kt + S - 1) >> 1);
            issue(kt + S - 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        const char* base = smem + (kt % S) * T::STAGE;
        if constexpr (P == 0) {
            const char* sc = smem + S * T::STAGE + ((kt >> 1) & 1) * T::SC;
            if constexpr (!A8)
#pragma unroll
                for (int t = 0; t < MT; ++t) as[t] = *reinterpret_cast<const unsigned short*>(sc + (arow + t * 16) * 8 + 2 * g);
#pragma unroll
            for (int j = 0; j < NT; ++j) bs[j] = *reinterpret_cast<const unsigned short*>(sc + T::SA_BYTES + (brow + frag_col<TO>(j)) * 8 + 2 * g);
        }
        v8i_t a[MT], b[NT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if constexpr (A8) a[t] = join(*reinterpret_cast<const v4i_t*>(base + a_lo + t * 16 * T::PA), *reinterpret_cast<const v4i_t*>(base + a_hi + t * 16 * T::PA));
            else a[t] = widen(*reinterpret_cast<const v4i_t*>(base + a_lo + t * 16 * T::PA));
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) b[j] = widen(*reinterpret_cast<const v4i_t*>(base + b_at + frag_col<TO>(j) * 64));
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) mma<A8, P>(b[j], a[t], acc[t][j], bs[j], as[t]);
    };

#pragma unroll
    for (int k = 0; k < S - 1; ++k)
        if (k < nk) {
            if ((k & 1) == 0) issue_scales(k >> 1);
            issue(k);
        }
    for (int kt = 0; kt < nk; kt += 2) {
        stage(std::integral_constant<int, 0>{}, kt);
        if (kt + 1 < nk) stage(std::integral_constant<int, 1>{}, kt + 1);
    }

    // ---- outputs
    const long mw = m0 + wm * MT * 16 + i;
    float rs[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) rs[t] = A8 && mw + t * 16 < p.M ? static_cast<const float*>(p.a_scale)[mw + t * 16] : 1.f;
    constexpr int G = sizeof(TO) == 2 ? 2 : 1, V = 4 * G;                          // fragments and outputs of one 16-byte store
#pragma unroll
    for (int j = 0; j < NT; j += G) {
        const int n = n0 + wn * NT * 16 + frag_col<TO>(j) + g * V;
        if (n >= p.N) continue;
        const bool whole = vec && n + V <= p.N;
        float bias[V];
#pragma unroll
        for (int e = 0; e < V; ++e) bias[e] = 0.f;
        if (p.bias) {
            if (whole) {
                if constexpr (V == 8) mx::load_v<8>(p.bias + n, bias);
                else load4(p.bias + n, bias);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) bias[e] = n + e < p.N ? p.bias[n + e] : 0.f;
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const long m = mw + t * 16;
            if (m >= p.M) continue;
            TO* C = static_cast<TO*>(p.C) + m * p.ldc + n;
            const TO* R = p.res ? static_cast<const TO*>(p.res) + m * p.ldres + n : nullptr;
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = (A8 ? acc[t][j + e / 4][e % 4] * rs[t] : acc[t][j + e / 4][e % 4]) + bias[e];
            if (whole) {
                float r[V];
                if constexpr (V == 8) {
                    if (R) { mx::load_v<8>(R, r);
#pragma unroll
                        for (int e = 0; e < V; ++e) v[e] += r[e]; }
                    mx::store_v<8>(C, v);
                } else {
                    if (R) { load4(R, r);
#pragma unroll
                        for (int e = 0; e < V; ++e) v[e] += r[e]; }
                    store4(C, v);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (n + e < p.N) C[e] = from_f<TO>(v[e] + (R ? to_f(R[e]) : 0.f));
            }
        }
    }
}

template <bool A8, typename TO, int WM, int WN, int MT, int NT, int S, int OCC> int launch_tile(const dist_gemm_mx_args& p, int vec, hipStream_t s) {
    using T = Tile<A8, TO, WM, WN, MT, NT, S>;
    const long ntm = (p.M + T::BM - 1) / T::BM, ntn = (p.N + T::BN - 1) / T::BN;
    if (ntm * ntn > 0x3fffffff) return DIST_ERR_ARG;
    const auto k = gemm_mx_tile_kernel<A8, TO, WM, WN, MT, NT, S, OCC>;
    static DistSmemOnce st;
    RUN_(dist_max_smem(st, reinterpret_cast<const void*>(k), T::LDS));
    hipLaunchKernelGGL(k, dim3((unsigned)(ntm * ntn)), dim3(64 * T::W), T::LDS, s, p, vec, (int)ntm, (int)ntn);
    HIP_CHECK_RET(hipGetLastError());
    return DIST_OK;
}

template <bool A8, typename TO> int launch(const dist_gemm_mx_args& p, hipStream_t s) {
    const size_t es = sizeof(TO);
    const int vec = (uintptr_t)p.C % 16 == 0 && p.ldc * es % 16 == 0 && (!p.res || ((uintptr_t)p.res % 16 == 0 && p.ldres * es % 16 == 0)) && (!p.bias || (uintptr_t)p.bias % 16 == 0);
    if (p.M > 64 && p.K <= 1 << 22 && p.lda <= 1 << 22) {
        return launch_tile<A8, TO, 2, 2, 4, 4, 3, 2>(p, vec, s);
    }
    const long ntm = (p.M + 127) / 128, ntn = (p.N + 127) / 128;
    if (ntm * ntn > 0x7fffffff) return DIST_ERR_ARG;
    hipLaunchKernelGGL((gemm_mx_direct_kernel<A8, TO, 4, 4>), dim3((unsigned)(ntm * ntn)), dim3(NT_), 0, s, p, vec, (int)ntn);
    HIP_CHECK_RET(hipGetLastError());
    return DIST_OK;
}

}  // namespace

extern "C" int64_t dist_op_gemm_mxfp4_scratch(int64_t M, int N, int K, int a_fmt) {
    if (M < 0 || N <= 0 || K <= 0 || K % 32 || (a_fmt != DIST_MX_A_MXFP4 && a_fmt != DIST_MX_A_E4M3)) return -1;
    return 0;
}

extern "C" int dist_op_gemm_mxfp4(const dist_gemm_mx_args* a, void* stream) {
    if (!a) return DIST_ERR_ARG;
    const dist_gemm_mx_args p = *a;
    if (p.a_fmt != DIST_MX_A_MXFP4 && p.a_fmt != DIST_MX_A_E4M3) return DIST_ERR_ARG;
    if ((p.dtype != DIST_BF16 && p.dtype != DIST_F32) || (p.a_fmt == DIST_MX_A_E4M3 && p.dtype != DIST_BF16)) return DIST_ERR_ARG;
    if (p.M < 0 || p.N <= 0 || p.K <= 0 || p.K % 32 || p.K > (1 << 30)) return DIST_ERR_ARG;
    if (p.M == 0) return DIST_OK;
    const uintptr_t es = p.dtype == DIST_BF16 ? 2 : 4;
    if (!p.A || !p.a_scale || !p.B || !p.b_scale || !p.C || p.ldc < p.N || (p.res && p.ldres < p.N)) return DIST_ERR_ARG;
    if ((uintptr_t)p.A % 16 || (uintptr_t)p.B % 16 || (uintptr_t)p.b_scale % 8 || (uintptr_t)p.a_scale % (p.a_fmt == DIST_MX_A_E4M3 ? 4 : 8)) return DIST_ERR_ARG;
    if (p.a_fmt == DIST_MX_A_E4M3 && (p.lda < p.K || p.lda % 16)) return DIST_ERR_ARG;
    if ((uintptr_t)p.C % es || (uintptr_t)p.res % es || (uintptr_t)p.bias % 4) return DIST_ERR_ARG;
    if (p.scratch_elems < dist_op_gemm_mxfp4_scratch(p.M, p.N, p.K, p.a_fmt)) return DIST_ERR_WORKSPACE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.a_fmt == DIST_MX_A_E4M3) return launch<true, bf16_t>(p, s);
    return p.dtype == DIST_BF16 ? launch<false, bf16_t>(p, s) : launch<false, float>(p, s);
}
