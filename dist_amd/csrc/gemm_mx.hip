// Products with an MXFP4 weight (dist_op_gemm_mxfp4): C[m][n] = a_scale[m] * sum_k A[m][k] B[n][k] + bias[n] + res[m][n], A in MXFP4 or in e4m3 with one scale per row.
//
// One v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 16 outputs over 128 elements, the block scales applied by the instruction.  A lane holds for its row (lane & 15)
// the 32 elements of block g = lane >> 4: 16 bytes of codes as they lie in memory.  An e4m3 operand has its 32 bytes in two runs of 16: elements 16 g .. and 64 + 16 g ..
// (measured with random operands; the scale of lane group g still belongs to block g, here 1 for all).
// The weight is the instruction's FIRST operand: the result has the outputs' n along the registers of a lane and m along the lanes, so a lane owns consecutive outputs of
// one row of C.
#include <type_traits>
#include "mx.h"

namespace {

typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef unsigned v4u_t __attribute__((ext_vector_type(4)));
typedef int v4i_t __attribute__((ext_vector_type(4)));
constexpr int NT_ = 256;

DEV v8i_t join(const v4i_t& lo, const v4i_t& hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
DEV v8i_t widen(const v4i_t& lo) { return join(lo, v4i_t{0, 0, 0, 0}); }

// acc (n x m) += B fragment x A fragment; S: which of the two scale bytes
template <bool A8, int S> DEV void mma(const v8i_t& b, const v8i_t& a, f32x4& acc, int bs, int as) {
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, acc, 4, A8 ? 0 : 4, S, bs, A8 ? 0 : S, as);
}

// ---- few rows (one token, a handful of sequences): bound by the weight's bytes and by latency --------------------------------------------------------------------------
// A workgroup owns 16 NT columns and all rows; its W waves share K, every wave's fragments come straight from global memory (a row's 128 elements are 64 bytes from four
// lanes), and the partial sums meet in LDS, added in the waves' order.
template <bool A8, typename TO, int MT, int NT, int W>
__global__ __launch_bounds__(64 * W) void gemm_mx_few_kernel(const dist_gemm_mx_args p) {
    constexpr int TILES = MT * NT;
    __shared__ f32x4 part[W][TILES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * (16 * NT);
    const unsigned char *A = static_cast<const unsigned char*>(p.A), *B = static_cast<const unsigned char*>(p.B);
    const unsigned char *SA = static_cast<const unsigned char*>(p.a_scale), *SB = static_cast<const unsigned char*>(p.b_scale);
    long am[MT], bn[NT];                                     // rows, clamped: what lies behind the last one is computed and not stored
#pragma unroll
    for (int t = 0; t < MT; ++t) am[t] = min((long)t * 16 + i, p.M - 1);
#pragma unroll
    for (int j = 0; j < NT; ++j) bn[j] = min((long)n0 + j * 16 + i, (long)p.N - 1);
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const v4i_t zero = {0, 0, 0, 0};
    for (int k = wave * 128; k < p.K; k += W * 128) {
        const long chunk = k >> 8;
        const int at = 2 * g + ((k >> 7) & 1);
        const bool in = k + g * 32 < p.K;
        v8i_t a[MT], b[NT];
        int as[MT], bs[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            b[j] = widen(in ? *reinterpret_cast<const v4i_t*>(B + bn[j] * (p.K / 2) + k / 2 + g * 16) : zero);
            bs[j] = SB[(chunk * p.N + bn[j]) * 8 + at];
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if constexpr (A8) {
                const unsigned char* q = A + am[t] * p.lda + k;
                a[t] = join(k + g * 16 < p.K ? *reinterpret_cast<const v4i_t*>(q + g * 16) : zero, k + 64 + g * 16 < p.K ? *reinterpret_cast<const v4i_t*>(q + 64 + g * 16) : zero);
                as[t] = 127;
            } else {
                a[t] = widen(in ? *reinterpret_cast<const v4i_t*>(A + am[t] * (p.K / 2) + k / 2 + g * 16) : zero);
                as[t] = SA[(chunk * p.M + am[t]) * 8 + at];
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int j = 0; j < NT; ++j) mma<A8, 0>(b[j], a[t], acc[t][j], bs[j], as[t]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][t * NT + j][lane] = acc[t][j];
    __syncthreads();
    for (int e = threadIdx.x; e < TILES * 64; e += 64 * W) {                       // four neighbouring columns of a row
        const int tile = e >> 6, l = e & 63;
        const long m = (tile / NT) * 16 + (l & 15);
        const int n = n0 + (tile % NT) * 16 + (l >> 4) * 4;
        if (m >= p.M || n >= p.N) continue;
        f32x4 s = part[0][tile][l];
#pragma unroll
        for (int w = 1; w < W; ++w) s += part[w][tile][l];
        const float rs = A8 ? static_cast<const float*>(p.a_scale)[m] : 1.f;
        TO* C = static_cast<TO*>(p.C) + m * p.ldc + n;
        const TO* R = p.res ? static_cast<const TO*>(p.res) + m * p.ldres + n : nullptr;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < p.N) C[r] = from_f<TO>((A8 ? s[r] * rs : s[r]) + (p.bias ? p.bias[n + r] : 0.f) + (R ? to_f(R[r]) : 0.f));
    }
}

// ---- tiles through LDS ------------------------------------------------------------------------------------------------------------------------------------------
// WM x WN waves, each a 16 MT x 16 NT tile of outputs.  K advances by 256 elements a stage (4-bit operands: two instructions deep) or 128 (e4m3): rows of 128 bytes of A and
// of 64 D bytes of B go to LDS by LDS-DMA into a ring of S stages, S - 1 of them in flight; one barrier per stage, behind a counted wait: when it opens, stage t has landed for
// every wave and stage t - 1 is read by nobody, so its place receives stage t + S - 1.  Scale bytes follow per 256 elements into a ring of their own, with the stage that needs
// them first.  A 16-byte chunk c of row r lies at chunk c ^ f(r), applied where the DMA reads (its LDS side is lane-linear).  Descriptors end behind the last row, and chunks
// behind K are sent past the end: all of these read as zeros.
// Measured, in graphs: 50432 x 2304 x 768, 4-bit operands, bf16 out, 79 us = 2.25 PF in 256 x 256 tiles and 82 in 128 x 128 (stages of 128 elements: 95); of it 43 us are the outputs' stores
// (5.4 TB/s), which with three stages a tile add to the loop more than they hide behind it.  4096^3: 38.5 us = 3.6 PF; 8192^3 264 us = 4.2 PF.  e4m3 rows: 8192^3 416 us = 2.65 PF;
// 24576 x 1024 x 4096 103 us = 2.0 PF in 128 x 128 tiles; of its clocks (87 us at 2.08 GHz one at a time) the matrix units are busy 54 % and the LDS 24 %: the three workgroups of a CU
// wait at their barriers at much the same time.  A width or pitch that 16-byte pieces do not divide takes the element-wise epilogue, many times slower: 50432 x 2299 x 768 340 us.
// Built and not faster: workgroups that stay and prefetch across tiles (in both depths of stages); in stages of 128 fragments read half a stage ahead, three or four stages in
// the ring, all reads in front of the matrix instructions, raised priority around them (all within 5 %).
typedef __attribute__((address_space(3))) void* lds_ptr;
DEV void regs_pin(unsigned& v) { asm volatile("" : "+v"(v)); }
template <int N> DEV void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
constexpr unsigned FAR_AWAY = 0x7ffffff0u;

// n of row i of fragment j inside a wave's columns.  16-bit outputs: two fragments share 32 columns, so that a lane's 8 outputs of the pair are 16 bytes and four lanes 64;
// 32-bit outputs: a lane's 4 outputs of one fragment are 16 bytes.
template <typename TO> DEV constexpr int frag_col(int j) { return sizeof(TO) == 2 ? (j >> 1) * 32 + (j & 1) * 4 : j * 16; }
template <typename TO> DEV int lane_col(int i) { return sizeof(TO) == 2 ? (i >> 2) * 8 + (i & 3) : i; }

// (8 lanes read 128 bytes at a time: their 8 rows - consecutive ones of A, 0 ... 3 and 8 ... 11 of a 16-bit B - must fall on different 16-byte places.  ds_read_b128 then
// moves about 240 bytes a clock and CU; patterns that are free of conflicts over 16 lanes only reach 126.)
DEV int a_swz(int r) { return (r >> 1) & 7; }
template <typename TO> DEV int b_swz(int r) { return sizeof(TO) == 2 ? ((r >> 1) & 1) | ((r >> 2) & 2) : (r >> 1) & 3; }

template <bool A8, typename TO, int WM, int WN, int MT, int NT, int S>
struct Tile {
    static constexpr int W = WM * WN, BM = WM * MT * 16, BN = WN * NT * 16;
    static constexpr int D = A8 ? 1 : 2, PB = 64 * D;                              // instructions along K in a stage; bytes of a row of B in it (of A: 128)
    static constexpr int A_BYTES = BM * 128, B_BYTES = BN * PB, STAGE = A_BYTES + B_BYTES;
    static constexpr int NA = A_BYTES / 1024 / W, NB = B_BYTES / 1024 / W, PER = NA + NB;   // DMA instructions of a stage, per wave: of A, of B
    static constexpr int NSA = A8 ? 0 : (BM * 8 + 1023) / 1024, NS = NSA + (BN * 8 + 1023) / 1024, SC = NS * 1024;      // of the scales of 256 elements, all waves
    static constexpr int SCN = A8 ? 2 : S, LDS = S * STAGE + SCN * SC;       // places in the scales' ring
    static_assert(A_BYTES % (1024 * W) == 0 && B_BYTES % (1024 * W) == 0 && NS <= W, "whole instructions for every wave, at most one of scales");
    static_assert(NA % 2 == 0 && (D == 1 || NB % 2 == 0), "a kilobyte of 128-byte rows is 8 of them, and the chunks' order repeats after 16");
};

// block -> tile: block b runs on XCD b % 8; every XCD takes a contiguous run of tiles, ordered in groups of 8 row tiles, so that the tiles an XCD works on at a time share row
// and column panels in its L2.  `magic`: quotients by a whole group's tiles as a multiplication
struct Grid { int ntm, ntn; unsigned magic; int shift; };
inline Grid make_grid(long ntm, long ntn) {
    Grid g{(int)ntm, (int)ntn, 0, 0};
    const unsigned long d = 8 * ntn;                          // q = t / d for 0 <= t < 2^30: magic = ceil(2^(30 + shift) / d), 2^shift >= d
    while ((1ul << g.shift) < d) ++g.shift;
    g.magic = (unsigned)(((1ul << (30 + g.shift)) + d - 1) / d);
    return g;
}

template <bool A8, bool RS, typename TO, int WM, int WN, int MT, int NT, int S, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void gemm_mx_tile_kernel(const dist_gemm_mx_args p, const Grid grid, const int fast, const int slice) {
    using T = Tile<A8, TO, WM, WN, MT, NT, S>;
    extern __shared__ char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    const int part = blockIdx.y, xcd = blockIdx.x & 7, each = gridDim.x >> 3, more = gridDim.x & 7;
    const int t0 = xcd * each + min(xcd, more) + (int)(blockIdx.x >> 3);
    const int grp = (int)(((unsigned long)(unsigned)t0 * grid.magic) >> (30 + grid.shift)), in = t0 - grp * 8 * grid.ntn, gm = grid.ntm - grp * 8;
    const int tn = gm >= 8 ? in >> 3 : in / gm, tm = grp * 8 + (gm >= 8 ? in & 7 : in - tn * gm);
    const long m0 = (long)tm * T::BM;
    const int n0 = tn * T::BN;

    // elements k0 ... k0 + K of the long axis: all of them, or slice number `part` (then C is its fp32 partial result, without bias, residual and row scales)
    const int k0 = part * slice, K = min(slice, p.K - k0), chunk0 = k0 >> 8;
    const int pitch_a = A8 ? (int)p.lda : p.K / 2, pitch_b = p.K / 2;
    const int mrows = (int)min((long)T::BM, p.M - m0), nrows = min(T::BN, p.N - n0), ka = A8 ? k0 : k0 / 2;
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(p.A) + m0 * pitch_a + ka), 0, mrows * pitch_a - ka, 0x00020000);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(p.B) + (long)n0 * pitch_b + k0 / 2), 0, nrows * pitch_b - k0 / 2, 0x00020000);
    constexpr int KS = 128 * T::D;
    const int nk = (K + KS - 1) / KS, tail = K - (nk - 1) * KS;                     // stages; elements of the last one

    // The lane's offsets: its row of the wave's first kilobyte and its chunk; the further kilobytes are steps of whole rows in the scalar offset, which the descriptor's range
    // check counts in.  (Registers of their own that change once, under a branch: hipcc waits for every load in flight before it reuses one that a load takes its address from.)
    constexpr int LB = T::PB / 16, RB = 64 / LB;                                   // lanes per row of B, rows of a kilobyte (of A: 8 and 8)
    unsigned va[2], vb[T::D];                                                      // (the chunks' order repeats after 16 rows)
    auto offsets = [&](const int limit) __attribute__((always_inline)) {           // limit: elements of the stage, what lies behind is sent away
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int r = wave * T::NA * 8 + (lane >> 3), c = (lane & 7) ^ a_swz(r + q * 8);
            va[q] = c * (A8 ? 16 : 32) >= limit ? FAR_AWAY : (unsigned)(r * pitch_a + c * 16);
            regs_pin(va[q]);
        }
#pragma unroll
        for (int q = 0; q < T::D; ++q) {
            const int r = wave * T::NB * RB + lane / LB, c = (lane % LB) ^ b_swz<TO>(r + q * RB);
            vb[q] = c * 32 >= limit ? FAR_AWAY : (unsigned)(r * pitch_b + c * 16);
            regs_pin(vb[q]);
        }
    };
    offsets(KS);
    // the wave's kilobyte of scales (a wave without one of its own repeats the last: the same bytes to the same place)
    const int sk = min(wave, T::NS - 1);
    const bool sa = sk < T::NSA;
    const long sstep = (sa ? p.M : (long)p.N) * 8;
    const int sfirst = (sa ? sk : sk - T::NSA) * 1024, sleft = max((sa ? mrows : nrows) * 8 - sfirst, 0);
    const char* const ssrc = (sa ? static_cast<const char*>(p.a_scale) + m0 * 8 : static_cast<const char*>(p.b_scale) + (long)n0 * 8) + chunk0 * sstep + sfirst;
    unsigned lane16 = lane * 16;
    regs_pin(lane16);
    auto issue_scales = [&](const int chunk) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(ssrc + chunk * sstep), 0, sleft, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(smem + S * T::STAGE + sk * 1024 + (chunk % T::SCN) * T::SC), 16, lane16, 0, 0, 0);
    };
    auto issue = [&](const int kt) __attribute__((always_inline)) {
        char* base = smem + (kt % S) * T::STAGE;
        if (!A8) issue_scales(kt);
        else if ((kt & 1) == 0) issue_scales(kt >> 1);
        if (kt == nk - 1 && tail < KS) offsets(tail);
#pragma unroll
        for (int q = 0; q < T::NA; ++q) {
            const unsigned v = va[q % 2];
            const int step = kt * 128 + q * 8 * pitch_a;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr)(base + (wave * T::NA + q) * 1024), 16, v, step, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < T::NB; ++q) {
            const unsigned v = vb[q % T::D];
            const int step = kt * T::PB + q * RB * pitch_b;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr)(base + T::A_BYTES + (wave * T::NB + q) * 1024), 16, v, step, 0, 0);
        }
    };

    // LDS addresses of this lane's fragments inside a stage
    const int arow = wm * MT * 16 + i, brow = wn * NT * 16 + lane_col<TO>(i);
    const int a_lo = arow * 128 + ((g ^ a_swz(arow)) << 4), a_hi = arow * 128 + (((4 + g) ^ a_swz(arow)) << 4);
    const int b_lo = T::A_BYTES + brow * T::PB + ((g ^ b_swz<TO>(brow)) << 4), b_hi = T::A_BYTES + brow * T::PB + (((4 + g) ^ b_swz<TO>(brow)) << 4);

    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    int as[MT], bs[NT];
#pragma unroll
    for (int t = 0; t < MT; ++t) as[t] = 127;

    // stage kt; P: which half of 256 elements it begins with (e4m3: kt & 1, 4-bit operands: 0)
    auto stage = [&](auto par, const int kt) __attribute__((always_inline)) {
        constexpr int P = decltype(par)::value, SCALES = A8 ? (S - 2 + P) / 2 : S - 2;     // kilobytes of scales among stages kt + 1 ... kt + S - 2, which may stay in flight
        if (kt + S - 2 < nk) wait_vm<(S - 2) * T::PER + SCALES>();
        else wait_vm<0>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (kt + S - 1 < nk) issue(kt + S - 1);
        __builtin_amdgcn_sched_barrier(0);
        const char* base = smem + (kt % S) * T::STAGE;
        if constexpr (P == 0) {
            const char* sc = smem + S * T::STAGE + ((A8 ? kt >> 1 : kt) % T::SCN) * T::SC;
            if constexpr (!A8)
#pragma unroll
                for (int t = 0; t < MT; ++t) as[t] = *reinterpret_cast<const unsigned short*>(sc + (arow + t * 16) * 8 + 2 * g);
#pragma unroll
            for (int j = 0; j < NT; ++j) bs[j] = *reinterpret_cast<const unsigned short*>(sc + T::NSA * 1024 + (brow + frag_col<TO>(j)) * 8 + 2 * g);
        }
        auto step = [&](auto half) __attribute__((always_inline)) {
            constexpr int H = decltype(half)::value;
            v8i_t a[MT], b[NT];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if constexpr (A8) a[t] = join(*reinterpret_cast<const v4i_t*>(base + a_lo + t * 2048), *reinterpret_cast<const v4i_t*>(base + a_hi + t * 2048));
                else a[t] = widen(*reinterpret_cast<const v4i_t*>(base + (H ? a_hi : a_lo) + t * 2048));
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j] = widen(*reinterpret_cast<const v4i_t*>(base + (!A8 && H ? b_hi : b_lo) + frag_col<TO>(j) * T::PB));
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int t = 0; t < MT; ++t) mma<A8, H>(b[j], a[t], acc[t][j], bs[j], as[t]);
        };
        step(par);
        if constexpr (!A8) step(std::integral_constant<int, 1>{});
    };

#pragma unroll
    for (int k = 0; k < S - 1; ++k)
        if (k < nk) issue(k);
    constexpr std::integral_constant<int, 0> zero{};
    constexpr std::integral_constant<int, 1> one{};
    if constexpr (A8) {
        for (int kt = 0; kt < nk; kt += 2) {
            stage(zero, kt);
            if (kt + 1 < nk) stage(one, kt + 1);
        }
    } else {
        for (int kt = 0; kt < nk; ++kt) stage(zero, kt);
    }

    // ---- outputs
    const long mw = m0 + wm * MT * 16 + i;
    float rs[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) rs[t] = A8 && RS && mw + t * 16 < p.M ? static_cast<const float*>(p.a_scale)[mw + t * 16] : 1.f;
    // 16-byte stores through a descriptor that ends behind the last row; columns behind N are sent past it.  Lanes i and i ^ 8 exchange, so that a store writes 8 rows of
    // 128 bytes and not 16 of 64, past the caches' keeping: a 232 MB output takes 43 us this way and 64 us in half lines kept in the L2
    // (The steps of the rows are in the lanes' offset: behind a 16-byte store whose scalar offset is a register hipcc writes the store's data anew in the very next instruction,
    // and gfx950 then stores the new value in some lanes.  With a constant scalar offset hipcc keeps the distance.)
    constexpr int U = sizeof(TO) == 2 ? 2 : 1, ES = sizeof(TO);                    // fragments of one 16-byte store
    const int rowl = wm * MT * 16 + i, coll = wn * NT * 16 + g * (4 * U);
    TO* const C = static_cast<TO*>(p.C) + part * (p.M * p.ldc);                    // (slices lie one behind the other)
    if (fast) {
        const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(C) + (m0 * p.ldc + n0) * ES, 0, (int)((mrows * p.ldc - n0) * ES), 0x00020000);
        const __amdgpu_buffer_rsrc_t rr = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(p.res)) + (m0 * p.ldres + n0) * ES, 0, p.res ? (int)((mrows * p.ldres - n0) * ES) : 0, 0x00020000);
        const bool up = (i & 8) != 0;
        const int colx = coll + (up ? frag_col<TO>(U) : 0), stepc = (int)(8 * p.ldc * ES), stepr = (int)(16 * p.ldres * ES);
        const unsigned cbase = (unsigned)((rowl - (up ? 8 : 0)) * (int)p.ldc + colx) * ES, rbase = (unsigned)(rowl * (int)p.ldres + coll) * ES;
#pragma unroll
        for (int j = 0; j < NT; j += 2 * U) {
            v4u_t q[MT][2];
            if (p.res) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const unsigned v = n0 + coll + frag_col<TO>(j + h * U) < p.N ? rbase + frag_col<TO>(j + h * U) * ES : FAR_AWAY;
#pragma unroll
                    for (int t = 0; t < MT; ++t) q[t][h] = __builtin_amdgcn_raw_buffer_load_b128(rr, v, t * stepr, 0);
                }
            }
            float bias[2][4 * U];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = n0 + coll + frag_col<TO>(j + h * U);
#pragma unroll
                for (int e = 0; e < 4 * U; ++e) bias[h][e] = 0.f;
                if (p.bias && n < p.N) {
                    if constexpr (U == 2) mx::load_v8(p.bias + n, bias[h]);
                    else load4(p.bias + n, bias[h]);
                }
            }
            const unsigned at = n0 + colx + frag_col<TO>(j) < p.N ? cbase + frag_col<TO>(j) * ES : FAR_AWAY;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                v4u_t out[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[4 * U];
#pragma unroll
                    for (int e = 0; e < 4 * U; ++e) v[e] = (A8 ? acc[t][j + h * U + e / 4][e % 4] * rs[t] : acc[t][j + h * U + e / 4][e % 4]) + bias[h][e];
                    if constexpr (U == 2) {
                        if (p.res) {
                            const bf16x8 f = __builtin_bit_cast(bf16x8, q[t][h]);
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] += (float)f[e];
                        }
                        Frag<bf16_t> f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) frag_set(f, e, v[e]);
                        out[h] = __builtin_bit_cast(v4u_t, f.v);
                    } else {
                        if (p.res) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] += __uint_as_float(q[t][h][e]);
                        }
                        out[h] = v4u_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
                    }
                }
                v4u_t o0, o1;                                                      // rows 0 ... 7: the upper lanes take the lower lanes' second half;  rows 8 ... 15 the other way
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o0[e] = (unsigned)__builtin_amdgcn_update_dpp((int)out[0][e], (int)out[1][e], 0x128 /* row_ror:8 */, 0xf, 0xc, false);
                    o1[e] = (unsigned)__builtin_amdgcn_update_dpp((int)out[1][e], (int)out[0][e], 0x128, 0xf, 0x3, false);
                }
                __builtin_amdgcn_raw_buffer_store_b128(o0, rc, at + 2 * t * stepc, 0, 2);
                __builtin_amdgcn_raw_buffer_store_b128(o1, rc, at + (2 * t + 1) * stepc, 0, 2);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const long m = mw + t * 16;
            const int c = wn * NT * 16 + frag_col<TO>(j & ~(U - 1)) + g * (4 * U) + (j & (U - 1)) * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (m < p.M && n0 + c + e < p.N) {
                    const float v = (A8 ? acc[t][j][e] * rs[t] : acc[t][j][e]) + (p.bias ? p.bias[n0 + c + e] : 0.f);
                    C[m * p.ldc + n0 + c + e] = from_f<TO>(v + (p.res ? to_f(static_cast<const TO*>(p.res)[m * p.ldres + n0 + c + e]) : 0.f));
                }
        }
}

// C = bias + res + a_scale * sum of the slices, in their order
template <bool A8, typename TO>
__global__ __launch_bounds__(NT_) void gemm_mx_join_kernel(const dist_gemm_mx_args p, const float* __restrict__ part, const int parts) {
    const long e = (long)blockIdx.x * NT_ + threadIdx.x, size = p.M * p.N;
    if (e >= size) return;
    const long m = e / p.N;
    const int n = (int)(e - m * p.N);
    float s = part[e];
    for (int k = 1; k < parts; ++k) s += part[k * size + e];
    if (A8) s *= static_cast<const float*>(p.a_scale)[m];
    static_cast<TO*>(p.C)[m * p.ldc + n] = from_f<TO>(s + (p.bias ? p.bias[n] : 0.f) + (p.res ? to_f(static_cast<const TO*>(p.res)[m * p.ldres + n]) : 0.f));
}

template <bool A8, bool RS, typename TO, int WM, int WN, int MT, int NT, int S, int OCC> int launch_tile(const dist_gemm_mx_args& p, int slice, hipStream_t s) {
    using T = Tile<A8, TO, WM, WN, MT, NT, S>;
    const long ntm = (p.M + T::BM - 1) / T::BM, ntn = (p.N + T::BN - 1) / T::BN, parts = (p.K + slice - 1) / slice;
    if (mx::too_many(ntm * ntn, 64 * T::W) || parts > 65535) return DIST_ERR_ARG;
    const auto k = gemm_mx_tile_kernel<A8, RS, TO, WM, WN, MT, NT, S, OCC>;
    static DistSmemOnce st;
    RUN_(dist_max_smem(st, reinterpret_cast<const void*>(k), T::LDS));
    constexpr size_t ES = sizeof(TO);
    const bool fast = p.N % (16 / ES) == 0 && (uintptr_t)p.C % 16 == 0 && p.ldc * ES % 16 == 0 && p.ldc <= 1 << 20 && (!p.bias || (uintptr_t)p.bias % 16 == 0) &&
                      (!p.res || ((uintptr_t)p.res % 16 == 0 && p.ldres * ES % 16 == 0 && p.ldres <= 1 << 20));
    hipLaunchKernelGGL(k, dim3((unsigned)(ntm * ntn), (unsigned)parts), dim3(64 * T::W), T::LDS, s, p, make_grid(ntm, ntn), (int)fast, slice);
    HIP_CHECK_RET(hipGetLastError());
    return DIST_OK;
}

enum { FEW = 0, SMALL = 1, SQUARE = 2, BIG = 3 };
struct Plan { int kind, slice; };
constexpr int LIMIT = 1 << 22;                               // bytes of a row (the 256 rows of a tile lie within 32-bit offsets)

// Which kernel (times in us, inputs out of the caches, bf16 out, bias; kernels of this file beside each other, the middle of seven graphs in turn):
//   FEW     M <= 64.  N = K = 4096: 16 rows 5.2 against 8.7 in 64 x 64 tiles, 48 rows 8.2 against 8.7, 64 rows 9.2 against 8.9.  Its time grows with the rows and with N, that of
//           the tiles hardly: with wide weights they would be the faster from 17 rows on (24 x 16384 x 4096 15.5 against 9.4, 64 x 8192 x 8192 26 against 14.6)
//   SMALL   64 x 64, where 128 x 128 would leave CUs without work (under 200 tiles): 788 x 2304 x 768 5.0 against 5.6; 2048 x 2048 x 1024 (256 tiles) 9.3 against 6.9 the other way.
//           2304 x 768 x 12608 (108 tiles) 33.5 against 43.4.
//           The long axis is cut where even these do not fill the 256 CUs, in slices of at least 2048 (shorter ones cost more in the joining pass than they gain:
//           200 x 520 x 2048 6.0 whole, 6.9 in two).  768 x 768 x 12608 (144 tiles) is 20.8 whole, 23.4 in two
//   SQUARE  128 x 128, two workgroups a CU (e4m3: three)
//   BIG     256 x 256, one a CU: four times the work of SQUARE, so it wins where its rounds over the 256 CUs are full.  4-bit rows: 4096^3 38.5 against 43, 8192^3 264 against 291,
//           32768 x 1024 x 4096 78 against 88, 6400 x 2304 x 768 (225 tiles) 12.9 against 14.1, but 16448 x 1024 x 4096 (260 tiles) 63 against 51.
//           e4m3 rows: only in a single round, or with a long axis beside which the outputs are short - nothing else runs on the CU while its one workgroup stores, and SQUARE has three:
//           4096^3 55 against 58, 16384 x 1024 x 4096 54 against 57.5, 6400 x 2304 x 768 16.5 against 17.9, 32768 x 1024 x 4096 118 against 131, 8192^3 416 against 414, but several rounds
//           of short axes 50432 x 2304 x 768 108 against 98, 25600 x 2304 x 768 61 against 54, 16384 x 2048 x 2048 63 against 59
Plan plan(int64_t M, int N, int K, bool a8) {
    const int64_t t64 = (M + 63) / 64 * ((N + 63) / 64), t128 = (M + 127) / 128 * ((N + 127) / 128), t256 = (M + 255) / 256 * ((N + 255) / 256);
    if (M <= 64) return Plan{FEW, K};
    if (t128 >= 200) return Plan{15 * ((t256 + 255) / 256) <= 4 * ((t128 + 255) / 256) && (!a8 || t256 <= 256 || K >= 4096) ? BIG : SQUARE, K};
    int parts = 1;
    while (t64 * parts < 256 && K / (2 * parts) >= 2048) parts *= 2;
    return Plan{SMALL, parts == 1 ? K : (K / parts + 255) / 256 * 256};
}

template <bool A8, typename TO, int MT, int NT, int W> int launch_few(const dist_gemm_mx_args& p, hipStream_t s) {
    const int64_t blocks = ((int64_t)p.N + 16 * NT - 1) / (16 * NT);
    if (mx::too_many(blocks, 64 * W)) return DIST_ERR_ARG;
    hipLaunchKernelGGL((gemm_mx_few_kernel<A8, TO, MT, NT, W>), dim3((unsigned)blocks), dim3(64 * W), 0, s, p);
    HIP_CHECK_RET(hipGetLastError());
    return DIST_OK;
}

template <bool A8, typename TO> int launch(const dist_gemm_mx_args& p, hipStream_t s) {
    const Plan w = plan(p.M, p.N, p.K, A8);
    if (w.kind == FEW) {
        if (p.M <= 16) return launch_few<A8, TO, 1, 1, 8>(p, s);
        if (p.M <= 32) return launch_few<A8, TO, 2, 1, 8>(p, s);
        return launch_few<A8, TO, 4, 1, 8>(p, s);
    }
    // (64 x 128 a wave where 128 x 64 needs more registers: e4m3 fragments, fp32 residuals)
    constexpr bool TALL = !A8 && sizeof(TO) == 2;
    if (w.kind == BIG) return launch_tile<A8, true, TO, TALL ? 2 : 4, TALL ? 4 : 2, TALL ? 8 : 4, TALL ? 4 : 8, 2, 2>(p, p.K, s);
    if (w.kind == SQUARE) return launch_tile<A8, true, TO, 2, 2, 4, 4, 2, A8 ? 3 : 2>(p, p.K, s);
    if (w.slice >= p.K) return launch_tile<A8, true, TO, 4, 1, 1, 4, 4, 4>(p, p.K, s);
    dist_gemm_mx_args q = p;
    q.C = p.scratch;
    q.ldc = p.N;
    q.bias = nullptr;
    q.res = nullptr;
    RUN_((launch_tile<A8, false, float, 4, 1, 1, 4, 4, 4>(q, w.slice, s)));
    const long blocks = (p.M * p.N + NT_ - 1) / NT_;
    hipLaunchKernelGGL((gemm_mx_join_kernel<A8, TO>), dim3((unsigned)blocks), dim3(NT_), 0, s, p, p.scratch, (p.K + w.slice - 1) / w.slice);
    HIP_CHECK_RET(hipGetLastError());
    return DIST_OK;
}

}  // namespace

extern "C" int64_t dist_op_gemm_mxfp4_scratch(int64_t M, int N, int K, int a_fmt) {
    if (M < 0 || N <= 0 || N > 1 << 30 || K <= 0 || K % 32 || (a_fmt != DIST_MX_A_MXFP4 && a_fmt != DIST_MX_A_E4M3)) return -1;
    const Plan w = plan(M, N, K, a_fmt == DIST_MX_A_E4M3);
    const int64_t parts = (K + w.slice - 1) / w.slice;
    return parts > 1 ? parts * M * N : 0;
}

extern "C" int dist_op_gemm_mxfp4(const dist_gemm_mx_args* a, void* stream) {
    if (!a) return DIST_ERR_ARG;
    const dist_gemm_mx_args p = *a;
    if (p.a_fmt != DIST_MX_A_MXFP4 && p.a_fmt != DIST_MX_A_E4M3) return DIST_ERR_ARG;
    if ((p.dtype != DIST_BF16 && p.dtype != DIST_F32) || (p.a_fmt == DIST_MX_A_E4M3 && p.dtype != DIST_BF16)) return DIST_ERR_ARG;
    if (p.M < 0 || p.N <= 0 || p.N > 1 << 30 || p.K <= 0 || p.K % 32 || p.K > LIMIT) return DIST_ERR_ARG;
    if (p.M == 0) return DIST_OK;
    const uintptr_t es = p.dtype == DIST_BF16 ? 2 : 4;
    if (!p.A || !p.a_scale || !p.B || !p.b_scale || !p.C || p.ldc < p.N || (p.res && p.ldres < p.N)) return DIST_ERR_ARG;
    if ((uintptr_t)p.A % 16 || (uintptr_t)p.B % 16 || (uintptr_t)p.b_scale % 8 || (uintptr_t)p.a_scale % (p.a_fmt == DIST_MX_A_E4M3 ? 4 : 8)) return DIST_ERR_ARG;
    if (p.a_fmt == DIST_MX_A_E4M3 && (p.lda < p.K || p.lda % 16 || p.lda > LIMIT)) return DIST_ERR_ARG;
    if ((uintptr_t)p.C % es || (uintptr_t)p.res % es || (uintptr_t)p.bias % 4) return DIST_ERR_ARG;
    const int64_t need = dist_op_gemm_mxfp4_scratch(p.M, p.N, p.K, p.a_fmt);
    if (need > 0 && (p.scratch_elems < need || !p.scratch || (uintptr_t)p.scratch % 16)) return DIST_ERR_WORKSPACE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.a_fmt == DIST_MX_A_E4M3) return launch<true, bf16_t>(p, s);
    return p.dtype == DIST_BF16 ? launch<false, bf16_t>(p, s) : launch<false, float>(p, s);
}
