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
constexpr int NT_ = 256;

DEV v8i_t widen(const int4& lo) { v8i_t r = {lo.x, lo.y, lo.z, lo.w, 0, 0, 0, 0}; return r; }
DEV v8i_t join(const int4& lo, const int4& hi) { v8i_t r = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}; return r; }

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
    const int4 zero = make_int4(0, 0, 0, 0);
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
            for (int j = 0; j < NT; ++j) b[j] = widen(k + g * 32 < p.K ? *reinterpret_cast<const int4*>(B + bn[j] * (p.K / 2) + k / 2 + g * 16) : zero);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if constexpr (A8) {
                    const unsigned char* q = A + am[t] * p.lda + k;
                    a[t] = join(k + g * 16 < p.K ? *reinterpret_cast<const int4*>(q + g * 16) : zero, k + 64 + g * 16 < p.K ? *reinterpret_cast<const int4*>(q + 64 + g * 16) : zero);
                } else a[t] = widen(k + g * 32 < p.K ? *reinterpret_cast<const int4*>(A + am[t] * (p.K / 2) + k / 2 + g * 16) : zero);
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

template <bool A8, typename TO> int launch(const dist_gemm_mx_args& p, hipStream_t s) {
    const size_t es = sizeof(TO);
    const int vec = (uintptr_t)p.C % 16 == 0 && p.ldc * es % 16 == 0 && (!p.res || ((uintptr_t)p.res % 16 == 0 && p.ldres * es % 16 == 0)) && (!p.bias || (uintptr_t)p.bias % 16 == 0);
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
