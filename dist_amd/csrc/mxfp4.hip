// MXFP4 quantisation (dist_op_quant_mxfp4) along the rows or the columns of a matrix, and the way back (dist_op_dequant_mxfp4).  mx.h holds the format.
// One pass each, HBM-bound: 2 (bf16) or 4 (fp32) bytes against 17 / 32 byte per element.
#include "mx.h"

namespace {

constexpr int NT = 256;

// Along the rows.  32 lanes own a chunk of 256 elements of one row, 8 consecutive elements a lane: a block is four neighbouring lanes, its maximum two shuffles.
template <typename T, bool AL>
__global__ __launch_bounds__(NT) void quant_rows_kernel(const T* __restrict__ x, const long rows, const long K, const long ld, const int Kp, const int chunks,
                                                        unsigned char* __restrict__ codes, unsigned char* __restrict__ scales) {
    const long item = (long)blockIdx.x * (NT / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const long row = item / chunks;
    const int chunk = (int)(item - row * chunks);
    if (row >= rows) return;                                 // (a whole half-wave: the shuffles below stay inside it)
    const long c0 = (long)chunk * mx::CHUNK + lane * 8;
    float v[8];
    mx::load8<AL>(x + row * ld + c0, K - c0, v);
    unsigned a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, mx::abs_bits(v[e]));
    a = max(a, (unsigned)__shfl_xor((int)a, 1, 64));
    a = max(a, (unsigned)__shfl_xor((int)a, 2, 64));
    const int byte = mx::scale_byte(a);
    if (c0 < Kp) *reinterpret_cast<unsigned*>(codes + row * (Kp / 2) + c0 / 2) = mx::pack8(v, byte);
    if ((lane & 3) == 0) scales[mx::scale_at(row, rows, chunk * 8 + (lane >> 2))] = (unsigned char)(c0 < Kp ? byte : 0);
}

// Along the columns: output row c holds the elements x[:, c].  A workgroup takes 256 rows of x (a chunk) and 64 VC columns, a wave one block of 32 rows: every load of a row is
// 64 VC neighbouring elements, a lane ends with the 32 elements of its VC blocks and needs no exchange.  Codes and scales go through LDS, so that a column's 128
// bytes of codes and the columns' 8 bytes of scales are written as whole lines.
template <typename T, int VC>
__global__ __launch_bounds__(512) void quant_cols_kernel(const T* __restrict__ x, const long R, const int C, const long ld, const long Kp, const int ctiles,
                                                         unsigned char* __restrict__ codes, unsigned char* __restrict__ scales) {
    __shared__ uint4 lc[64 * VC][9];                          // (a 16-byte pad: the waves' columns fall on different banks)
    __shared__ unsigned char ls[64 * VC][8];
    typedef T vec_t __attribute__((ext_vector_type(VC)));
    const int chunk = blockIdx.x / ctiles, lane = threadIdx.x & 63, b = threadIdx.x >> 6, ct0 = (blockIdx.x - chunk * ctiles) * 64 * VC, c = ct0 + lane * VC;
    const long r0 = (long)chunk * mx::CHUNK + b * mx::BLOCK;
    float v[VC][32];
    if (c < C) {
        const T* src = x + r0 * ld + c;
        if (r0 + 32 <= R) {
            vec_t w[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) w[e] = *reinterpret_cast<const vec_t*>(src + e * ld);
#pragma unroll
            for (int e = 0; e < 32; ++e)
#pragma unroll
                for (int k = 0; k < VC; ++k) v[k][e] = to_f((T)w[e][k]);
        } else {
#pragma unroll
            for (int e = 0; e < 32; ++e)
#pragma unroll
                for (int k = 0; k < VC; ++k) v[k][e] = r0 + e < R ? to_f(src[e * ld + k]) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < VC; ++k) {
            unsigned a = 0;
#pragma unroll
            for (int e = 0; e < 32; ++e) a = max(a, mx::abs_bits(v[k][e]));
            const int byte = mx::scale_byte(a);
            uint4 w;
            w.x = mx::pack8(v[k], byte); w.y = mx::pack8(v[k] + 8, byte); w.z = mx::pack8(v[k] + 16, byte); w.w = mx::pack8(v[k] + 24, byte);
            lc[lane * VC + k][b] = w;
            ls[lane * VC + k][2 * (b & 3) + (b >> 2)] = (unsigned char)(r0 < Kp ? byte : 0);
        }
    }
    __syncthreads();
    for (int q = threadIdx.x; q < 64 * VC * 8; q += 512) {
        const int col = q >> 3, blk = q & 7;
        const long k = (long)chunk * mx::CHUNK + blk * mx::BLOCK;
        if (ct0 + col < C && k < Kp) *reinterpret_cast<uint4*>(codes + (ct0 + col) * (Kp / 2) + k / 2) = lc[col][blk];
    }
    if (threadIdx.x < 64 * VC && ct0 + (int)threadIdx.x < C)
        *reinterpret_cast<uint2*>(scales + ((long)chunk * C + ct0 + threadIdx.x) * 8) = *reinterpret_cast<const uint2*>(ls[threadIdx.x]);
}

template <typename T>
__global__ __launch_bounds__(NT) void dequant_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales, const long rows, const int Kp,
                                                     T* __restrict__ y) {
    const long i = (long)blockIdx.x * NT + threadIdx.x;       // eight elements
    const int per = Kp / 8;
    const long row = i / per;
    const int v8 = (int)(i - row * per);
    if (row >= rows) return;
    float v[8];
    mx::unpack8(reinterpret_cast<const unsigned*>(codes)[i], scales[mx::scale_at(row, rows, v8 / 4)], v);
    mx::store8<true>(y + i * 8, 8, v);
}

}  // namespace

extern "C" int64_t dist_op_mxfp4_scale_bytes(int64_t rows, int64_t K) {
    return rows < 0 || K <= 0 ? -1 : (K + mx::CHUNK - 1) / mx::CHUNK * 8 * rows;
}

extern "C" int dist_op_quant_mxfp4(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, int transpose, void* codes, void* scales, void* stream) {
    if (rows < 0 || cols < 0 || ld < cols || (dtype != DIST_BF16 && dtype != DIST_F32)) return DIST_ERR_ARG;
    const int64_t out_rows = transpose ? cols : rows, K = transpose ? rows : cols;
    if (K <= 0 || K > (1l << 30) || out_rows > (1l << 30)) return DIST_ERR_ARG;
    if (out_rows == 0) return DIST_OK;
    if (!x || !codes || !scales || (uintptr_t)codes % 16 || (uintptr_t)scales % 8 || (uintptr_t)x % (dtype == DIST_BF16 ? 2 : 4)) return DIST_ERR_ARG;
    hipStream_t s = static_cast<hipStream_t>(stream);
    unsigned char *q = static_cast<unsigned char*>(codes), *sc = static_cast<unsigned char*>(scales);
    const int64_t Kp = (K + 31) / 32 * 32, chunks = (K + mx::CHUNK - 1) / mx::CHUNK;
    if (!transpose) {
        const int64_t blocks = (rows * chunks + NT / 32 - 1) / (NT / 32);
        if (mx::too_many(blocks, NT)) return DIST_ERR_ARG;
        const bool al = cols % 8 == 0 && ld % 8 == 0 && (uintptr_t)x % 16 == 0;
#define DIST_QR(T, AL) hipLaunchKernelGGL((quant_rows_kernel<T, AL>), dim3((unsigned)blocks), dim3(NT), 0, s, static_cast<const T*>(x), (long)rows, (long)K, (long)ld, (int)Kp, (int)chunks, q, sc)
        if (dtype == DIST_BF16) { if (al) DIST_QR(bf16_t, true); else DIST_QR(bf16_t, false); }
        else { if (al) DIST_QR(float, true); else DIST_QR(float, false); }
#undef DIST_QR
    } else {
        const bool two = dtype == DIST_BF16 && cols % 2 == 0 && ld % 2 == 0 && (uintptr_t)x % 4 == 0;        // two bf16 columns a lane
        const int64_t ctiles = two ? (cols + 127) / 128 : (cols + 63) / 64, blocks = ctiles * chunks;
        if (mx::too_many(blocks, 512)) return DIST_ERR_ARG;
#define DIST_QC(T, VC) hipLaunchKernelGGL((quant_cols_kernel<T, VC>), dim3((unsigned)blocks), dim3(512), 0, s, static_cast<const T*>(x), (long)rows, (int)cols, (long)ld, (long)Kp, (int)ctiles, q, sc)
        if (two) DIST_QC(bf16_t, 2); else if (dtype == DIST_BF16) DIST_QC(bf16_t, 1); else DIST_QC(float, 1);
#undef DIST_QC
    }
    HIP_CHECK_RET(hipGetLastError());
    return DIST_OK;
}

extern "C" int dist_op_dequant_mxfp4(const void* codes, const void* scales, int64_t rows, int64_t K, void* y, int dtype, void* stream) {
    if (rows < 0 || K <= 0 || K % 32 || K > (1l << 30) || rows > (1l << 30) || (dtype != DIST_BF16 && dtype != DIST_F32)) return DIST_ERR_ARG;
    if (rows == 0) return DIST_OK;
    if (!codes || !scales || !y || (uintptr_t)codes % 16 || (uintptr_t)y % 16) return DIST_ERR_ARG;
    const int64_t blocks = (rows * (K / 8) + NT - 1) / NT;
    if (mx::too_many(blocks, NT)) return DIST_ERR_ARG;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned char *q = static_cast<const unsigned char*>(codes), *sc = static_cast<const unsigned char*>(scales);
    if (dtype == DIST_BF16) hipLaunchKernelGGL(dequant_kernel<bf16_t>, dim3((unsigned)blocks), dim3(NT), 0, s, q, sc, (long)rows, (int)K, static_cast<bf16_t*>(y));
    else hipLaunchKernelGGL(dequant_kernel<float>, dim3((unsigned)blocks), dim3(NT), 0, s, q, sc, (long)rows, (int)K, static_cast<float*>(y));
    HIP_CHECK_RET(hipGetLastError());
    return DIST_OK;
}
