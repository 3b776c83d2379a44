// MXFP4 quantisation (dist_op_quant_mxfp4) along the rows or the columns of a matrix, and the way back (dist_op_dequant_mxfp4).  mx.h holds the format.
// One pass each, HBM-bound: 2 (bf16) or 4 (fp32) bytes against 17 / 32 byte per element.
#include "mx.h"

namespace {

constexpr int NT = 256;

// Along the rows.  32 lanes own a chunk of 256 elements of one row, 8 consecutive elements a lane: a block is four neighbouring lanes, its maximum two shuffles.
// V = 1: any alignment and any tail, elements read one by one (a lane's loads past K give zeros).
template <typename T, int V>
__global__ __launch_bounds__(NT) void quant_rows_kernel(const T* __restrict__ x, const long rows, const long K, const long ld, const int Kp, const int chunks,
                                                        unsigned char* __restrict__ codes, unsigned char* __restrict__ scales) {
    const long item = (long)blockIdx.x * (NT / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const long row = item / chunks;
    const int chunk = (int)(item - row * chunks);
    if (row >= rows) return;                                 // (a whole half-wave: the shuffles below stay inside it)
    const long c0 = (long)chunk * mx::CHUNK + lane * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    const T* xr = x + row * ld;
    if constexpr (V == 8) {
        if (c0 < K) mx::load_v<8>(xr + c0, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c0 + e < K) v[e] = to_f(xr[c0 + e]);
    }
    unsigned a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, mx::abs_bits(v[e]));
    a = max(a, (unsigned)__shfl_xor((int)a, 1, 64));
    a = max(a, (unsigned)__shfl_xor((int)a, 2, 64));
    const int byte = mx::scale_byte(a);
    if (c0 < Kp) *reinterpret_cast<unsigned*>(codes + row * (Kp / 2) + c0 / 2) = mx::pack8(v, byte);
    if ((lane & 3) == 0) scales[mx::scale_at(row, rows, chunk * 8 + (lane >> 2))] = (unsigned char)(c0 < Kp ? byte : 0);
}

// Along the columns: output row c holds the elements x[:, c].  A wave owns one block (32 rows of x) of 64 columns: every load of a row is 64 neighbouring elements,
// a lane ends with the 32 elements of its block and needs no exchange.
template <typename T>
__global__ __launch_bounds__(NT) void quant_cols_kernel(const T* __restrict__ x, const long R, const int C, const long ld, const long Kp, const long nblk, const int ctiles,
                                                        unsigned char* __restrict__ codes, unsigned char* __restrict__ scales) {
    const long item = (long)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
    const long ct = item / nblk, b = item - ct * nblk;
    const int c = (int)ct * 64 + (threadIdx.x & 63);
    if (ct >= ctiles || c >= C) return;
    const long r0 = b * mx::BLOCK;
    float v[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = r0 + e < R ? to_f(x[(r0 + e) * ld + c]) : 0.f;
    unsigned a = 0;
#pragma unroll
    for (int e = 0; e < 32; ++e) a = max(a, mx::abs_bits(v[e]));
    const int byte = mx::scale_byte(a);
    if (r0 < Kp) {
        uint4 w;
        w.x = mx::pack8(v, byte); w.y = mx::pack8(v + 8, byte); w.z = mx::pack8(v + 16, byte); w.w = mx::pack8(v + 24, byte);
        *reinterpret_cast<uint4*>(codes + (long)c * (Kp / 2) + r0 / 2) = w;
    }
    scales[mx::scale_at(c, C, (int)b)] = (unsigned char)(r0 < Kp ? byte : 0);
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
    mx::store_v<8>(y + i * 8, v);
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
    if (!x || !codes || !scales || (uintptr_t)codes % 16 || (uintptr_t)x % (dtype == DIST_BF16 ? 2 : 4)) return DIST_ERR_ARG;
    hipStream_t s = static_cast<hipStream_t>(stream);
    unsigned char *q = static_cast<unsigned char*>(codes), *sc = static_cast<unsigned char*>(scales);
    const int64_t Kp = (K + 31) / 32 * 32, chunks = (K + mx::CHUNK - 1) / mx::CHUNK;
    if (!transpose) {
        const int64_t blocks = (rows * chunks + NT / 32 - 1) / (NT / 32);
        if (blocks > 0x7fffffff) return DIST_ERR_ARG;
        const bool vec = cols % 8 == 0 && ld % 8 == 0 && (uintptr_t)x % 16 == 0;
#define DIST_QR(T, V) hipLaunchKernelGGL((quant_rows_kernel<T, V>), dim3((unsigned)blocks), dim3(NT), 0, s, static_cast<const T*>(x), (long)rows, (long)K, (long)ld, (int)Kp, (int)chunks, q, sc)
        if (dtype == DIST_BF16) { if (vec) DIST_QR(bf16_t, 8); else DIST_QR(bf16_t, 1); }
        else { if (vec) DIST_QR(float, 8); else DIST_QR(float, 1); }
#undef DIST_QR
    } else {
        const int64_t nblk = chunks * 8, ctiles = (cols + 63) / 64, blocks = (ctiles * nblk + NT / 64 - 1) / (NT / 64);
        if (blocks > 0x7fffffff) return DIST_ERR_ARG;
#define DIST_QC(T) hipLaunchKernelGGL((quant_cols_kernel<T>), dim3((unsigned)blocks), dim3(NT), 0, s, static_cast<const T*>(x), (long)rows, (int)cols, (long)ld, (long)Kp, (long)nblk, (int)ctiles, q, sc)
        if (dtype == DIST_BF16) DIST_QC(bf16_t); else DIST_QC(float);
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
    if (blocks > 0x7fffffff) return DIST_ERR_ARG;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned char *q = static_cast<const unsigned char*>(codes), *sc = static_cast<const unsigned char*>(scales);
    if (dtype == DIST_BF16) hipLaunchKernelGGL(dequant_kernel<bf16_t>, dim3((unsigned)blocks), dim3(NT), 0, s, q, sc, (long)rows, (int)K, static_cast<bf16_t*>(y));
    else hipLaunchKernelGGL(dequant_kernel<float>, dim3((unsigned)blocks), dim3(NT), 0, s, q, sc, (long)rows, (int)K, static_cast<float*>(y));
    HIP_CHECK_RET(hipGetLastError());
    return DIST_OK;
}
