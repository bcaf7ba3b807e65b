// ffn_experts.cu -- matrix products of rows grouped by expert, ragged sizes.  A translation unit of its own.
//
// Rows are sorted by expert; expert e has rows offsets[e] .. offsets[e+1] - 1 and weights W_e [m][k]:
//
//   y[r] = x[r] W_e^T        (16-bit operands, or e4m3 with a scale per row and per output channel)
//   dx[r] = dy[r] W_e,       dW_e = sum over the rows of e of dy[r]^T x[r]
//
// Rows after offsets[experts] belong to no expert: their y and dx are zero.
#include "ffn_ops.cuh"

namespace ffn {
namespace {

// An expert's rows, kept inside [0, n] whatever the offsets hold.
__device__ __forceinline__ void expert_rows(const int32_t* off, int e, int64_t n, int64_t& b, int64_t& end) {
    b = e == 0 ? 0 : min(max((int64_t)__ldg(off + e), (int64_t)0), n);
    end = min(max((int64_t)__ldg(off + e + 1), b), n);
}

// C[i][j] = sum_l A[i][l] B[j][l] with any strides, 64 x 64 outputs per block, fp32 throughout.
struct Plain {
    const void* a; const void* b; void* c;
    const float* a_scale; const float* b_scale;
    const int32_t* offsets;
    int64_t n, a_row, a_col, b_row, b_col, b_expert, c_row, c_expert;
    int rows, cols, depth, experts, mode;     // mode 0: rows are ragged, 1: depth is ragged
};

template <typename T, typename TO>
__global__ void __launch_bounds__(256) experts_plain_kernel(const Plain p) {
    __shared__ float sa[16][65], sb[16][65];
    int64_t begin = 0, end = 0;
    int e = 0;
    int64_t i0 = 0;
    if (p.mode == 0) {
        int64_t tile = blockIdx.x;
        for (e = 0; e < p.experts; ++e) {
            expert_rows(p.offsets, e, p.n, begin, end);
            const int64_t tiles = (end - begin + 63) / 64;
            if (tile < tiles) break;
            tile -= tiles;
        }
        if (e == p.experts) {            // rows of no expert
            int64_t b, last;
            expert_rows(p.offsets, p.experts - 1, p.n, b, last);
            for (int64_t r = last + tile * 64; r < min(last + tile * 64 + 64, p.n); ++r)
                for (int j = threadIdx.x + blockIdx.y * 64; j < min((int)blockIdx.y * 64 + 64, p.cols); j += 256)
                    static_cast<TO*>(p.c)[r * p.c_row + j] = from_f<TO>(0.0f);
            return;
        }
        i0 = begin + tile * 64;
    } else {
        e = blockIdx.z;
        expert_rows(p.offsets, e, p.n, begin, end);
        i0 = (int64_t)blockIdx.x * 64;
    }
    const int64_t i_end = p.mode == 0 ? end : p.rows;
    const int64_t l0 = p.mode == 0 ? 0 : begin, l1 = p.mode == 0 ? p.depth : end;
    const int64_t j0 = (int64_t)blockIdx.y * 64;
    const T* A = static_cast<const T*>(p.a);
    const T* B = static_cast<const T*>(p.b) + (int64_t)e * p.b_expert;
    float acc[4][4] = {};
    const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
    for (int64_t l = l0; l < l1; l += 16) {
        for (int q = threadIdx.x; q < 1024; q += 256) {
            const int64_t i = i0 + q / 16, j = j0 + q / 16, ll = l + q % 16;
            sa[q % 16][q / 16] = i < i_end && ll < l1 ? to_f(A[i * p.a_row + ll * p.a_col]) : 0.0f;
            sb[q % 16][q / 16] = j < p.cols && ll < l1 ? to_f(B[j * p.b_row + ll * p.b_col]) : 0.0f;
        }
        __syncthreads();
        for (int s = 0; s < 16; ++s)
            for (int u = 0; u < 4; ++u)
                for (int v = 0; v < 4; ++v) acc[u][v] = fmaf(sa[s][ti + 16 * u], sb[s][tj + 16 * v], acc[u][v]);
        __syncthreads();
    }
    TO* C = static_cast<TO*>(p.c) + (int64_t)e * p.c_expert;
    for (int u = 0; u < 4; ++u)
        for (int v = 0; v < 4; ++v) {
            const int64_t i = i0 + ti + 16 * u, j = j0 + tj + 16 * v;
            if (i >= i_end || j >= p.cols) continue;
            float r = acc[u][v];
            if (p.a_scale) r *= p.a_scale[i] * p.b_scale[(int64_t)e * p.cols + j];
            C[i * p.c_row + j] = from_f<TO>(r);
        }
}

int check(const char* who, int64_t n, int32_t experts, int32_t k, int32_t m) {
    if (n < 0 || n > 0x7fffffff || experts < 1 || experts > FFN_MAX_EXPERTS || k < 1 || m < 1)
        return op_fail(FFN_E_CONFIG, std::string(who) + ": need 0 <= n < 2^31, 1 <= experts <= FFN_MAX_EXPERTS, k >= 1, m >= 1");
    return FFN_OK;
}

}  // namespace
}  // namespace ffn

using namespace ffn;

extern "C" {

int ffn_expert_mm(const void* x, int64_t x_ld, const void* w, const int32_t* offsets, const float* x_scale,
                  const float* w_scale, void* y, int64_t n, int32_t experts, int32_t k, int32_t m, int dtype,
                  int out_dtype, void* workspace, uint64_t workspace_bytes, void* stream) {
    (void)workspace; (void)workspace_bytes;
    if (int rc = check("ffn_expert_mm", n, experts, k, m)) return rc;
    if (dtype == FFN_E4M3 ? (out_dtype != FFN_F16 && out_dtype != FFN_BF16)
                          : ((dtype != FFN_F16 && dtype != FFN_BF16) || out_dtype != dtype))
        return op_fail(FFN_E_CONFIG, "ffn_expert_mm: dtype must be FFN_F16 or FFN_BF16 with out_dtype the same, or FFN_E4M3 "
                                     "with out_dtype FFN_F16 or FFN_BF16");
    if (dtype == FFN_E4M3 && (!x_scale || !w_scale))
        return op_fail(FFN_E_CONFIG, "ffn_expert_mm: FFN_E4M3 operands need x_scale and w_scale");
    if (n == 0) return FFN_OK;
    if (!x || !w || !offsets || !y) return op_fail(FFN_E_CONFIG, "ffn_expert_mm: a required pointer is NULL");
    if (x_ld < k) return op_fail(FFN_E_CONFIG, "ffn_expert_mm: the row stride is below k");
    Plain p{x, w, y, x_scale, w_scale, offsets, n, x_ld, 1, k, 1, (int64_t)m * k, m, 0, 0, m, k, experts, 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((n + 63) / 64 + experts + 1), (unsigned)((m + 63) / 64));
    if (dtype == FFN_F16) experts_plain_kernel<__half, __half><<<grid, 256, 0, st>>>(p);
    else if (dtype == FFN_BF16) experts_plain_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
    else if (out_dtype == FFN_F16) experts_plain_kernel<__nv_fp8_e4m3, __half><<<grid, 256, 0, st>>>(p);
    else experts_plain_kernel<__nv_fp8_e4m3, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
    return op_launched("ffn_expert_mm");
}

uint64_t ffn_expert_mm_workspace(const void*, int64_t, const void*, int64_t, int32_t, int32_t, int32_t, int) { return 0; }

uint64_t ffn_expert_mm_bwd_workspace(const void*, int64_t, const void*, int64_t, const void*, int64_t, int32_t, int32_t,
                                     int32_t, int) { return 0; }

int ffn_expert_mm_bwd(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, const void* w, const int32_t* offsets,
                      void* dx, void* dw, int64_t n, int32_t experts, int32_t k, int32_t m, int dtype, int dw_dtype,
                      void* workspace, uint64_t workspace_bytes, void* stream) {
    (void)workspace; (void)workspace_bytes;
    if (int rc = check("ffn_expert_mm_bwd", n, experts, k, m)) return rc;
    if (dtype != FFN_F16 && dtype != FFN_BF16)
        return op_fail(FFN_E_CONFIG, "ffn_expert_mm_bwd: dtype must be FFN_F16 or FFN_BF16");
    if (dw_dtype != dtype && dw_dtype != FFN_F32)
        return op_fail(FFN_E_CONFIG, "ffn_expert_mm_bwd: dw_dtype must be dtype or FFN_F32");
    if (!dx && !dw) return FFN_OK;
    if (!offsets || (n > 0 && (!dy || !x || !w)))
        return op_fail(FFN_E_CONFIG, "ffn_expert_mm_bwd: a required pointer is NULL");
    if (dy_ld < m || x_ld < k) return op_fail(FFN_E_CONFIG, "ffn_expert_mm_bwd: a row stride is below the columns");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dx && n > 0) {
        Plain p{dy, w, dx, nullptr, nullptr, offsets, n, dy_ld, 1, 1, k, (int64_t)m * k, k, 0, 0, k, m, experts, 0};
        const dim3 grid((unsigned)((n + 63) / 64 + experts + 1), (unsigned)((k + 63) / 64));
        if (dtype == FFN_F16) experts_plain_kernel<__half, __half><<<grid, 256, 0, st>>>(p);
        else experts_plain_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
    }
    if (dw) {
        Plain p{dy, x, dw, nullptr, nullptr, offsets, n, 1, dy_ld, 1, x_ld, 0, k, (int64_t)m * k, m, k, 0, experts, 1};
        const dim3 grid((unsigned)((m + 63) / 64), (unsigned)((k + 63) / 64), (unsigned)experts);
        if (dw_dtype == FFN_F32) {
            if (dtype == FFN_F16) experts_plain_kernel<__half, float><<<grid, 256, 0, st>>>(p);
            else experts_plain_kernel<__nv_bfloat16, float><<<grid, 256, 0, st>>>(p);
        } else if (dtype == FFN_F16) experts_plain_kernel<__half, __half><<<grid, 256, 0, st>>>(p);
        else experts_plain_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
    }
    return op_launched("ffn_expert_mm_bwd");
}

}  // extern "C"
