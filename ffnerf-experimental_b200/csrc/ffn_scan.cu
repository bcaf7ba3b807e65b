// ffn_scan.cu -- the gated linear recurrence over packed sequences, forward and backward.
// A translation unit of its own.
//
//   linear:   h_t = a_t h_{t-1} + v_t                                      (gate = a)
//   sigmoid:  a_t = 1 / (1 + exp(-g_t)),  h_t = a_t h_{t-1} + (1 - a_t) v_t  (gate = g)
//
// per channel, h_0 given or zero.  With 1 - a as a sample's opacity and v as its feature vector the
// sigmoid form, run from the last sample to the first, is the compositing of features along a ray.
// Backward, with G_t the gradient that reaches h_t:
//
//   G_t = dh_t + a_{t+1} G_{t+1}  (G_T = dh_T + dlast),   dh_0 = a_1 G_1
//   linear:   da_t = G_t h_{t-1},                      dv_t = G_t
//   sigmoid:  dg_t = G_t (h_{t-1} - v_t) a_t (1 - a_t), dv_t = G_t (1 - a_t)
//
// In M_t = a_t G_t the backward pass is the same kind of recurrence without a shifted gate:
// M_t = a_t M_{t+1} + a_t dh_t, and G_t = dh_t + M_{t+1}.  So both passes run one scheme: an affine map
// (P, H): m -> P m + H per step, composed along time.  All state is fp32.
//
// A thread owns C neighbouring channels of one sequence and walks along time, U steps at a time, whose
// loads are all issued before the first is used.  Threads are numbered over (sequence, channels) so
// that narrow rows fill warps too.  Every element is read and written once: HBM is the bound, and what
// the kernel needs is enough loads in flight.  Where sequences x channels give too few threads for
// that, time is split: a block of W warps takes W parts of U steps each, the blocks of a cluster take
// W parts each, every thread first composes the map of its own part, the maps are exchanged through
// shared memory (within the block) and distributed shared memory (within the cluster), and each thread
// then enters its part with the state that the maps before it give.  The elements stay in registers in
// between, so the split costs no second read; no global memory and no waiting on flags is involved.
#include <cooperative_groups.h>

#include "ffn_ops.cuh"

namespace cg = cooperative_groups;

namespace ffn {
namespace {

struct ScanArgs {
    const void* gate; const void* value; const void* dh; const void* h_in;
    const float* h0; const float* dlast;
    void* h; void* dgate; void* dvalue;
    float* last;                              // forward: final state; backward: gradient of h0
    const int32_t* offsets;
    int64_t gate_ld, value_ld, dh_ld, h_ld, rows;
    int64_t len;                              // steps of every sequence when offsets is NULL
    int64_t items;                            // sequences x channel groups
    int seqs, d, groups;                      // groups = d / C
    int reverse;
};

struct Affine { float p, h; };

// A state that is exactly zero stays out of the product: a composed p may have overflowed (linear gates
// above 1 over many steps), and inf * 0 would turn a sequence of zeros into NaN.
__device__ __forceinline__ float apply(const Affine& m, float x) { return x == 0.0f ? m.h : fmaf(m.p, x, m.h); }

// The gate's a and 1 - a from the value in memory.
template <bool SIG>
__device__ __forceinline__ void gate_of(float g, float& a, float& na) {
    if constexpr (SIG) {
        // 1 / (1 + e) with e = exp(-|g|) never overflows; a and 1 - a are both formed without cancellation
        const float e = __expf(-fabsf(g)), r = __frcp_rn(1.0f + e);
        a = g >= 0.0f ? r : e * r;
        na = g >= 0.0f ? e * r : r;
        if (g != g) { a = g; na = g; }
    } else {
        a = g;
        na = 1.0f;
    }
}

// Where a thread's sequence lies: rows begin .. begin + len - 1, entered at `first`, stepping by `dir`.
struct Span { int64_t first, len; int dir; };

template <bool BACK>
__device__ __forceinline__ Span span_of(const ScanArgs& a, int seq) {
    int64_t b, e;
    if (a.offsets) {
        b = min(max((int64_t)__ldg(a.offsets + seq), (int64_t)0), a.rows);
        e = min(max((int64_t)__ldg(a.offsets + seq + 1), b), a.rows);
    } else {
        b = (int64_t)seq * a.len;
        e = b + a.len;
    }
    const bool from_end = BACK != (a.reverse != 0);
    Span s;
    s.len = e - b;
    s.first = from_end ? e - 1 : b;
    s.dir = from_end ? -1 : 1;
    return s;
}

// U steps of C channels: the packed values in memory, and what the scan needs of them.
template <typename T, bool SIG, bool BACK, int C, int U>
struct Chunk {
    Pack<T, C> gate[U], value[U], dh[BACK ? U : 1], before[BACK ? U : 1];

    __device__ __forceinline__ void load(const ScanArgs& a, const Span& s, int64_t t0, int ch) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (t0 + i < s.len) {
                const int64_t row = s.first + (t0 + i) * s.dir;
                gate[i] = load_pack<T, C>(static_cast<const T*>(a.gate) + row * a.gate_ld + ch);
                if (SIG || !BACK) value[i] = load_pack<T, C>(static_cast<const T*>(a.value) + row * a.value_ld + ch);
                if constexpr (BACK) {
                    dh[i] = load_pack<T, C>(static_cast<const T*>(a.dh) + row * a.dh_ld + ch);
                    // the state before this step: the next row of this walk (the last step's is h0)
                    if (t0 + i + 1 < s.len)
                        before[i] = load_pack<T, C>(static_cast<const T*>(a.h_in) + (row + s.dir) * a.h_ld + ch);
                }
            }
        }
    }

    // The map of step i for channel j (steps beyond the end leave the state alone).
    __device__ __forceinline__ Affine map(int i, int j, bool on) const {
        float al, na;
        gate_of<SIG>(to_f(gate[i].v[j]), al, na);
        Affine m;
        m.p = on ? al : 1.0f;
        if constexpr (BACK) m.h = on ? al * to_f(dh[i].v[j]) : 0.0f;
        else m.h = on ? (SIG ? na * to_f(value[i].v[j]) : to_f(value[i].v[j])) : 0.0f;
        return m;
    }

    // Goes through the steps from `state` and writes the results.
    __device__ __forceinline__ void finish(const ScanArgs& a, const Span& s, int64_t t0, int ch, int seq,
                                           float (&state)[C]) const {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (t0 + i >= s.len) break;
            const int64_t row = s.first + (t0 + i) * s.dir;
            Pack<T, C> o, og;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                float al, na;
                gate_of<SIG>(to_f(gate[i].v[j]), al, na);
                if constexpr (!BACK) {
                    state[j] = fmaf(al, state[j], SIG ? na * to_f(value[i].v[j]) : to_f(value[i].v[j]));
                    o.v[j] = from_f<T>(state[j]);
                } else {
                    const float g = to_f(dh[i].v[j]) + state[j];
                    float hb;
                    if (t0 + i + 1 < s.len) hb = to_f(before[i].v[j]);
                    else hb = a.h0 ? __ldg(a.h0 + (int64_t)seq * a.d + ch + j) : 0.0f;
                    if constexpr (SIG) {
                        og.v[j] = from_f<T>(g * (hb - to_f(value[i].v[j])) * al * na);
                        o.v[j] = from_f<T>(g * na);
                    } else {
                        og.v[j] = from_f<T>(g * hb);
                        o.v[j] = from_f<T>(g);
                    }
                    state[j] = al * g;
                }
            }
            if constexpr (!BACK) store_pack<T, C>(static_cast<T*>(a.h) + row * a.d + ch, o);
            else {
                store_pack<T, C>(static_cast<T*>(a.dgate) + row * a.d + ch, og);
                store_pack<T, C>(static_cast<T*>(a.dvalue) + row * a.d + ch, o);
            }
        }
    }
};

// Rows that belong to no sequence (before the first, after the last) get zeros.
template <typename T, bool BACK, int C>
__device__ __forceinline__ void clear_outside(const ScanArgs& a, int seq, int ch) {
    if (!a.offsets || (seq != 0 && seq != a.seqs - 1)) return;
    const int64_t lo = min(max((int64_t)__ldg(a.offsets), (int64_t)0), a.rows);
    const int64_t hi = min(max((int64_t)__ldg(a.offsets + a.seqs), lo), a.rows);
    const Pack<T, C> z{};
    auto zero = [&](int64_t row) {
        if constexpr (!BACK) store_pack<T, C>(static_cast<T*>(a.h) + row * a.d + ch, z);
        else {
            store_pack<T, C>(static_cast<T*>(a.dgate) + row * a.d + ch, z);
            store_pack<T, C>(static_cast<T*>(a.dvalue) + row * a.d + ch, z);
        }
    };
    if (seq == 0) for (int64_t r = 0; r < lo; ++r) zero(r);
    if (seq == a.seqs - 1) for (int64_t r = hi; r < a.rows; ++r) zero(r);
}

template <bool BACK, int C>
__device__ __forceinline__ void first_state(const ScanArgs& a, int seq, int ch, float (&state)[C]) {
    const float* p = BACK ? a.dlast : a.h0;
#pragma unroll
    for (int j = 0; j < C; ++j) state[j] = p ? p[(int64_t)seq * a.d + ch + j] : 0.0f;   // h0 may be h_last's buffer
}

template <int C>
__device__ __forceinline__ void put_state(const ScanArgs& a, int seq, int ch, const float (&state)[C]) {
    if (!a.last) return;
#pragma unroll
    for (int j = 0; j < C; ++j) a.last[(int64_t)seq * a.d + ch + j] = state[j];
}

// Enough sequences and channels: one thread goes through a whole sequence.
template <typename T, bool SIG, bool BACK, int C, int U>
__global__ void __launch_bounds__(256) scan_kernel(const ScanArgs a) {
    const int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (item >= a.items) return;
    const int seq = (int)(item / a.groups), ch = (int)(item % a.groups) * C;
    const Span s = span_of<BACK>(a, seq);
    float state[C];
    first_state<BACK, C>(a, seq, ch, state);
    for (int64_t t = 0; t < s.len; t += U) {
        Chunk<T, SIG, BACK, C, U> k;
        k.load(a, s, t, ch);
        k.finish(a, s, t, ch, seq, state);
    }
    put_state<C>(a, seq, ch, state);
    clear_outside<T, BACK, C>(a, seq, ch);
}

constexpr int MAX_WARPS = 8;

// Few sequences and channels: 32 items per cluster, time split over the warps of its blocks.
template <typename T, bool SIG, bool BACK, int C, int U>
__global__ void __launch_bounds__(32 * MAX_WARPS) scan_split_kernel(const ScanArgs a) {
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ Affine part[2][MAX_WARPS][C][32];      // the maps of this block's parts
    __shared__ Affine whole[2][C][32];                // their composition, read by the cluster's other blocks
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int64_t item = (int64_t)(blockIdx.x / ranks) * 32 + lane;
    const bool live = item < a.items;
    const int seq = live ? (int)(item / a.groups) : 0, ch = live ? (int)(item % a.groups) * C : 0;
    Span s = span_of<BACK>(a, seq);
    if (!live) s.len = 0;
    int64_t most = s.len;                              // the same in every warp of the cluster
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, (int64_t)__shfl_xor_sync(0xffffffffu, (long long)most, o));
    float state[C];
    first_state<BACK, C>(a, seq, ch, state);
    const int64_t stride = (int64_t)U * warps * ranks;
    int buf = 0;
    for (int64_t base = 0; base < most; base += stride, buf ^= 1) {
        const int64_t t0 = base + (int64_t)(rank * warps + w) * U;
        Chunk<T, SIG, BACK, C, U> k;
        k.load(a, s, t0, ch);
#pragma unroll
        for (int j = 0; j < C; ++j) {
            Affine m{1.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const Affine n = k.map(i, j, t0 + i < s.len);
                m.p *= n.p;
                m.h = fmaf(n.p, m.h, n.h);
            }
            part[buf][w][j][lane] = m;
        }
        __syncthreads();
        // the map of the parts of this block before this warp's, and of all of them
        Affine before[C], all[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            Affine m{1.0f, 0.0f};
            before[j] = m;
            for (int q = 0; q < warps; ++q) {
                if (q == w) before[j] = m;
                const Affine n = part[buf][q][j][lane];
                m.p *= n.p;
                m.h = apply(n, m.h);
            }
            all[j] = m;
        }
        float enter[C];
        if (ranks > 1) {
            if (w == 0)
#pragma unroll
                for (int j = 0; j < C; ++j) whole[buf][j][lane] = all[j];
            cluster.sync();
#pragma unroll
            for (int j = 0; j < C; ++j) {
                float x = state[j];
                enter[j] = x;
                for (int q = 0; q < ranks; ++q) {
                    if (q == rank) enter[j] = x;
                    x = apply(*cluster.map_shared_rank(&whole[buf][j][lane], q), x);
                }
                state[j] = x;
            }
        } else {
#pragma unroll
            for (int j = 0; j < C; ++j) {
                enter[j] = state[j];
                state[j] = apply(all[j], state[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < C; ++j) enter[j] = apply(before[j], enter[j]);
        if (live) k.finish(a, s, t0, ch, seq, enter);
    }
    if (live && rank == 0 && w == 0) {
        put_state<C>(a, seq, ch, state);
        clear_outside<T, BACK, C>(a, seq, ch);
    }
    if (ranks > 1) cluster.sync();                     // no block leaves while another reads its maps
}

template <typename T, bool SIG, bool BACK, int C>
int scan_launch(ScanArgs a, int64_t longest, cudaStream_t st) {
    constexpr int U = 8;
    const int sms = op_sms();
    if (sms <= 0) return op_fail(FFN_E_CUDA, "no CUDA device");
    a.groups = a.d / C;
    a.items = (int64_t)a.seqs * a.groups;
    const int64_t warps = (a.items + 31) / 32;
    // parts of time that are wanted for about 16 warps an SM, and that the length has
    const int64_t parts = (longest + U - 1) / U;
    int64_t want = ((int64_t)sms * 16 + warps - 1) / warps;
    want = want < parts ? want : parts;
    if (want <= 1) {
        const int64_t blocks = (a.items + 255) / 256;
        if (blocks > 0x7fffffff) return op_fail(FFN_E_CAPACITY, "ffn_gated_scan: too many sequences x channels");
        scan_kernel<T, SIG, BACK, C, U><<<(unsigned)blocks, 256, 0, st>>>(a);
        return op_launched("ffn_gated_scan");
    }
    int w = 2, ranks = 1;
    while (w < MAX_WARPS && w < want) w *= 2;
    while (ranks < 8 && (int64_t)w * ranks < want) ranks *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(warps * ranks));
    cfg.blockDim = dim3(32 * w);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)ranks;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, scan_split_kernel<T, SIG, BACK, C, U>, a);
    return e == cudaSuccess ? FFN_OK : op_fail(FFN_E_CUDA, std::string("ffn_gated_scan: ") + cudaGetErrorString(e));
}

template <bool BACK>
int scan_dispatch(const ScanArgs& a, int dtype, int form, bool paired, int64_t longest, cudaStream_t st) {
#define FFN_SCAN(T)                                                                                                     \
    (form == FFN_SCAN_SIGMOID                                                                                           \
         ? (paired ? scan_launch<T, true, BACK, 2>(a, longest, st) : scan_launch<T, true, BACK, 1>(a, longest, st))     \
         : (paired ? scan_launch<T, false, BACK, 2>(a, longest, st) : scan_launch<T, false, BACK, 1>(a, longest, st)))
    if (dtype == FFN_F32) return FFN_SCAN(float);
    if (dtype == FFN_F16) return FFN_SCAN(__half);
    return FFN_SCAN(__nv_bfloat16);
#undef FFN_SCAN
}

int scan_check(const char* who, int64_t n_rows, int32_t n_seq, int64_t max_len, int32_t d, int dtype, int form,
               const int32_t* offsets) {
    auto bad = [&](const char* what) { return op_fail(FFN_E_CONFIG, std::string(who) + ": " + what); };
    if (dtype != FFN_F32 && dtype != FFN_F16 && dtype != FFN_BF16) return bad("dtype must be FFN_F32, FFN_F16 or FFN_BF16");
    if (form != FFN_SCAN_LINEAR && form != FFN_SCAN_SIGMOID) return bad("form must be FFN_SCAN_LINEAR or FFN_SCAN_SIGMOID");
    if (n_rows < 0 || n_seq < 0 || d < 1 || max_len < 0) return bad("sizes must not be negative, d at least 1");
    if (offsets && n_rows > 0x7fffffff) return bad("offsets are 32 bits: at most 2^31 - 1 rows");
    if (!offsets && (int64_t)n_seq * max_len != n_rows) return bad("without offsets n_rows must be n_seq * max_len");
    return FFN_OK;
}

}  // namespace
}  // namespace ffn

using namespace ffn;

extern "C" {

int ffn_gated_scan(const void* gate, int64_t gate_ld, const void* value, int64_t value_ld, const float* h0,
                   const int32_t* offsets, void* h, float* h_last, int64_t n_rows, int32_t n_seq, int64_t max_len,
                   int32_t d, int dtype, int form, int reverse, void* stream) {
    if (int rc = scan_check("ffn_gated_scan", n_rows, n_seq, max_len, d, dtype, form, offsets)) return rc;
    if (n_seq == 0) return FFN_OK;
    if (n_rows > 0 && (!gate || !value || !h)) return op_fail(FFN_E_CONFIG, "ffn_gated_scan: a required pointer is NULL");
    if (gate_ld < d || value_ld < d) return op_fail(FFN_E_CONFIG, "ffn_gated_scan: a row stride is below d");
    const size_t pair = dtype == FFN_F32 ? 8 : 4;
    const bool paired = d % 2 == 0 && gate_ld % 2 == 0 && value_ld % 2 == 0 && op_aligned(gate, pair) &&
                        op_aligned(value, pair) && op_aligned(h, pair);
    ScanArgs a{};
    a.gate = gate; a.value = value; a.h0 = h0; a.h = h; a.last = h_last; a.offsets = offsets;
    a.gate_ld = gate_ld; a.value_ld = value_ld; a.rows = n_rows; a.len = max_len; a.seqs = n_seq; a.d = d;
    a.reverse = reverse;
    return scan_dispatch<false>(a, dtype, form, paired, max_len, static_cast<cudaStream_t>(stream));
}

int ffn_gated_scan_bwd(const void* dh, int64_t dh_ld, const float* dh_last, const void* gate, int64_t gate_ld,
                       const void* value, int64_t value_ld, const void* h, int64_t h_ld, const float* h0,
                       const int32_t* offsets, void* dgate, void* dvalue, float* dh0, int64_t n_rows, int32_t n_seq,
                       int64_t max_len, int32_t d, int dtype, int form, int reverse, void* stream) {
    if (int rc = scan_check("ffn_gated_scan_bwd", n_rows, n_seq, max_len, d, dtype, form, offsets)) return rc;
    if (n_seq == 0) return FFN_OK;
    if (n_rows > 0 && (!dh || !gate || (!value && form == FFN_SCAN_SIGMOID) || !h || !dgate || !dvalue))
        return op_fail(FFN_E_CONFIG, "ffn_gated_scan_bwd: a required pointer is NULL");
    if (gate_ld < d || (value && value_ld < d) || dh_ld < d || h_ld < d)
        return op_fail(FFN_E_CONFIG, "ffn_gated_scan_bwd: a row stride is below d");
    const size_t pair = dtype == FFN_F32 ? 8 : 4;
    const bool paired = d % 2 == 0 && gate_ld % 2 == 0 && (!value || value_ld % 2 == 0) && dh_ld % 2 == 0 && h_ld % 2 == 0 &&
                        op_aligned(gate, pair) && op_aligned(value, pair) && op_aligned(dh, pair) && op_aligned(h, pair) &&
                        op_aligned(dgate, pair) && op_aligned(dvalue, pair);
    ScanArgs a{};
    a.gate = gate; a.value = value; a.dh = dh; a.h_in = h; a.h0 = h0; a.dlast = dh_last; a.dgate = dgate; a.dvalue = dvalue;
    a.last = dh0; a.offsets = offsets; a.gate_ld = gate_ld; a.value_ld = value_ld; a.dh_ld = dh_ld; a.h_ld = h_ld;
    a.rows = n_rows; a.len = max_len; a.seqs = n_seq; a.d = d; a.reverse = reverse;
    return scan_dispatch<true>(a, dtype, form, paired, max_len, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
