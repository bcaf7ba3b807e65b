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
#include <atomic>
#include <initializer_list>
#include <type_traits>
#include <cooperative_groups.h>

#include "ffn_ops.cuh"
#include "ffn_tcgen05.cuh"

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

// The gate's a and 1 - a from the value in memory.  With e = exp(-g), a = 1 / (1 + e) and 1 - a = e a,
// so neither cancels; e is held below 2^126, where a has long reached 0 and 1 - a one (min.NaN keeps a NaN).
// exp2 and the reciprocal are the hardware's approximations (2 and 1 units in the last place).
template <bool SIG>
__device__ __forceinline__ void gate_of(float g, float& a, float& na) {
    if constexpr (SIG) {
        float x = g * -1.4426950408889634f, e;
        asm("min.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(x));            // 126
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(1.0f + e));
        na = e * a;
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

// C neighbouring channels as they lie in memory; they stay packed in registers until they are used.
template <typename T, int C>
struct Word {
    typename Raw<sizeof(T) * C>::type r;
    __device__ __forceinline__ void load(const T* p) { r = __ldg(reinterpret_cast<const decltype(r)*>(p)); }
    // Copies a word to shared memory without waiting (4 bytes or more).
    static __device__ __forceinline__ void copy(Word* to, const T* p) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;"
                     :: "r"((uint32_t)__cvta_generic_to_shared(to)), "l"(p), "n"((int)sizeof(Word)) : "memory");
    }
    __device__ __forceinline__ float at(int j) const {
        if constexpr (sizeof(T) == 4) {
            if constexpr (C == 1) return __uint_as_float(r);
            else return __uint_as_float(j ? r.y : r.x);
        } else if constexpr (C == 1) {
            return to_f(*reinterpret_cast<const T*>(&r));
        } else {
            uint32_t w;
            if constexpr (C == 2) w = r;
            else w = j < 2 ? r.x : r.y;
            if constexpr (std::is_same<T, __nv_bfloat16>::value)
                return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
            else
                return __half2float(__ushort_as_half((unsigned short)(j & 1 ? w >> 16 : w & 0xffffu)));
        }
    }
};

// U steps of C channels.
template <typename T, bool SIG, bool BACK, int C, int U>
struct Chunk {
    Word<T, C> gate[U], value[SIG || !BACK ? U : 1], dh[BACK ? U : 1], before[BACK ? U : 1];

    // Calls f(stream, step, address) for each word of the chunk that lies before the sequence's end.
    // Streams: 0 gate, 1 value, 2 dh, 3 the state before the step.
    template <typename F>
    static __device__ __forceinline__ void each(const ScanArgs& a, const Span& s, int64_t t0, int ch, F&& f) {
        const int64_t row = s.first + t0 * s.dir;
        const T* pg = static_cast<const T*>(a.gate) + row * a.gate_ld + ch;
        const T* pv = static_cast<const T*>(a.value) + row * a.value_ld + ch;
        const T* pd = static_cast<const T*>(a.dh) + row * a.dh_ld + ch;
        const T* pb = static_cast<const T*>(a.h_in) + (row + s.dir) * a.h_ld + ch;
        const int64_t sg = a.gate_ld * s.dir, sv = a.value_ld * s.dir, sd = a.dh_ld * s.dir, sb = a.h_ld * s.dir;
        const int left = (int)min(max(s.len - t0, (int64_t)0), (int64_t)(U + 1));
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (i < left) {
                f(0, i, pg);
                pg += sg;
                if constexpr (SIG || !BACK) {
                    f(1, i, pv);
                    pv += sv;
                }
                if constexpr (BACK) {
                    f(2, i, pd);
                    pd += sd;
                    // the state before this step: the next row of this walk (the last step's is h0)
                    if (i + 1 < left) f(3, i, pb);
                    pb += sb;
                }
            }
        }
    }
    __device__ __forceinline__ Word<T, C>& word(int stream, int i) {
        return stream == 0 ? gate[i] : stream == 1 ? value[SIG || !BACK ? i : 0] : stream == 2 ? dh[BACK ? i : 0] : before[BACK ? i : 0];
    }
    __device__ __forceinline__ void load(const ScanArgs& a, const Span& s, int64_t t0, int ch) {
        each(a, s, t0, ch, [&](int q, int i, const T* p) { word(q, i).load(p); });
    }
};

// One step of C channels in fp32: the map is m -> a m + b (forward) or m -> a (m + b) (backward, b = dh).
template <bool SIG, bool BACK, int C>
struct Step {
    float a[C], na[SIG && BACK ? C : 1], b[C];

    template <typename T, int U>
    __device__ __forceinline__ void form(const Chunk<T, SIG, BACK, C, U>& k, int i) {
#pragma unroll
        for (int j = 0; j < C; ++j) {
            float n;
            gate_of<SIG>(k.gate[i].at(j), a[j], n);
            if constexpr (BACK) {
                b[j] = k.dh[i].at(j);
                if constexpr (SIG) na[j] = n;
            } else {
                b[j] = SIG ? n * k.value[i].at(j) : k.value[i].at(j);
            }
        }
    }

    // Takes the state through the step and writes its results (element offset `at`); last: the walk's last step.
    template <typename T, int U>
    __device__ __forceinline__ void take(const ScanArgs& p, const Chunk<T, SIG, BACK, C, U>& k, int i, bool last, int64_t at,
                                         int64_t seq_at, float (&state)[C]) const {
        Pack<T, C> o, og;
#pragma unroll
        for (int j = 0; j < C; ++j) {
            if constexpr (!BACK) {
                state[j] = fmaf(a[j], state[j], b[j]);
                o.v[j] = from_f<T>(state[j]);
            } else {
                const float g = b[j] + state[j];
                float hb;
                if (!last) hb = k.before[i].at(j);
                else hb = p.h0 ? __ldg(p.h0 + seq_at + j) : 0.0f;
                if constexpr (SIG) {
                    const float gn = g * na[j];
                    og.v[j] = from_f<T>(gn * a[j] * (hb - k.value[i].at(j)));
                    o.v[j] = from_f<T>(gn);
                } else {
                    og.v[j] = from_f<T>(g * hb);
                    o.v[j] = from_f<T>(g);
                }
                state[j] = a[j] * g;
            }
        }
        if constexpr (!BACK) store_pack<T, C>(static_cast<T*>(p.h) + at, o);
        else {
            store_pack<T, C>(static_cast<T*>(p.dgate) + at, og);
            store_pack<T, C>(static_cast<T*>(p.dvalue) + at, o);
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
__global__ void __launch_bounds__(256, 2) scan_kernel(const ScanArgs a) {
    const int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (item >= a.items) return;
    const int seq = (int)(item / a.groups), ch = (int)(item % a.groups) * C;
    const Span s = span_of<BACK>(a, seq);
    float state[C];
    first_state<BACK, C>(a, seq, ch, state);
#pragma unroll 1
    for (int64_t t = 0; t < s.len; t += U) {
        Chunk<T, SIG, BACK, C, U> k;
        k.load(a, s, t, ch);
        int64_t at = (s.first + t * s.dir) * a.d + ch;
        const int left = (int)min(s.len - t, (int64_t)(U + 1));
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (i < left) {
                Step<SIG, BACK, C> f;
                f.form(k, i);
                f.take(a, k, i, i + 1 == left, at, (int64_t)seq * a.d + ch, state);
                at += (int64_t)s.dir * a.d;
            }
    }
    put_state<C>(a, seq, ch, state);
    clear_outside<T, BACK, C>(a, seq, ch);
}

constexpr int WARPS = 8, MOST_RANKS = 8;

// The maps of a lane's C channels.
template <int C> struct alignas(8 * C) Maps { Affine m[C]; };

// The split form: steps of a warp's part, and the stages of its ring of chunks in shared memory.  Each
// thread copies the words that it will use itself, so the ring needs no barrier; words of 2 bytes, which
// have no asynchronous copy, are prefetched one chunk ahead in registers instead.
template <typename T, bool SIG, bool BACK, int C>
struct Split {
    static constexpr int W = sizeof(T) * C;
    static constexpr bool RING = W >= 4;
    static constexpr int U = !RING ? 8 : (BACK ? 32 : 64) / W;
    static constexpr int STREAMS = BACK ? 4 : 2;
    static constexpr int STAGES = RING ? 3 : 0;
    static constexpr size_t BYTES = (size_t)STAGES * STREAMS * U * W * 32 * WARPS;   // at most 96 KB: two blocks an SM
};

__device__ int g_scan_status;                         // ST_TC_TIMEOUT's bit when a wait ran out (ffn_ops_status)
constexpr uint32_t WAIT_POLLS = 1u << 22;

// Writes a lane's maps into block `rank`'s shared memory and counts their bytes on that block's mbarrier.
template <int C>
__device__ __forceinline__ void send_maps(const Maps<C>* to, uint64_t* bar, int rank, const Maps<C>& v) {
    uint32_t ra, rb;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"((uint32_t)__cvta_generic_to_shared(to)), "r"(rank));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rb) : "r"((uint32_t)__cvta_generic_to_shared(bar)), "r"(rank));
    if constexpr (C == 2)
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
                     :: "r"(ra), "f"(v.m[0].p), "f"(v.m[0].h), "f"(v.m[1].p), "f"(v.m[1].h), "r"(rb) : "memory");
    else
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];"
                     :: "r"(ra), "f"(v.m[0].p), "f"(v.m[0].h), "r"(rb) : "memory");
}

// Few sequences and channels: 32 items per cluster, time split over the WARPS warps of its blocks, U steps
// a warp.  The loads of the next chunks are in flight while the maps of this one go round: a block's map is
// written straight into the shared memory of the cluster's blocks (warp q writes to block q), and each
// block waits on its own mbarrier for the bytes of all.  A cluster barrier in its place costs more than
// the rest of a turn: its release waits until the results that the last turn stored have reached L2.
// Two buffers are enough: a block sends its maps of the next turn after it has read those of this one,
// and nobody sends those of the turn after without having them.
template <typename T, bool SIG, bool BACK, int C>
__global__ void __launch_bounds__(32 * WARPS, 2) scan_split_kernel(const ScanArgs a) {
    using S = Split<T, SIG, BACK, C>;
    constexpr int U = S::U;
    using K = Chunk<T, SIG, BACK, C, U>;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) unsigned char ring_bytes[];
    [[maybe_unused]] Word<T, C>* ring = reinterpret_cast<Word<T, C>*>(ring_bytes) + threadIdx.x;   // [stage][stream][step][thread]
    __shared__ Maps<C> part[2][WARPS][32];            // the maps of this block's parts
    __shared__ Maps<C> whole[2][MOST_RANKS][32];      // the maps of the cluster's blocks
    __shared__ uint64_t arrived[2];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
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
    if (ranks > 1) {
        if (threadIdx.x == 0) { tc::mbar_init(arrived, 1); tc::mbar_init(arrived + 1, 1); }
        cluster.sync();                                // every block runs, its barriers ready, before it is written to
    }
    bool ok = true;                                    // no wait has run out (else the rest of them is left out)
    const int64_t stride = (int64_t)U * WARPS * ranks;
    int64_t t0 = (int64_t)(rank * WARPS + w) * U;
    K next;
    int fill = 0, drain = 0;                           // stages of the ring
    auto fetch = [&](int64_t t) {
        if constexpr (S::RING) {
            K::each(a, s, t, ch, [&](int q, int i, const T* p) {
                Word<T, C>::copy(ring + ((fill * S::STREAMS + q) * U + i) * (32 * WARPS), p);
            });
            asm volatile("cp.async.commit_group;" ::: "memory");
            fill = fill + 1 == S::STAGES ? 0 : fill + 1;
        } else {
            next.load(a, s, t, ch);
        }
    };
    fetch(t0);
    if constexpr (S::RING) fetch(t0 + stride);
    int buf = 0;
    uint32_t phase = 0;
    for (int64_t base = 0; base < most; base += stride, t0 += stride, phase ^= buf, buf ^= 1) {
        K k;
        if constexpr (S::RING) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            fetch(t0 + 2 * stride);                    // into the stage that the last turn has read
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int q = 0; q < S::STREAMS; ++q)
                    if (q != 1 || SIG || !BACK) k.word(q, i) = ring[((drain * S::STREAMS + q) * U + i) * (32 * WARPS)];
            drain = drain + 1 == S::STAGES ? 0 : drain + 1;
        } else {
            k = next;
        }
        Step<SIG, BACK, C> f[BACK ? 1 : U];            // forward: kept for the second walk over the steps
        const int left = (int)min(max(s.len - t0, (int64_t)0), (int64_t)(U + 1));
        Maps<C> mine;
#pragma unroll
        for (int j = 0; j < C; ++j) mine.m[j] = Affine{1.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < U; ++i) {
            Step<SIG, BACK, C>& g = f[BACK ? 0 : i];
            g.form(k, i);
            if (i < left)                              // steps beyond the end leave the state alone
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    Affine& m = mine.m[j];
                    m.p *= g.a[j];
                    m.h = BACK ? g.a[j] * (m.h + g.b[j]) : fmaf(g.a[j], m.h, g.b[j]);
                }
        }
        part[buf][w][lane] = mine;
        __syncthreads();
        // the map of the parts of this block before this warp's, and of all of them
        Maps<C> before, all;
#pragma unroll
        for (int j = 0; j < C; ++j) all.m[j] = before.m[j] = Affine{1.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < WARPS; ++q) {
            const Maps<C> n = part[buf][q][lane];
#pragma unroll
            for (int j = 0; j < C; ++j) {
                if (q == w) before.m[j] = all.m[j];
                all.m[j].h = apply(n.m[j], all.m[j].h);
                all.m[j].p *= n.m[j].p;
            }
        }
        float enter[C];
        if (ranks > 1) {
            if (threadIdx.x == 0)
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                             :: "r"(tc::smem_u32(arrived + buf)), "r"(ranks * 32 * (int)sizeof(Maps<C>)) : "memory");
            if (w < ranks) send_maps<C>(&whole[buf][rank][lane], arrived + buf, w, all);
            if constexpr (!S::RING) if (base + stride < most) fetch(t0 + stride);
            if (ok && !tc::mbar_wait(arrived + buf, phase, WAIT_POLLS)) {
                ok = false;
                atomicOr(&g_scan_status, 4);
            }
#pragma unroll
            for (int j = 0; j < C; ++j) enter[j] = state[j];
#pragma unroll
            for (int q = 0; q < MOST_RANKS; ++q)
                if (q < ranks) {
                    const Maps<C> n = whole[buf][q][lane];
#pragma unroll
                    for (int j = 0; j < C; ++j) {
                        if (q == rank) enter[j] = state[j];
                        state[j] = apply(n.m[j], state[j]);
                    }
                }
        } else {
            if constexpr (!S::RING) if (base + stride < most) fetch(t0 + stride);
#pragma unroll
            for (int j = 0; j < C; ++j) {
                enter[j] = state[j];
                state[j] = apply(all.m[j], state[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < C; ++j) enter[j] = apply(before.m[j], enter[j]);
        int64_t at = (s.first + t0 * s.dir) * a.d + ch;
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (i < left) {
                if constexpr (BACK) f[0].form(k, i);   // formed again: registers are short here
                f[BACK ? 0 : i].take(a, k, i, i + 1 == left, at, (int64_t)seq * a.d + ch, enter);
                at += (int64_t)s.dir * a.d;
            }
    }
    if constexpr (S::RING) asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (live && rank == 0 && w == 0) {
        put_state<C>(a, seq, ch, state);
        clear_outside<T, BACK, C>(a, seq, ch);
    }
    if (ranks > 1) cluster.sync();                     // no block leaves while another writes to it
}

template <typename T, bool SIG, bool BACK, int C>
int scan_launch(ScanArgs a, int64_t longest, int sms, cudaStream_t st) {
    constexpr int U = 8;
    a.groups = a.d / C;
    a.items = (int64_t)a.seqs * a.groups;
    const int64_t warps = (a.items + 31) / 32;
    // parts of time that are wanted for about 16 warps an SM, and that the length has
    constexpr int US = Split<T, SIG, BACK, C < 4 ? C : 2>::U;
    const int64_t parts = (longest + US - 1) / US;
    int64_t want = ((int64_t)sms * 16 + warps - 1) / warps;
    want = want < parts ? want : parts;
    if (want <= 1) {
        const int64_t blocks = (a.items + 255) / 256;
        if (blocks > 0x7fffffff) return op_fail(FFN_E_CAPACITY, "ffn_gated_scan: too many sequences x channels");
        scan_kernel<T, SIG, BACK, C, U><<<(unsigned)blocks, 256, 0, st>>>(a);
        return op_launched("ffn_gated_scan");
    }
    if constexpr (C <= 2) {
        using S = Split<T, SIG, BACK, C>;
        auto kernel = scan_split_kernel<T, SIG, BACK, C>;
        static std::atomic<uint64_t> ready{0};        // devices whose limit is set
        int dev = 0;
        cudaGetDevice(&dev);
        cudaError_t e = cudaSuccess;
        if (S::BYTES > 40960 && (dev > 63 || !(ready.load(std::memory_order_acquire) >> dev & 1))) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::BYTES);
            if (e == cudaSuccess && dev <= 63) ready.fetch_or(1ull << dev, std::memory_order_release);
        }
        int ranks = 1;
        while (ranks < MOST_RANKS && (int64_t)WARPS * ranks < want) ranks *= 2;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(warps * ranks));
        cfg.blockDim = dim3(32 * WARPS);
        cfg.dynamicSmemBytes = S::BYTES;
        cfg.stream = st;
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = (unsigned)ranks;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, a);
        return e == cudaSuccess ? FFN_OK : op_fail(FFN_E_CUDA, std::string("ffn_gated_scan: ") + cudaGetErrorString(e));
    }
    return op_fail(FFN_E_CONFIG, "ffn_gated_scan: no split form for this width");   // scan_width gives C = 4 enough threads
}

// Channels of a thread: as many as an 8-byte access holds, where the rows allow it and enough threads are left.
template <typename T, bool BACK>
int scan_width(const ScanArgs& a, int form, int width, int64_t longest, cudaStream_t st) {
    const int sms = op_sms();
    if (sms <= 0) return op_fail(FFN_E_CUDA, "no CUDA device");
    const bool sig = form == FFN_SCAN_SIGMOID;
    if constexpr (sizeof(T) == 2) {
        if (width == 4 && (int64_t)a.seqs * (a.d / 4) >= (int64_t)sms * 16 * 32)
            return sig ? scan_launch<T, true, BACK, 4>(a, longest, sms, st) : scan_launch<T, false, BACK, 4>(a, longest, sms, st);
    }
    if (width >= 2) return sig ? scan_launch<T, true, BACK, 2>(a, longest, sms, st) : scan_launch<T, false, BACK, 2>(a, longest, sms, st);
    return sig ? scan_launch<T, true, BACK, 1>(a, longest, sms, st) : scan_launch<T, false, BACK, 1>(a, longest, sms, st);
}

template <bool BACK>
int scan_dispatch(const ScanArgs& a, int dtype, int form, int width, int64_t longest, cudaStream_t st) {
    if (dtype == FFN_F32) return scan_width<float, BACK>(a, form, width, longest, st);
    if (dtype == FFN_F16) return scan_width<__half, BACK>(a, form, width, longest, st);
    return scan_width<__nv_bfloat16, BACK>(a, form, width, longest, st);
}

// The widest group of channels that every row of these matrices holds aligned: 4, 2 or 1.
int scan_channels(int d, int dtype, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> lds) {
    const size_t z = dtype == FFN_F32 ? 4 : 2;
    for (int c = 4; c > 1; c /= 2) {
        bool ok = d % c == 0;
        for (const void* p : ptrs) ok = ok && op_aligned(p, c * z);
        for (int64_t ld : lds) ok = ok && ld % c == 0;
        if (ok) return c;
    }
    return 1;
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

// The scan's share of the status word (ffn_ops_status): reads and clears it.
cudaError_t scan_status(int* v) {
    cudaError_t e = cudaMemcpyFromSymbol(v, g_scan_status, sizeof *v);
    const int zero = 0;
    if (e == cudaSuccess && *v) e = cudaMemcpyToSymbol(g_scan_status, &zero, sizeof zero);
    return e;
}

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
    const int width = scan_channels(d, dtype, {gate, value, h}, {gate_ld, value_ld});
    ScanArgs a{};
    a.gate = gate; a.value = value; a.h0 = h0; a.h = h; a.last = h_last; a.offsets = offsets;
    a.gate_ld = gate_ld; a.value_ld = value_ld; a.rows = n_rows; a.len = max_len; a.seqs = n_seq; a.d = d;
    a.reverse = reverse;
    return scan_dispatch<false>(a, dtype, form, width, max_len, static_cast<cudaStream_t>(stream));
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
    const int width = scan_channels(d, dtype, {gate, value, dh, h, dgate, dvalue},
                                    {gate_ld, value ? value_ld : 0, dh_ld, h_ld});
    ScanArgs a{};
    a.gate = gate; a.value = value; a.dh = dh; a.h_in = h; a.h0 = h0; a.dlast = dh_last; a.dgate = dgate; a.dvalue = dvalue;
    a.last = dh0; a.offsets = offsets; a.gate_ld = gate_ld; a.value_ld = value_ld; a.dh_ld = dh_ld; a.h_ld = h_ld;
    a.rows = n_rows; a.len = max_len; a.seqs = n_seq; a.d = d; a.reverse = reverse;
    return scan_dispatch<true>(a, dtype, form, width, max_len, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
