// Distillation from a teacher's top logits: the k greatest logits of every position (with the logsumexp of all of them), and the
// loss between those and a student's logits with its gradient.
//
// For a position with student logits s over C classes, kept teacher logits t_j at classes i_j and temperature T:
//     q   = softmax(s / T) over all classes
//     p_j = softmax over the kept t_j / T                (no teacher logsumexp given),   r = 0
//     p_j = exp(t_j / T - lse), r = 1 - sum_j p_j        (logsumexp of the teacher given: r is what it gave to the other classes)
//     loss = T^2 [ sum_j p_j (log p_j - log q_{i_j}) + r (log r - log R) ],   R = sum of q over the classes that were not kept
//     d loss / d s_c = T [ M q_c - p_c - [c not kept] r q_c / R ],            M = sum_j p_j + r,  p_c = sum of the p_j with i_j = c
// All sums run over exp2((s - max) log2(e) / T) in fp32, the difference first: a mask of the type's lowest value times log2(e) would
// overflow.  The classes outside the kept ones have a maximum and a sum of their own
// (K_out, S_out): R and q_c / R then never come out of a difference of two almost equal sums, and cannot underflow.
//
// The loss is summed as  sum D(P_c, q_c) + D(r, R),  D(p, q) = p log(p / q) - p + q,  over the kept classes: the probabilities on either
// side sum to 1, so what D adds cancels.  D has no negative value and is taken from q - p where the two are alike.  The terms
// p log(p / q) themselves are of the order 1 / T and cancel to 1 / T^2 at high temperatures (1000 classes, 8 kept, worst of 64 rows:
// 3e-3 of the loss lost at T = 20, 0.8 at T = 256).
#include "common.h"

namespace segk {

constexpr int kTopMax = 64;               // kept logits of a position: one lane each
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A rest 1 - sum p of up to 2^-20 is rounding of at most 64 fp32 terms and of the logsumexp, not mass: it counts as none.
constexpr float kRestFloor = 0x1p-20f;
constexpr int kCountBlocks = 256;         // partial counts that the main kernels add up

struct DistillArgs {
    const void* z;             // student logits
    int64_t ld;                // elements from one row / image to the next
    int64_t s_c, s_p;          // elements from class to class and from position to position (thread-per-position kernel)
    int64_t inner;             // positions of an image
    int V;                     // classes
    int k;
    const void* t;             // kept teacher logits
    const void* idx;           // their classes
    const float* tlse;         // the teacher's logsumexp, or none
    int64_t ts_c, ts_p;        // strides of t and idx
    int t_bf16, idx64;
    float T, invT, weight;
    const float* upstream;     // gradient that reaches the loss: none (1), one value, or one for each position
    int up_each, skip_if_one;
    int* counts;               // partial counts of the positions with a kept logit (mean), or none (sum)
    int count_here, log_kp;    // few rows: so many rows are counted by whoever needs the number (0: counts hold it)
    int count_losses;          // no gradient waits for the number: the row losses that are not -0 are counted with their final sum
                               // (1: by the finalize kernel, 2: by the collect kernel into counts)
    float* row_loss;           // loss of each position
    float* partial;            // sums that the finalize kernel adds (thread-per-position kernel)
    void* dz;
    int64_t ld_d, d_c, d_p;
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Reductions over a wave with data moved between lanes by the ALU (DPP): six dependent instructions, where shuffles through LDS
// take several hundred cycles.  The result is the same in every lane.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t lanes(uint32_t other, uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)other, (int)v, CTRL, ROWS, 0xF, false);
}
template <typename V, typename F> __device__ __forceinline__ V wave_all(V v, V nothing, F&& f) {
    const uint32_t none = __builtin_bit_cast(uint32_t, nothing);
    auto step = [&](uint32_t moved) { v = f(v, __builtin_bit_cast(V, moved)); };
    step(lanes<0x111, 0xF>(none, __builtin_bit_cast(uint32_t, v)));       // from 1, 2, 4, 8 lanes below, within 16
    step(lanes<0x112, 0xF>(none, __builtin_bit_cast(uint32_t, v)));
    step(lanes<0x114, 0xF>(none, __builtin_bit_cast(uint32_t, v)));
    step(lanes<0x118, 0xF>(none, __builtin_bit_cast(uint32_t, v)));
    step(lanes<0x142, 0xA>(none, __builtin_bit_cast(uint32_t, v)));       // lane 15 into the next 16, lane 31 into the upper half
    step(lanes<0x143, 0xC>(none, __builtin_bit_cast(uint32_t, v)));
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float wave_max(float v) { return wave_all(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float sum_wave(float v) { return wave_all(v, 0.f, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ int wave_sum_i(int v) { return wave_all(v, 0, [](int a, int b) { return a + b; }); }

// the class of a kept logit; -1 where it is none of [0, V): such an entry does not exist
__device__ __forceinline__ int load_class(const DistillArgs& a, int64_t at) {
    const int64_t i = a.idx64 ? static_cast<const int64_t*>(a.idx)[at] : (int64_t) static_cast<const int32_t*>(a.idx)[at];
    return i >= 0 && i < a.V ? (int)i : -1;
}
// the same with the type known: a branch on it between two loads would make the second wait for the first
template <typename I> __device__ __forceinline__ int load_class_as(const DistillArgs& a, int64_t at) {
    const I i = static_cast<const I*>(a.idx)[at];
    return i >= 0 && i < a.V ? (int)i : -1;
}
// loss of a row; -0 says that it has no entry, where the final sum counts them, and no other row has that value
__device__ __forceinline__ float loss_of_empty(const DistillArgs& a) { return a.count_losses ? -0.f : 0.f; }
__device__ __forceinline__ float loss_of_row(const DistillArgs& a, float l) {
    l *= a.T * a.T * a.weight;
    return l == 0.f ? 0.f : l;
}
__device__ __forceinline__ float load_kept(const DistillArgs& a, int64_t at) {
    return a.t_bf16 ? (float)static_cast<const bf16*>(a.t)[at] : static_cast<const float*>(a.t)[at];
}
// Rows (of k contiguous entries) with at least one kept logit among every `step`-th group of 64 / kp rows from `first` on, for a
// whole wave, four groups in flight
template <typename I> __device__ __forceinline__ int count_rows_as(const DistillArgs& a, int64_t rows, int log_kp, int64_t first, int64_t step, int lane) {
    const int per = 64 >> log_kp, j = lane & ((1 << log_kp) - 1);
    const int64_t groups = (rows + per - 1) / per;
    int n = 0;
    for (int64_t g = first; g < groups; g += 4 * step) {
        bool have[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t row = (g + u * step) * per + (lane >> log_kp);
            have[u] = load_class_as<I>(a, (row < rows ? row : 0) * a.k + (j < a.k ? j : 0)) >= 0 && j < a.k && row < rows;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            uint64_t m = __ballot(have[u]);
            for (int d = 1; d < (1 << log_kp); d *= 2) m |= m >> d;         // any entry of a row into the bit of its first
            n += j == 0 && ((m >> lane) & 1ull);
        }
    }
    return wave_sum_i(n);
}

__device__ __forceinline__ int count_rows(const DistillArgs& a, int64_t rows, int log_kp, int64_t first, int64_t step, int lane) {
    return a.idx64 ? count_rows_as<int64_t>(a, rows, log_kp, first, step, lane) : count_rows_as<int32_t>(a, rows, log_kp, first, step, lane);
}

// the number of positions with a kept logit, at least 1; every lane of the wave has to call it
__device__ __forceinline__ int count_of(const DistillArgs& a) {
    int n = 0;
    if (a.count_here) {
        n = count_rows(a, a.count_here, a.log_kp, 0, 1, threadIdx.x & 63);
    } else {
#pragma unroll
        for (int i = 0; i < kCountBlocks / 64; ++i) n += a.counts[i * 64 + (threadIdx.x & 63)];
        n = wave_sum_i(n);
    }
    return n > 0 ? n : 1;
}
// the same for VP neighbouring positions: 16-byte loads for four of them
template <int VP> __device__ __forceinline__ void load_classes(const DistillArgs& a, int64_t at, int (&c)[VP]) {
    if constexpr (VP == 4) {
        if (a.idx64) {
            typedef int64_t i64x2 __attribute__((ext_vector_type(2)));
            const i64x2 lo = *reinterpret_cast<const i64x2*>(static_cast<const int64_t*>(a.idx) + at), hi = *reinterpret_cast<const i64x2*>(static_cast<const int64_t*>(a.idx) + at + 2);
            const int64_t i[4] = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
            for (int v = 0; v < 4; ++v) c[v] = i[v] >= 0 && i[v] < a.V ? (int)i[v] : -1;
        } else {
            const int4 i = *reinterpret_cast<const int4*>(static_cast<const int32_t*>(a.idx) + at);
            c[0] = i.x; c[1] = i.y; c[2] = i.z; c[3] = i.w;
#pragma unroll
            for (int v = 0; v < 4; ++v) c[v] = c[v] >= 0 && c[v] < a.V ? c[v] : -1;
        }
    } else {
        c[0] = load_class(a, at);
    }
}
template <int VP> __device__ __forceinline__ void load_kepts(const DistillArgs& a, int64_t at, float (&t)[VP]) {
    if constexpr (VP == 4) {
        if (a.t_bf16) Elem<bf16>::load4(static_cast<const bf16*>(a.t) + at, t);
        else Elem<float>::load4(static_cast<const float*>(a.t) + at, t);
    } else {
        t[0] = load_kept(a, at);
    }
}
// what multiplies T * (M q - p ...) of a position; every lane of the wave has to call it
__device__ __forceinline__ float grad_scale(const DistillArgs& a, int64_t position) {
    float g = a.weight * a.T;
    if (a.counts) g /= (float)count_of(a);
    if (a.upstream) g *= a.upstream[a.up_each ? position : 0];
    return g;
}
// exp of a logit over a base; c = log2(e) / T
__device__ __forceinline__ float exp_over(float z, float base, float c) { return fast_exp2((z - base) * c); }
// the same for a maximum that may be "no element" (-inf), whatever the base
__device__ __forceinline__ float rebase(float k, float base, float c) { return k == -INFINITY ? 0.f : exp_over(k, base, c); }

// p ln(p / q) - p + q = p (y - 1 - ln y), y = q / p; log_ratio(): the logarithm (base 2) of p / q, used where y leaves the range.  Near 1, y - 1
// is exact and the logarithm good to one unit of its own last place (all y in [1/2, 2]), so y - 1 - ln y is off by at most 2^-22 |y - 1|, as if y were
// off by 2^-22; what that leaves below 0 is 0.
template <typename F> __device__ __forceinline__ float divergence(float p, float q, F&& log_ratio) {
    const float y = q * __builtin_amdgcn_rcpf(p);
    if (y > 0x1p-100f && y < 0x1p100f) {
        const float h = fmaf(-kLn2, __builtin_amdgcn_logf(y), y - 1.f);
        return p * (h < 0.f ? 0.f : h);
    }
    return p == 0.f ? q : (q - p) + p * (log_ratio() * kLn2);
}
// What an entry adds to its row's loss.  p, lp: its own probability and logarithm; total: that of all entries with its class, for which
// the first of them stands.
__device__ __forceinline__ float entry_loss(bool first, float p, float lp, float total, float q, float lq) {
    float l = first ? divergence(total, q, [&] { return (total == p ? lp : log2f(total)) - lq; }) : 0.f;
    if (total != p && p != 0.f) l += p * ((lp - log2f(total)) * kLn2);
    return l;
}
// The same for everything outside the kept classes (R: the student's probability there, lr its logarithm).  Where the teacher has no rest
// there, what D added does not cancel: mass - 1 + R is left (a row whose entries have no probability at all counts as 0).
__device__ __forceinline__ float rest_loss(const DistillArgs& a, float l, float rest, float mass, float R, float lr) {
    if (rest > 0.f) return l + divergence(rest, R, [&] { return log2f(rest) - lr; });
    return mass == 0.f ? 0.f : l + (a.tlse ? mass - 1.f : 0.f) + R;
}

// ------------------------------------------------------------------------------------------------ rows in registers
// A row is read in 16-byte pieces that are aligned in memory; the row may begin and end inside a piece.
template <typename T> struct Piece {
    static constexpr int VEC = 16 / (int)sizeof(T);
    uint32_t w[4];
    __device__ __forceinline__ float get(int v) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[v]);
        else return __uint_as_float((v & 1) ? (w[v >> 1] & 0xFFFF0000u) : (w[v >> 1] << 16));
    }
    __device__ __forceinline__ void clear(int v) {      // element v <- -inf
        if constexpr (sizeof(T) == 4) w[v] = 0xFF800000u;
        else w[v >> 1] = (v & 1) ? ((w[v >> 1] & 0x0000FFFFu) | 0xFF800000u) : ((w[v >> 1] & 0xFFFF0000u) | 0x0000FF80u);
    }
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Between two passes over packed pieces: makes the compiler unpack them again instead of keeping every element as a float of its
// own from the first pass on (twice the registers, and spills in the tiers with 16 pieces).
template <typename T, int N> __device__ __forceinline__ void stay_packed(Piece<T> (&x)[N]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) asm volatile("" : "+v"(x[i].w[w]));
    }
}

// The greatest element of a lane's pieces.  Pairs of bf16 are compared as 16-bit integers, which order positive floats as the floats
// do and put all negative ones below them; a lane that has no positive element looks again, as floats.  (A quarter of the
// instructions; 4096 rows of 32000, selection: 61.3 -> 60.0 us.)
template <typename T, int N> __device__ __forceinline__ float lane_max(const Piece<T> (&x)[N]) {
    float m = -INFINITY;
    if constexpr (sizeof(T) == 2) {
        typedef short s16x2 __attribute__((ext_vector_type(2)));
        s16x2 best = {-32768, -32768};
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) best = __builtin_elementwise_max(best, __builtin_bit_cast(s16x2, x[i].w[w]));
        const int top = best[0] > best[1] ? best[0] : best[1];
        if (top >= 0) return __uint_as_float((uint32_t)top << 16);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < Piece<T>::VEC; ++v) m = fmaxf(m, x[i].get(v));
    return m;
}
// whether a piece may have an element of at least `bound` (certain for fp32; never a miss)
template <typename T> __device__ __forceinline__ bool may_reach(const Piece<T>& x, float bound) {
    if constexpr (sizeof(T) == 2) {
        if (bound > 0.f) {
            typedef short s16x2 __attribute__((ext_vector_type(2)));
            const short b = (short)(__float_as_uint(bound) >> 16);
            s16x2 best = __builtin_bit_cast(s16x2, x.w[0]);
#pragma unroll
            for (int w = 1; w < 4; ++w) best = __builtin_elementwise_max(best, __builtin_bit_cast(s16x2, x.w[w]));
            return best[0] >= b || best[1] >= b;
        }
        return true;
    } else {
        return fmaxf(fmaxf(x.get(0), x.get(1)), fmaxf(x.get(2), x.get(3))) >= bound;
    }
}

template <typename T> struct Row {
    const T* p;      // element 0
    int phase, V, pieces;
    __device__ __forceinline__ Row(const T* row, int V_) : p(row), V(V_) {
        constexpr int VEC = Piece<T>::VEC;
        phase = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % VEC);
        pieces = (int)(((int64_t)V + phase + VEC - 1) / VEC);
    }
    // piece g: elements [g*VEC - phase, +VEC); what lies outside the row reads as -inf
    __device__ __forceinline__ Piece<T> load(int g) const {
        constexpr int VEC = Piece<T>::VEC;
        Piece<T> r;
        const int e0 = g * VEC - phase;
        if (e0 >= 0 && e0 <= V - VEC) {
            const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + e0));
#pragma unroll
            for (int i = 0; i < 4; ++i) r.w[i] = x[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) r.w[i] = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int e = e0 + v;
                if (e >= 0 && e < V) {
                    if constexpr (sizeof(T) == 4) r.w[v] = reinterpret_cast<const uint32_t*>(p)[e];
                    else {
                        const uint32_t h = reinterpret_cast<const uint16_t*>(p)[e];
                        r.w[v >> 1] = (v & 1) ? ((r.w[v >> 1] & 0x0000FFFFu) | (h << 16)) : ((r.w[v >> 1] & 0xFFFF0000u) | h);
                    }
                }
            }
        }
        return r;
    }
};

template <typename T>
__device__ __forceinline__ void store_piece(T* dst, bool vec_ok, int e0, int V, const float (&f)[Piece<T>::VEC]) {
    constexpr int VEC = Piece<T>::VEC;
    if (vec_ok && e0 >= 0 && e0 <= V - VEC) {
        if constexpr (sizeof(T) == 4) {
            __builtin_nontemporal_store(f32x4{f[0], f[1], f[2], f[3]}, reinterpret_cast<f32x4*>(dst + e0));
        } else {
            bf16x8 o;
#pragma unroll
            for (int v = 0; v < 8; ++v) o[v] = (bf16)f[v];
            __builtin_nontemporal_store(o, reinterpret_cast<bf16x8*>(dst + e0));
        }
    } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            if (e0 + v >= 0 && e0 + v < V) dst[e0 + v] = Elem<T>::from_f(f[v]);
    }
}

// Kept classes that lie in the 64 pieces from g0 on (one for each lane): f(lane has it, element in the piece, entry)
template <int VEC, typename F>
__device__ __forceinline__ void for_kept(int cls, int phase, int g0, int lane, F&& f) {
    const int rel = cls + phase - g0 * VEC;
    uint64_t in = __ballot(cls >= 0 && rel >= 0 && rel < 64 * VEC);
    while (in) {
        const int j = __builtin_ctzll(in);
        in &= in - 1;
        const int at = __builtin_amdgcn_readlane(rel, j);
        f(lane == at / VEC, at % VEC, j);
    }
}

// between accesses of one wave to LDS, which serves it in order: only the compiler has to keep it
__device__ __forceinline__ void one_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The kept entries of a row, one for each lane of a wave (cls: this lane's class or -1).
struct Kept {
    float p, lp, z;          // probability, its logarithm (base 2), the student's logit
    float total;             // p of all entries with this class
    float rest, mass;        // of the row: what the teacher gave to the other classes; sum of p and rest
    float top, sum;          // of the row: the student's maximum over the kept classes and the sum of exp over it
    bool first;              // the first entry with this class
};
template <typename T>
__device__ __forceinline__ Kept kept_entries(const DistillArgs& a, int64_t row, const T* __restrict__ z, int cls, int lane, float c) {
    Kept e;
    e.p = 0.f;
    e.lp = e.z = -INFINITY;
    float t = -INFINITY;
    if (cls >= 0) {
        t = load_kept(a, row * a.k + lane);
        e.z = Elem<T>::to_f(z[cls]);
    }
    if (a.tlse) {
        e.lp = cls >= 0 ? fmaf(t, a.invT, -a.tlse[row]) * kLog2e : -INFINITY;
        e.p = cls >= 0 ? fast_exp2(e.lp) : 0.f;
    } else {
        const float top = wave_max(t);
        const float x = t == -INFINITY ? 0.f : fast_exp2((t - top) * c);      // NaN stays, also where nothing else was kept
        const float sum = sum_wave(x);
        e.p = sum == 0.f ? 0.f : x / sum;
        e.lp = (t - top) * c - log2f(sum);
    }
    const float mass = sum_wave(e.p);
    e.total = e.p;
    // Entries of one class: the first of them stands for it, each carries their sum.  Comparing all with all is a loop over k; of more
    // than 8 only those are compared that lose their place in a table of 256 to a higher lane, as every repeated entry does but one,
    // whose share the others get from the winner of their place.  (Joining rows with 64 entries:
    // 8 -> 5 us.)
    bool first = cls >= 0;
    uint64_t compare = a.k == 64 ? ~0ull : (1ull << a.k) - 1;
    if (a.k > 8) {
        __shared__ int winner[256];
#pragma unroll
        for (int i = 0; i < 4; ++i) winner[i * 64 + lane] = -1;
        one_wave_sync();
        if (cls >= 0) atomicMax(&winner[cls & 255], lane);
        one_wave_sync();
        const int w = cls >= 0 ? winner[cls & 255] : lane;
        compare = __ballot(w != lane);
        if (compare) {
            const int cw = __shfl(cls, w, 64);
            const float pw = __shfl(e.p, w, 64);
            if (w != lane && cw == cls) e.total += pw;
        }
    }
    while (compare) {
        const int j = __builtin_ctzll(compare);
        compare &= compare - 1;
        const int cj = __builtin_amdgcn_readlane(cls, j);
        const float pj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e.p), j));
        if (cj == cls && j != lane) {
            e.total += pj;
            if (j < lane) first = false;
        }
    }
    e.first = first;
    const int distinct = __popcll(__ballot(first));
    e.rest = a.tlse ? 1.f - mass : 0.f;
    if (!(e.rest > kRestFloor) || distinct == a.V) e.rest = 0.f;
    e.mass = mass + e.rest;
    e.top = wave_max(first ? e.z : -INFINITY);
    // no maximum: -inf, whose exp is 0, or NaN, which has to reach the row
    e.sum = sum_wave(!first ? 0.f : e.top != -INFINITY ? exp_over(e.z, e.top, c) : e.z != e.z ? e.z : 0.f);
    return e;
}
// maximum and sum of exp over all classes, from those outside (ko, so) and those kept; share: exp of ko over the maximum
struct Joined { float top, sum, share; };
__device__ __forceinline__ Joined join(float ko, float so, float km, float sm, float c) {
    Joined w;
    w.top = fmaxf(ko, km);
    w.share = rebase(ko, w.top, c);
    w.sum = so * w.share + sm * rebase(km, w.top, c) + (so != so ? so : 0.f);      // a NaN among the logits reaches the row
    return w;
}
// the row's loss in units of T^2, for a whole wave
__device__ __forceinline__ float kept_loss(const DistillArgs& a, const Kept& e, const Joined& w, float ko, float so, float c) {
    const float ls = log2f(w.sum), inv = __builtin_amdgcn_rcpf(w.sum), q = exp_over(e.z, w.top, c) * inv;
    const float l = sum_wave(entry_loss(e.first, e.p, e.lp, e.total, q, (e.z - w.top) * c - ls));
    return rest_loss(a, l, e.rest, e.mass, so * w.share * inv, log2f(so) + (ko - w.top) * c - ls);
}
// the gradient of a class outside is this times exp of its logit over ko
__device__ __forceinline__ float outside_factor(const Joined& w, float so, float rest, float mass, float gs) {
    return gs * (mass * w.share / w.sum - (rest > 0.f ? rest / so : 0.f));
}

// One workgroup per row; with NCH > 0 the row stays in registers (NCH pieces per thread), with NCH == 0 it is read twice.
// In registers the forward pass and the gradient cost one read and one write of the logits, and memory bounds it: 4096 rows of 32000
// bf16 logits, 32 kept, a tenth of the rows without: 509 MB in 98 us, 5.2 TB/s (a copy of that size: 5.4).  The first wave handles the kept entries, one for
// each lane, while the others wait for their pieces; their classes are taken out of the registers, so the two groups of classes have
// separate maxima without a second pass.
template <typename T, int NT, int NCH, bool GRAD>
__global__ __launch_bounds__(NT) void distill_rows_kernel(const DistillArgs a) {
    constexpr int VEC = Piece<T>::VEC, NW = NT / 64;
    __shared__ float sh_k[NW], sh_s[NW], sh_p[kTopMax], sh_z[kTopMax], sh_x[6];
    if (a.skip_if_one && a.upstream[0] == 1.f) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x;
    const float c = a.invT * kLog2e;
    const Row<T> r(static_cast<const T*>(a.z) + row * a.ld, a.V);
    T* dst = GRAD ? static_cast<T*>(a.dz) + row * a.ld_d : nullptr;
    const bool vec_ok = GRAD && (reinterpret_cast<uintptr_t>(dst) / sizeof(T)) % VEC == (unsigned)r.phase;

    const int cls = lane < a.k ? load_class(a, row * a.k + lane) : -1;
    if (__ballot(cls >= 0) == 0) {                       // nothing was kept here: no loss, no gradient, the row is not read
        if (threadIdx.x == 0) a.row_loss[row] = loss_of_empty(a);
        if constexpr (GRAD) {
            const float zero[VEC] = {};
            for (int g = threadIdx.x; g < r.pieces; g += NT) store_piece<T>(dst, vec_ok, g * VEC - r.phase, a.V, zero);
        }
        return;
    }

    Piece<T> x[NCH > 0 ? NCH : 1];
    if constexpr (NCH > 0) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int g = i * NT + (int)threadIdx.x;
            if (g < r.pieces) x[i] = r.load(g);
            else
#pragma unroll
                for (int w = 0; w < 4; ++w) x[i].w[w] = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
        }
    }

    // ---- the kept entries, one for each lane of the first wave
    Kept e = {};
    if (wave == 0) {
        e = kept_entries<T>(a, row, r.p, cls, lane, c);
        const float gs = GRAD ? grad_scale(a, row) : 0.f;
        sh_p[lane] = e.total;
        sh_z[lane] = e.z;
        if (lane == 0) { sh_x[0] = e.top; sh_x[1] = e.sum; sh_x[2] = e.rest; sh_x[3] = e.mass; sh_x[4] = gs; }
    }

    // ---- maximum and sum of the classes that were not kept
    float kw = -INFINITY, sw = 0.f;
    if constexpr (NCH > 0) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
            for_kept<VEC>(cls, r.phase, i * NT + wave * 64, lane, [&](bool here, int v, int) {
#pragma unroll
                for (int u = 0; u < VEC; ++u)
                    if (here && u == v) x[i].clear(u);
            });
        const float m = wave_max(lane_max<T, NCH>(x));
        const float base = m == -INFINITY ? 0.f : m;
        stay_packed(x);
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) sw += exp_over(x[i].get(v), base, c);
        sw = sum_wave(sw);
        kw = m;
    } else {
        float m = -INFINITY;                              // of this lane
        for (int g0 = wave * 64; g0 < r.pieces; g0 += NT) {
            const int g = g0 + lane;
            Piece<T> y;
#pragma unroll
            for (int w = 0; w < 4; ++w) y.w[w] = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
            if (g < r.pieces) y = r.load(g);
            for_kept<VEC>(cls, r.phase, g0, lane, [&](bool here, int v, int) {
#pragma unroll
                for (int u = 0; u < VEC; ++u)
                    if (here && u == v) y.clear(u);
            });
            float mg = y.get(0);
#pragma unroll
            for (int v = 1; v < VEC; ++v) mg = fmaxf(mg, y.get(v));
            if (mg > m) {
                sw *= rebase(m, mg, c);
                m = mg;
            }
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int v = 0; v < VEC; ++v) sw += exp_over(y.get(v), base, c);
        }
        kw = wave_max(m);
        sw = sum_wave(m == -INFINITY ? sw : sw * exp_over(m, kw, c));      // sw of an empty lane is 0 (or NaN, which stays)
    }
    if (lane == 0) { sh_k[wave] = kw; sh_s[wave] = sw; }
    __syncthreads();

    float ko = sh_k[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) ko = fmaxf(ko, sh_k[w]);
    float so = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) so += sh_k[w] == -INFINITY ? sh_s[w] : sh_s[w] * exp_over(sh_k[w], ko, c);
    const Joined w = join(ko, so, sh_x[0], sh_x[1], c);
    if (wave == 0) {
        const float l = kept_loss(a, e, w, ko, so, c);
        if (lane == 0) a.row_loss[row] = loss_of_row(a, l);
    }
    if constexpr (GRAD) {
        const float gs = sh_x[4];
        const float gj = lane < a.k ? gs * (sh_x[3] * exp_over(sh_z[lane], w.top, c) / w.sum - sh_p[lane]) : 0.f;
        const float b = outside_factor(w, so, sh_x[2], sh_x[3], gs);
        const float base = ko == -INFINITY ? 0.f : ko;
        auto write = [&](const Piece<T>& y, int g0) {
            float f[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) f[v] = b * exp_over(y.get(v), base, c);
            for_kept<VEC>(cls, r.phase, g0, lane, [&](bool here, int v, int j) {
                const float gv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(gj), j));
#pragma unroll
                for (int u = 0; u < VEC; ++u)
                    if (here && u == v) f[u] = gv;
            });
            const int g = g0 + lane;
            if (g < r.pieces) store_piece<T>(dst, vec_ok, g * VEC - r.phase, a.V, f);
        };
        if constexpr (NCH > 0) {
            stay_packed(x);
#pragma unroll
            for (int i = 0; i < NCH; ++i) write(x[i], i * NT + wave * 64);
        } else {
            for (int g0 = wave * 64; g0 < r.pieces; g0 += NT) {
                Piece<T> y;
#pragma unroll
                for (int w = 0; w < 4; ++w) y.w[w] = 0;
                if (g0 + lane < r.pieces) y = r.load(g0 + lane);
                write(y, g0);
            }
        }
    }
}

// Few long rows: a row is shared by S workgroups.  Maximum and sum of the classes outside, one pair for each share; one wave per row
// joins them (loss, and what the gradient needs); the gradient of each share.
constexpr int kShares = 64;
constexpr int kRowFloats = 2 + kTopMax;      // of a joined row: maximum outside, factor outside, gradients of the kept entries

template <typename T> struct Share {         // the pieces [lo, hi) of a row, whole groups of 64
    int lo, hi;
    __device__ __forceinline__ Share(const Row<T>& r) {
        const int groups = (r.pieces + 63) / 64, per = (groups + gridDim.x - 1) / gridDim.x;
        lo = (int)blockIdx.x * per * 64;
        hi = lo + per * 64 < r.pieces ? lo + per * 64 : r.pieces;
    }
};

template <typename T>
__global__ __launch_bounds__(256) void distill_share_kernel(const DistillArgs a, float* __restrict__ parts, int* __restrict__ rows_done) {
    constexpr int VEC = Piece<T>::VEC, U = 4;
    if (a.skip_if_one && a.upstream[0] == 1.f) return;
    if (rows_done && (blockIdx.x | blockIdx.y | threadIdx.x) == 0) *rows_done = 0;
    __shared__ float sh_k[4], sh_s[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.y;
    const float c = a.invT * kLog2e;
    const Row<T> r(static_cast<const T*>(a.z) + row * a.ld, a.V);
    const Share<T> part(r);
    const int cls = lane < a.k ? load_class(a, row * a.k + lane) : -1;
    if (__ballot(cls >= 0) == 0) return;
    float m = -INFINITY, s = 0.f;                        // of this lane
    for (int g0 = part.lo + wave * 64; g0 < part.hi; g0 += 256 * U) {
        Piece<T> y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int g = g0 + u * 256 + lane;
            if (g < part.hi) y[u] = r.load(g);
            else
#pragma unroll
                for (int w = 0; w < 4; ++w) y[u].w[w] = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            for_kept<VEC>(cls, r.phase, g0 + u * 256, lane, [&](bool here, int v, int) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (here && i == v) y[u].clear(i);
            });
#pragma unroll
            for (int v = 0; v < VEC; ++v) top = fmaxf(top, y[u].get(v));
        }
        s *= rebase(m, top, c);
        m = top;
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int v = 0; v < VEC; ++v) s += exp_over(y[u].get(v), base, c);
    }
    const float k = wave_max(m);
    s = sum_wave(m == -INFINITY ? s : s * exp_over(m, k, c));
    if (lane == 0) { sh_k[wave] = k; sh_s[wave] = s; }
    __syncthreads();
    if (threadIdx.x == 0) {
        const float ko = fmaxf(fmaxf(sh_k[0], sh_k[1]), fmaxf(sh_k[2], sh_k[3]));
        float so = 0.f;
        for (int w = 0; w < 4; ++w) so += sh_k[w] == -INFINITY ? sh_s[w] : sh_s[w] * exp_over(sh_k[w], ko, c);
        float* out = parts + (row * kShares + blockIdx.x) * 2;
        out[0] = ko;
        out[1] = so;
    }
}

// The loss of a joined row.  Whichever wave is the last of all adds the rows' losses, in their order (a launch less: 61 rows of 128011
// fp32 classes 24 -> 21 us).  The counter only says who is last; the losses pass between the XCDs' caches as atomic accesses.
__device__ __forceinline__ void deliver(const DistillArgs& a, int64_t row, float l, int* __restrict__ rows_done, float* __restrict__ loss, int lane) {
    if (!rows_done) {
        if (lane == 0) a.row_loss[row] = l;
        return;
    }
    int before = 0;
    if (lane == 0) {
        __hip_atomic_store(a.row_loss + row, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        before = __hip_atomic_fetch_add(rows_done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    const int rows = (int)gridDim.x;
    if (__builtin_amdgcn_readfirstlane(before) != rows - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    int m = a.counts && !a.count_losses ? count_of(a) : 1, own = 0;
    double s = 0.0;
    for (int i = lane; i < rows; i += 64) {
        const float v = __hip_atomic_load(a.row_loss + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s += (double)v;
        own += __float_as_uint(v) != 0x80000000u;
    }
    s = wave_sum_d(s);
    own = wave_sum_i(own);
    if (a.count_losses) m = own > 0 ? own : 1;
    if (lane == 0) loss[0] = (float)(s / (double)m);
}

template <typename T>
__global__ __launch_bounds__(64) void distill_join_kernel(const DistillArgs a, const float* __restrict__ parts, int shares, float* __restrict__ joined,
                                                          int* __restrict__ rows_done, float* __restrict__ loss) {
    if (a.skip_if_one && a.upstream[0] == 1.f) return;
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const float c = a.invT * kLog2e;
    const T* z = static_cast<const T*>(a.z) + row * a.ld;
    const int cls = lane < a.k ? load_class(a, row * a.k + lane) : -1;
    if (__ballot(cls >= 0) == 0) {
        deliver(a, row, loss_of_empty(a), rows_done, loss, lane);
        return;
    }
    const float* in = parts + (row * kShares + lane) * 2;
    const float k = lane < shares ? in[0] : -INFINITY, s = lane < shares ? in[1] : 0.f;
    const float ko = wave_max(k), so = sum_wave(k == -INFINITY ? s : s * exp_over(k, ko, c));
    const Kept e = kept_entries<T>(a, row, z, cls, lane, c);
    const Joined w = join(ko, so, e.top, e.sum, c);
    const float l = kept_loss(a, e, w, ko, so, c);
    if (joined) {
        const float gs = grad_scale(a, row);
        float* out = joined + row * kRowFloats;
        if (lane == 0) {
            out[0] = ko;
            out[1] = outside_factor(w, so, e.rest, e.mass, gs);
        }
        out[2 + lane] = gs * (e.mass * exp_over(e.z, w.top, c) / w.sum - e.total);
    }
    deliver(a, row, loss_of_row(a, l), rows_done, loss, lane);
}

template <typename T>
__global__ __launch_bounds__(256) void distill_share_grad_kernel(const DistillArgs a, const float* __restrict__ joined) {
    constexpr int VEC = Piece<T>::VEC, U = 4;
    if (a.skip_if_one && a.upstream[0] == 1.f) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.y;
    const float c = a.invT * kLog2e;
    const Row<T> r(static_cast<const T*>(a.z) + row * a.ld, a.V);
    const Share<T> part(r);
    T* dst = static_cast<T*>(a.dz) + row * a.ld_d;
    const bool vec_ok = (reinterpret_cast<uintptr_t>(dst) / sizeof(T)) % VEC == (unsigned)r.phase;
    const int cls = lane < a.k ? load_class(a, row * a.k + lane) : -1;
    const bool any = __ballot(cls >= 0) != 0;
    const float* in = joined + row * kRowFloats;
    const float ko = any ? in[0] : 0.f, b = any ? in[1] : 0.f, gj = any ? in[2 + lane] : 0.f;
    const float base = ko == -INFINITY ? 0.f : ko;
    for (int g0 = part.lo + wave * 64; g0 < part.hi; g0 += 256 * U) {
        Piece<T> y[U];
        if (any) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int g = g0 + u * 256 + lane;
                if (g < part.hi) y[u] = r.load(g);
                else
#pragma unroll
                    for (int w = 0; w < 4; ++w) y[u].w[w] = 0;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[VEC] = {};
            if (any) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) f[v] = b * exp_over(y[u].get(v), base, c);
                for_kept<VEC>(cls, r.phase, g0 + u * 256, lane, [&](bool here, int v, int j) {
                    const float gv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(gj), j));
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (here && i == v) f[i] = gv;
                });
            }
            const int g = g0 + u * 256 + lane;
            if (g < part.hi) store_piece<T>(dst, vec_ok, g * VEC - r.phase, a.V, f);
        }
    }
}

// ------------------------------------------------------------------------------------------------ one thread per position
// Few classes (up to 32), all of them in the registers of one thread, VP neighbouring positions per thread: the class planes of
// [N, C, ...] logits are read with coalesced 16-byte loads (VP = 4), class-last rows with strided ones (VP = 1).
// Memory bounds it: 32 x 4 x 384 x 384 fp32 logits with 2 kept entries, loss and gradient: 246 MB in 53 us, 4.6 TB/s (a copy: 5.4).
// With scalar loads of the kept entries all kernels of that call took 168 us instead of 97.  The loss class by class, not entry by entry
// with their logits looked up again: 65 against 94 us of kernels.
template <typename T, int CM, int VP, bool GRAD>
__global__ __launch_bounds__(256) void distill_pixels_kernel(const DistillArgs a, int blocks_each) {
    if (a.skip_if_one && a.upstream[0] == 1.f) return;
    __shared__ float red[4];
    const int64_t o = blockIdx.x / blocks_each;
    const int64_t i0 = ((int64_t)(blockIdx.x % blocks_each) * 256 + threadIdx.x) * VP;
    const float c = a.invT * kLog2e;
    const T* z = static_cast<const T*>(a.z) + o * a.ld;
    const int64_t t0 = o * a.k * a.inner;
    const float gs = GRAD && !a.up_each ? grad_scale(a, 0) : 0.f;
    float block = 0.f;
    if (i0 < a.inner) {
        float x[CM][VP];
#pragma unroll
        for (int q = 0; q < CM; ++q) {
            if (q < a.V) {
                if constexpr (VP == 4) Elem<T>::load4(z + q * a.s_c + i0, x[q]);
                else x[q][0] = Elem<T>::to_f(z[q * a.s_c + i0 * a.s_p]);
            } else {
#pragma unroll
                for (int v = 0; v < VP; ++v) x[q][v] = -INFINITY;
            }
        }
        float e[CM][VP], top[VP], sum[VP], lse[VP];
        bool twice[VP];                       // two entries have the same class
        uint32_t kept[VP];
        if constexpr (VP == 4) {
            if (a.tlse) Elem<float>::load4(a.tlse + o * a.inner + i0, lse);
        } else if (a.tlse) lse[0] = a.tlse[o * a.inner + i0];
#pragma unroll
        for (int v = 0; v < VP; ++v) {
            top[v] = -INFINITY;
            sum[v] = 0.f;
            kept[v] = 0;
            twice[v] = false;
#pragma unroll
            for (int q = 0; q < CM; ++q) e[q][v] = 0.f;
        }
        const int64_t at = t0 + i0 * a.ts_p;
        if (!a.tlse)                          // renormalised: the greatest of the kept logits first
            for (int j = 0; j < a.k; ++j) {
                int cj[VP];
                float t[VP];
                load_classes<VP>(a, at + j * a.ts_c, cj);
                load_kepts<VP>(a, at + j * a.ts_c, t);
#pragma unroll
                for (int v = 0; v < VP; ++v) top[v] = cj[v] >= 0 ? fmaxf(top[v], t[v]) : top[v];
            }
        auto log_p = [&](float t, int v) {    // base 2, before it is normalised where no logsumexp is given
            return a.tlse ? fmaf(t, a.invT, -lse[v]) * kLog2e : (t == -INFINITY ? -INFINITY : (t - top[v]) * c);
        };
        for (int j = 0; j < a.k; ++j) {
            int cj[VP];
            float t[VP];
            load_classes<VP>(a, at + j * a.ts_c, cj);
            load_kepts<VP>(a, at + j * a.ts_c, t);
#pragma unroll
            for (int v = 0; v < VP; ++v) {
                const float ej = cj[v] >= 0 ? fast_exp2(log_p(t[v], v)) : 0.f;
                const uint32_t bit = cj[v] >= 0 ? 1u << cj[v] : 0u;
                twice[v] = twice[v] || (kept[v] & bit);
                kept[v] |= bit;
                sum[v] += ej;
#pragma unroll
                for (int q = 0; q < CM; ++q) e[q][v] += q == cj[v] ? ej : 0.f;
            }
        }
#pragma unroll
        for (int v = 0; v < VP; ++v) {
            const int64_t pos = o * a.inner + i0 + v;
            float l = 0.f, g = gs;
            if constexpr (GRAD)
                if (a.up_each) g = a.weight * a.T * a.upstream[pos];       // no mean goes with one gradient for each position
            float mass = sum[v], rest = 0.f, norm = 1.f;
            if (a.tlse) {
                rest = 1.f - mass;
                if (!(rest > kRestFloor) || __popc(kept[v]) == a.V) rest = 0.f;
            } else {
                norm = sum[v] == 0.f ? 0.f : 1.f / sum[v];
#pragma unroll
                for (int q = 0; q < CM; ++q) e[q][v] *= norm;
                mass = sum[v] * norm;
            }
            const float all = mass + rest;
            float zo = -INFINITY, zm = -INFINITY;
#pragma unroll
            for (int q = 0; q < CM; ++q) {
                const bool in = (kept[v] >> q) & 1u;
                zo = fmaxf(zo, in ? -INFINITY : x[q][v]);
                zm = fmaxf(zm, in ? x[q][v] : -INFINITY);
            }
            const float ko = zo, km = zm, kk = fmaxf(ko, km);
            const float bo = ko == -INFINITY ? 0.f : ko, bm = km == -INFINITY ? 0.f : km;
            float so = 0.f, sm = 0.f, w[CM];
#pragma unroll
            for (int q = 0; q < CM; ++q) {
                const bool in = (kept[v] >> q) & 1u;
                w[q] = exp_over(x[q][v], in ? bm : bo, c);
                so += in ? 0.f : w[q];
                sm += in ? w[q] : 0.f;
            }
            const float fo = rebase(ko, kk, c), fm = rebase(km, kk, c);
            const float s = so * fo + sm * fm + (so != so ? so : 0.f);
            const float inv = 1.f / s;
            if (kept[v]) {
                const float ls = log2f(s);
                if (!twice[v]) {
#pragma unroll
                    for (int q = 0; q < CM; ++q)
                        if (q < a.V) {
                            const bool in = (kept[v] >> q) & 1u;
                            if (CM > 8 && !in) continue;      // neighbours often share their classes; of few, D(1, 1) = 0 costs less than a branch
                            const float p = in ? e[q][v] : 1.f;
                            l += divergence(p, in ? w[q] * (fm * inv) : 1.f, [&] { return log2f(p) - ((x[q][v] - kk) * c - ls); });
                        }
                } else {                                      // two entries share a class: entry by entry
                    uint32_t seen = 0;
                    for (int j = 0; j < a.k; ++j) {
                        const int cls = load_class(a, at + v + j * a.ts_c);
                        if (cls < 0) continue;
                        float z = x[0][v], total = e[0][v];
#pragma unroll
                        for (int q = 1; q < CM; ++q) {
                            z = q == cls ? x[q][v] : z;
                            total = q == cls ? e[q][v] : total;
                        }
                        const float lp = log_p(load_kept(a, at + v + j * a.ts_c), v);
                        l += entry_loss(!(seen >> cls & 1u), fast_exp2(lp) * norm, a.tlse ? lp : lp - log2f(sum[v]), total, exp_over(z, kk, c) * inv, (z - kk) * c - ls);
                        seen |= 1u << cls;
                    }
                }
                l = rest_loss(a, l, rest, mass, so * fo * inv, log2f(so) + (ko - kk) * c - ls);
                l *= a.T * a.T * a.weight;
            }
            if (a.row_loss) a.row_loss[pos] = l;
            block += l;
            if constexpr (GRAD) {
                const float fk = g * all * fm * inv, fr = g * (all * fo * inv - (rest > 0.f ? rest / so : 0.f));
#pragma unroll
                for (int q = 0; q < CM; ++q)
                    x[q][v] = !kept[v] ? 0.f : ((kept[v] >> q) & 1u) ? w[q] * fk - g * e[q][v] : w[q] * fr;
            }
        }
        if constexpr (GRAD) {
            T* d = static_cast<T*>(a.dz) + o * a.ld_d;
#pragma unroll
            for (int q = 0; q < CM; ++q)
                if (q < a.V) {
                    if constexpr (VP == 4) Elem<T>::store4(d + q * a.d_c + i0, x[q]);
                    else d[q * a.d_c + i0 * a.d_p] = Elem<T>::from_f(x[q][0]);
                }
        }
    }
    if (a.partial) {
        block = sum_wave(block);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = block;
        __syncthreads();
        if (threadIdx.x == 0) a.partial[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
    }
}

// Class planes of 33 to 256 classes: one thread for a position again, but its classes do not fit its registers: they are read once for
// the maximum and the sum of those outside (running, eight loads in flight) and once more for the gradient.  The kept classes are bits
// of eight registers; their logits are gathered in the loops over the entries, and their gradients overwrite what the second pass
// wrote there.  8 x 80 x 256 x 256 fp32 logits, 1 (8) kept, with
// gradient: 126 (320) us, 4.0 (1.6) TB/s of three passes; copied into rows first 553 (829).  With many entries their gathers bound it.
constexpr int kPlaneClasses = 256, kPlaneTop = 8;

// f(first class, eight logits, the bits of those kept) for all classes of a position; beyond the last: -inf
template <typename T, typename F> __device__ __forceinline__ void each_eight(const T* z, int64_t stride, int V, const uint32_t (&kept)[kPlaneClasses / 32], F&& f) {
#pragma unroll
    for (int w = 0; w < kPlaneClasses / 32; ++w) {
        const int end = V < w * 32 + 32 ? V : w * 32 + 32;
        for (int q0 = w * 32; q0 < end; q0 += 8) {
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = q0 + u < V ? Elem<T>::to_f(z[(q0 + u) * stride]) : -INFINITY;
            f(q0, x, (kept[w] >> (q0 & 31)) & 0xFFu);
        }
    }
}

template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void distill_planes_kernel(const DistillArgs a, int blocks_each) {
    if (a.skip_if_one && a.upstream[0] == 1.f) return;
    __shared__ float red[4];
    const int64_t o = blockIdx.x / blocks_each, i = (int64_t)(blockIdx.x % blocks_each) * 256 + threadIdx.x;
    const float c = a.invT * kLog2e;
    const float gs = GRAD && !a.up_each ? grad_scale(a, 0) : 0.f;
    float l = 0.f;
    if (i < a.inner) {
        const T* z = static_cast<const T*>(a.z) + o * a.ld + i;
        const int64_t pos = o * a.inner + i, at = o * a.k * a.inner + i;
        const float lse = a.tlse ? a.tlse[pos] : 0.f;
        auto logit = [&](int cls) { return Elem<T>::to_f(z[cls * a.inner]); };
        float top = -INFINITY;
        if (!a.tlse)                          // renormalised: the greatest of the kept logits first
            for (int j = 0; j < a.k; ++j)
                if (load_class(a, at + j * a.inner) >= 0) top = fmaxf(top, load_kept(a, at + j * a.inner));
        auto log_p = [&](int j) {             // base 2, before it is normalised where no logsumexp is given
            const float t = load_kept(a, at + j * a.inner);
            return a.tlse ? fmaf(t, a.invT, -lse) * kLog2e : (t == -INFINITY ? -INFINITY : (t - top) * c);
        };
        uint32_t kept[kPlaneClasses / 32] = {};
        bool twice = false;
        float mass = 0.f, km = -INFINITY, sm = 0.f;
        for (int j = 0; j < a.k; ++j) {
            const int cls = load_class(a, at + j * a.inner);
            if (cls < 0) continue;
            mass += fast_exp2(log_p(j));
            bool seen = false;
#pragma unroll
            for (int w = 0; w < kPlaneClasses / 32; ++w) {
                const uint32_t bit = cls >> 5 == w ? 1u << (cls & 31) : 0u;
                seen = seen || (kept[w] & bit);
                kept[w] |= bit;
            }
            twice = twice || seen;
            if (!seen) {
                const float zj = logit(cls);
                if (zj > km) {
                    sm *= rebase(km, zj, c);
                    km = zj;
                }
                sm += exp_over(zj, km == -INFINITY ? 0.f : km, c);
            }
        }
        int distinct = 0;
#pragma unroll
        for (int w = 0; w < kPlaneClasses / 32; ++w) distinct += __popc(kept[w]);
        float ko = -INFINITY, so = 0.f;
        if (distinct)
            each_eight(z, a.inner, a.V, kept, [&](int, float (&x)[8], uint32_t in) {
                float m = ko;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    x[u] = (in >> u) & 1u ? -INFINITY : x[u];
                    m = fmaxf(m, x[u]);
                }
                so *= m > ko ? rebase(ko, m, c) : 1.f;
                ko = m;
                const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int u = 0; u < 8; ++u) so += exp_over(x[u], base, c);
            });
        float rest = 0.f, norm = 1.f, log_norm = 0.f;
        if (a.tlse) {
            rest = 1.f - mass;
            if (!(rest > kRestFloor) || distinct == a.V) rest = 0.f;
        } else {
            norm = mass == 0.f ? 0.f : 1.f / mass;
            log_norm = log2f(mass);
            mass *= norm;
        }
        const float all = mass + rest;
        const float kk = fmaxf(ko, km), bo = ko == -INFINITY ? 0.f : ko, bm = km == -INFINITY ? 0.f : km;
        const float fo = rebase(ko, kk, c), fm = rebase(km, kk, c), s = so * fo + sm * fm + (so != so ? so : 0.f);
        if (distinct) {
            const float ls = log2f(s), inv = 1.f / s;
            for (int j = 0; j < a.k; ++j) {
                const int cls = load_class(a, at + j * a.inner);
                if (cls < 0) continue;
                const float lp = log_p(j), p = fast_exp2(lp), zj = logit(cls);
                float total = p;
                bool first = true;
                if (twice) {
                    total = 0.f;
                    for (int h = 0; h < a.k; ++h)
                        if (load_class(a, at + h * a.inner) == cls) {
                            total += fast_exp2(log_p(h));
                            first = first && h >= j;
                        }
                }
                l += entry_loss(first, p * norm, lp - log_norm, total * norm, exp_over(zj, kk, c) * inv, (zj - kk) * c - ls);
            }
            l = rest_loss(a, l, rest, mass, so * fo * inv, log2f(so) + (ko - kk) * c - ls);
            l *= a.T * a.T * a.weight;
        }
        if (a.row_loss) a.row_loss[pos] = l;
        if constexpr (GRAD) {
            const float g = a.up_each ? a.weight * a.T * a.upstream[pos] : gs;           // no mean goes with one gradient for each position
            const float inv = 1.f / s, fk = g * all * fm * inv, fr = g * (all * fo * inv - (rest > 0.f ? rest / so : 0.f));
            T* d = static_cast<T*>(a.dz) + o * a.ld_d + i;
            if (distinct) {
                each_eight(z, a.inner, a.V, kept, [&](int q0, float (&x)[8], uint32_t) {
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (q0 + u < a.V) d[(q0 + u) * a.inner] = Elem<T>::from_f(exp_over(x[u], bo, c) * fr);
                });
                for (int j = 0; j < a.k; ++j) {
                    const int cls = load_class(a, at + j * a.inner);
                    if (cls < 0) continue;
                    float p = fast_exp2(log_p(j));
                    if (twice) {
                        p = 0.f;
                        for (int h = 0; h < a.k; ++h)
                            if (load_class(a, at + h * a.inner) == cls) p += fast_exp2(log_p(h));
                    }
                    d[cls * a.inner] = Elem<T>::from_f(exp_over(logit(cls), bm, c) * fk - g * (p * norm));
                }
            } else {
                for (int q = 0; q < a.V; ++q) d[q * a.inner] = Elem<T>::from_f(0.f);
            }
        }
    }
    if (a.partial) {
        l = sum_wave(l);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = l;
        __syncthreads();
        if (threadIdx.x == 0) a.partial[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
    }
}

// Positions with at least one kept logit: one partial count for each workgroup.
// Rows: the entries of 64 / kp rows at a time, one for each lane, kp = k rounded up to a power of two.
__global__ __launch_bounds__(256) void distill_count_rows_kernel(const DistillArgs a, int64_t rows, int log_kp, int* __restrict__ counts) {
    __shared__ int red[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = count_rows(a, rows, log_kp, (int64_t)blockIdx.x * 4 + wave, (int64_t)kCountBlocks * 4, lane);
    if (lane == 0) red[wave] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}
// Planes: a thread takes 16 loads of positions at a time and reads entry after entry until each has one (the first decides most of
// them); all loads of an entry are in flight together.  Four neighbouring positions for each load where the plane allows it (4.7
// million positions, 2 entries, a tenth without: 12 us; one position for each load 16 us).
__global__ __launch_bounds__(1024) void distill_count_planes4_kernel(const DistillArgs a, int64_t positions, int* __restrict__ counts) {
    __shared__ int red[16];
    constexpr int U = 6, STEP = 1024 * 4;
    int n = 0;
    const int64_t per = (positions / 4 + kCountBlocks - 1) / kCountBlocks * 4, lo = per * blockIdx.x, hi = lo + per < positions ? lo + per : positions;
    for (int64_t p = lo + threadIdx.x * 4; p < hi; p += STEP * U) {
        int64_t at[U];
        int c[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t q = (uint32_t)(p + u * STEP < hi ? p + u * STEP : p), o = q / (uint32_t)a.inner;       // positions < 2^31
            at[u] = (int64_t)o * a.k * a.inner + (q - o * (uint32_t)a.inner);
#pragma unroll
            for (int v = 0; v < 4; ++v) c[u][v] = -1;
        }
        for (int j = 0; j < a.k; ++j) {
            int lowest = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int4 i = *reinterpret_cast<const int4*>(static_cast<const int32_t*>(a.idx) + at[u] + j * a.inner);
                const int d[4] = {i.x, i.y, i.z, i.w};
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    c[u][v] = d[v] >= 0 && d[v] < a.V ? d[v] : c[u][v];
                    lowest = c[u][v] < lowest ? c[u][v] : lowest;
                }
            }
            if (lowest >= 0) break;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int v = 0; v < 4; ++v) n += p + u * STEP < hi && c[u][v] >= 0;
    }
    n = wave_sum_i(n);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        int t = 0;
        for (int i = 0; i < 16; ++i) t += red[i];
        counts[blockIdx.x] = t;
    }
}
template <typename I> __global__ __launch_bounds__(1024) void distill_count_planes_kernel(const DistillArgs a, int64_t positions, int* __restrict__ counts) {
    __shared__ int red[16];
    constexpr int U = 16;
    int n = 0;
    const int64_t per = (positions + kCountBlocks - 1) / kCountBlocks, lo = per * blockIdx.x, hi = lo + per < positions ? lo + per : positions;
    for (int64_t p = lo + threadIdx.x; p < hi; p += 1024 * U) {
        int64_t at[U], o = p / a.inner, i = p - o * a.inner;
        int c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            at[u] = p + u * 1024 < hi ? o * a.k * a.inner + i * a.ts_p : at[0];
            c[u] = -1;
            i += 1024;
            if (a.inner >= 1024) {
                if (i >= a.inner) { i -= a.inner; ++o; }
            } else {
                o += i / a.inner;
                i %= a.inner;
            }
        }
        for (int j = 0; j < a.k; ++j) {
            int lowest = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int d = load_class_as<I>(a, at[u] + j * a.ts_c);
                c[u] = d > c[u] ? d : c[u];
                lowest = c[u] < lowest ? c[u] : lowest;
            }
            if (lowest >= 0) break;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) n += p + u * 1024 < hi && c[u] >= 0;
    }
    n = wave_sum_i(n);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        int t = 0;
        for (int i = 0; i < 16; ++i) t += red[i];
        counts[blockIdx.x] = t;
    }
}

__device__ __forceinline__ double block_sum_1024(double s, double* red) {
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    double t = 0.0;
    if (threadIdx.x == 0)
        for (int i = 0; i < 16; ++i) t += red[i];
    return t;
}
__device__ __forceinline__ int block_sum_i(int n, double* red) {
    n = wave_sum_i(n);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = (double)n;
    __syncthreads();
    int t = 0;
    for (int i = 0; i < 16; ++i) t += (int)red[i];
    return t;
}
// level 1 of the final sum (many positions): workgroup b adds its own range in double
__global__ __launch_bounds__(1024) void distill_collect_kernel(const DistillArgs a, const float* __restrict__ v, int64_t n, float* __restrict__ out) {
    __shared__ double red[16];
    const int64_t per = (n + gridDim.x - 1) / gridDim.x, lo = per * blockIdx.x, hi = lo + per < n ? lo + per : n;
    double s = 0.0;
    int m = 0;
    for (int64_t i = lo + threadIdx.x; i < hi; i += 1024) {
        s += (double)v[i];
        m += __float_as_uint(v[i]) != 0x80000000u;
    }
    s = block_sum_1024(s, red);
    if (threadIdx.x == 0) out[blockIdx.x] = (float)s;
    if (a.count_losses) {
        m = block_sum_i(m, red);
        if (threadIdx.x == 0) a.counts[blockIdx.x] = m;
    }
}
__global__ __launch_bounds__(1024) void distill_finalize_kernel(const DistillArgs a, const float* __restrict__ v, int n, float* __restrict__ loss) {
    __shared__ double red[16];
    int m = a.counts && a.count_losses != 1 ? count_of(a) : 1;
    int own = 0;
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) {
        s += (double)v[i];
        own += __float_as_uint(v[i]) != 0x80000000u;
    }
    s = block_sum_1024(s, red);
    if (a.count_losses == 1) {
        own = block_sum_i(own, red);
        m = own > 0 ? own : 1;
    }
    if (threadIdx.x == 0) loss[0] = (float)(s / (double)m);
}

// ------------------------------------------------------------------------------------------------ the k greatest of a row
// A float as an integer that orders like it: NaN above everything, both zeros alike.
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t b = __float_as_uint(f + 0.f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

constexpr int kMostCandidates = 1024;

// Rows of one wave: four of them share a workgroup while their lists are short, and do not wait for each other.  A million rows of 80
// (300) fp32 logits: 645 -> 455 (761 -> 537) us, 8000 rows of 80: 7.9 -> 7.0.  With the lists of longer rows fewer waves fit a CU: 32000
// rows of 1000 logits 34 -> 39.  (Lists of 512 entries: 100000 rows of 600 bf16 logits 131 -> 81 us.)
constexpr int rows_per_group(int nt, int nch) { return nt == 64 && nch <= 2 ? 4 : 1; }
template <int R> __device__ __forceinline__ void sync_row() {
    if constexpr (R > 1) one_wave_sync();
    else __syncthreads();
}

// Selection in three steps.  (1) Every thread takes the maximum of its part of the row (and the row's logsumexp is formed).
// (2) The first wave finds a value that at least k of these maxima reach, by a binary search over the bits with ballots: at least
// k elements of the row reach it, and hardly more than k in unordered data.  (3) The elements that reach it are collected in LDS
// and ranked by counting; ties go to the lower index.  Where more than the list holds reach it (many ties) or a NaN is in the row,
// the exact k-th key and then the last index that still belongs are found by binary searches over the whole row.
// The row is read once: 4096 rows of 32000 bf16 logits, 32 kept: 262 MB in 57 us, 4.6 TB/s (the read alone: 48).  What is left are
// the search of (2), during which one wave works, and the exponentials; other rows on the CU cover most of both.
template <typename T, int NT, int NCH>
__global__ __launch_bounds__(NT * rows_per_group(NT, NCH), NT * NCH == 4096 ? 6 : 1) void top_rows_kernel(const T* __restrict__ z, int64_t rows, int64_t ld, int V, int k, float invT, T* __restrict__ values,
                                                      int32_t* __restrict__ indices, float* __restrict__ lse) {
    constexpr int VEC = Piece<T>::VEC, NW = NT / 64, R = rows_per_group(NT, NCH);
    constexpr int kMost = R > 1 ? kMostCandidates / 2 : kMostCandidates, kCandidates = NCH > 0 && NT * NCH * VEC < kMost ? NT * NCH * VEC : kMost;
    __shared__ struct {
        float m[NT], k[NW], s[NW];
        uint32_t ck[kCandidates], bound;
        int ci[kCandidates], n[NW], count, slow;
    } shared[R];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int of = R == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.y);
    const int64_t row = (int64_t)blockIdx.x * R + of;
    if (R > 1 && row >= rows) return;
    auto& sh = shared[of];
    const float c = invT * kLog2e;
    const Row<T> r(z + row * ld, V);
    Piece<T> x[NCH > 0 ? NCH : 1];
    float m = -INFINITY, sw = 0.f, kw;
    if constexpr (NCH > 0) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int g = i * NT + (int)threadIdx.x;
            if (g < r.pieces) x[i] = r.load(g);
            else
#pragma unroll
                for (int w = 0; w < 4; ++w) x[i].w[w] = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
        }
        m = lane_max<T, NCH>(x);
        const float mw = wave_max(m);
        kw = mw;
        const float base = mw == -INFINITY ? 0.f : mw;
        stay_packed(x);
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) sw += exp_over(x[i].get(v), base, c);
        sw = sum_wave(sw);
    } else {
        for (int g = threadIdx.x; g < r.pieces; g += NT) {
            const Piece<T> y = r.load(g);
            float mg = y.get(0);
#pragma unroll
            for (int v = 1; v < VEC; ++v) mg = fmaxf(mg, y.get(v));
            if (mg > m) {
                sw *= rebase(m, mg, c);
                m = mg;
            }
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int v = 0; v < VEC; ++v) sw += exp_over(y.get(v), base, c);
        }
        kw = wave_max(m);
        sw = sum_wave(m == -INFINITY ? sw : sw * exp_over(m, kw, c));
    }
    sh.m[threadIdx.x] = m;
    if (lane == 0) { sh.k[wave] = kw; sh.s[wave] = sw; }
    if (threadIdx.x == 0) sh.count = 0;
    sync_row<R>();
    if (wave == 0) {
        float kk = sh.k[0], s = 0.f;
#pragma unroll
        for (int w = 1; w < NW; ++w) kk = fmaxf(kk, sh.k[w]);
#pragma unroll
        for (int w = 0; w < NW; ++w) s += sh.k[w] == -INFINITY ? sh.s[w] : sh.s[w] * exp_over(sh.k[w], kk, c);
        if (lane == 0 && lse) lse[row] = (kk == -INFINITY && s == 0.f) ? -INFINITY : kk * invT + log2f(s) * kLn2;
        // 64 to 256 groups of threads, whatever the workgroup's size: 1024 rows of 128011 bf16 (fp32) logits with up to 1024 groups 100 (234)
        // us, with 256 85 (156)
        constexpr int NG = NW < 4 ? NW : 4;
        uint32_t key[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float mg = sh.m[g * 64 + lane];
#pragma unroll
            for (int w = g + NG; w < NW; w += NG) mg = fmaxf(mg, sh.m[w * 64 + lane]);
            key[g] = order_key(mg);
        }
        uint32_t bound = 0;
        for (int bit = 31; bit >= (sizeof(T) == 2 ? 16 : 0); --bit) {
            const uint32_t cand = bound | (1u << bit);
            int n = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g) n += __popcll(__ballot(key[g] >= cand));
            if (n >= k) {
                bound = cand;
                if (n <= k + (k >> 2) + 2) break;
            }
        }
        if (lane == 0) {
            sh.bound = bound;
            sh.slow = s != s;
        }
    }
    sync_row<R>();

    auto take = [&](uint32_t key, int e) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kCandidates) { sh.ck[at] = key; sh.ci[at] = e; }
    };
    auto each_in_memory = [&](auto&& f) {
        for (int g = threadIdx.x; g < r.pieces; g += NT) {
            const Piece<T> y = r.load(g);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int e = g * VEC - r.phase + v;
                if (e >= 0 && e < V) f(y.get(v), e);
            }
        }
    };
    const uint32_t bound = sh.bound;
    bool slow = sh.slow != 0;
    if (!slow) {
        // the bound as a float: keys of floats order as the floats do, so the elements are compared unconverted
        const float fb = bound <= 0x007FFFFFu ? -INFINITY      // no key lies between 0 and that of -inf: everything belongs
                                              : __uint_as_float((bound & 0x80000000u) ? bound & 0x7FFFFFFFu : ~bound);
        if constexpr (NCH > 0) {
            if (m >= fb) {
                stay_packed(x);
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    if (!may_reach<T>(x[i], fb)) continue;
                    uint32_t hit = 0;
#pragma unroll
                    for (int v = 0; v < VEC; ++v) hit |= x[i].get(v) >= fb ? 1u << v : 0u;
                    const int e0 = (i * NT + (int)threadIdx.x) * VEC - r.phase;
                    while (hit) {
                        const int v = __builtin_ctz(hit);
                        hit &= hit - 1;
                        float f = x[i].get(0);
#pragma unroll
                        for (int u = 1; u < VEC; ++u) f = u == v ? x[i].get(u) : f;
                        if (e0 + v >= 0 && e0 + v < V) take(order_key(f), e0 + v);
                    }
                }
            }
        } else {
            if (m >= fb)
                each_in_memory([&](float f, int e) {
                    if (f >= fb) take(order_key(f), e);
                });
        }
        sync_row<R>();
        slow = sh.count > kCandidates;
    }
    if (slow) {
        auto count = [&](auto&& pred) {
            int n = 0;
            each_in_memory([&](float f, int e) { n += pred(order_key(f), e) ? 1 : 0; });
            n = wave_sum_i(n);
            sync_row<R>();
            if (lane == 0) sh.n[wave] = n;
            sync_row<R>();
            int t = 0;
            for (int w = 0; w < NW; ++w) t += sh.n[w];
            return t;
        };
        uint32_t kth = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t cand = kth | (1u << bit);
            if (count([&](uint32_t q, int) { return q >= cand; }) >= k) kth = cand;
        }
        const int need = k - count([&](uint32_t q, int) { return q > kth; });     // of the elements equal to the k-th
        int last = 0;
        for (int bit = 30; bit >= 0; --bit) {
            const int cand = last | (1 << bit);
            if (cand < V && count([&](uint32_t q, int e) { return q == kth && e < cand; }) < need) last = cand;
        }
        sync_row<R>();
        if (threadIdx.x == 0) sh.count = 0;
        sync_row<R>();
        each_in_memory([&](float f, int e) {
            const uint32_t q = order_key(f);
            if (q > kth || (q == kth && e <= last)) take(q, e);
        });
        sync_row<R>();
    }
    int n = sh.count < kCandidates ? sh.count : kCandidates;
    // Many candidates (ties, k near the number of groups): the first wave keeps exactly k of them, so that the ranking, which compares
    // each with all, stays short (20000 rows of 300 fp32 logits, 64 kept: 378 -> 72 us).
    if (n > (NT == 64 ? 64 : 128)) {
        if (wave == 0) {
            // from LDS each time: in registers they would cost the whole kernel a wave per SIMD
            auto count = [&](auto&& pred) {
                int t = 0;
                for (int j = 0; j < n; j += 64) {
                    const int i = j + lane;
                    t += __popcll(__ballot(i < n && pred(sh.ck[i < n ? i : 0], sh.ci[i < n ? i : 0])));
                }
                return t;
            };
            uint32_t kth = 0;
            int reach = n;
            for (int bit = 31; bit >= 0 && reach > k; --bit) {
                const uint32_t cand = kth | (1u << bit);
                const int t = count([&](uint32_t q, int) { return q >= cand; });
                if (t >= k) {
                    kth = cand;
                    reach = t;
                }
            }
            int last = 0x7FFFFFFF;                            // of the elements equal to the k-th, the index of the last that belongs
            if (reach > k) {
                const int need = k - count([&](uint32_t q, int) { return q > kth; });
                last = 0;
                for (int bit = 30; bit >= 0; --bit) {
                    const int cand = last | (1 << bit);
                    if (cand < V && count([&](uint32_t q, int e) { return q == kth && e < cand; }) < need) last = cand;
                }
            }
            int to = 0;
            for (int j = 0; j < n; j += 64) {                 // forward and never past what has been read
                const int i = j + lane;
                const uint32_t q = sh.ck[i < n ? i : 0];
                const int e = sh.ci[i < n ? i : 0];
                const bool keep = i < n && (q > kth || (q == kth && e <= last));
                const uint64_t mask = __ballot(keep);
                if (keep) {
                    const int d = to + __popcll(mask & ((1ull << lane) - 1));
                    sh.ck[d] = q;
                    sh.ci[d] = e;
                }
                to += __popcll(mask);
            }
        }
        n = k;
        sync_row<R>();
    }
    for (int i = threadIdx.x; i < n; i += NT) {
        const uint32_t q = sh.ck[i];
        const int e = sh.ci[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += (sh.ck[j] > q || (sh.ck[j] == q && sh.ci[j] < e)) ? 1 : 0;
        if (rank < k) {
            indices[row * k + rank] = e;
            values[row * k + rank] = r.p[e];
        }
    }
}

// elements widened to floats and written back with their bits as they were: a conversion may turn one NaN into another
__device__ __forceinline__ float load_same(const float* p) { return *p; }
__device__ __forceinline__ float load_same(const bf16* p) { return __uint_as_float((uint32_t) * reinterpret_cast<const uint16_t*>(p) << 16); }
__device__ __forceinline__ void load_same4(const float* p, float (&v)[4]) { Elem<float>::load4(p, v); }
__device__ __forceinline__ void load_same4(const bf16* p, float (&v)[4]) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(w.x << 16);
    v[1] = __uint_as_float(w.x & 0xFFFF0000u);
    v[2] = __uint_as_float(w.y << 16);
    v[3] = __uint_as_float(w.y & 0xFFFF0000u);
}
__device__ __forceinline__ void store_same(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_same(bf16* p, float v) { *reinterpret_cast<uint16_t*>(p) = (uint16_t)(__float_as_uint(v) >> 16); }
__device__ __forceinline__ void store_same4(float* p, const float (&v)[4]) { Elem<float>::store4(p, v); }
__device__ __forceinline__ void store_same4(bf16* p, const float (&v)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2((__float_as_uint(v[0]) >> 16) | (__float_as_uint(v[1]) & 0xFFFF0000u),
                                              (__float_as_uint(v[2]) >> 16) | (__float_as_uint(v[3]) & 0xFFFF0000u));
}

// one thread per position, up to 32 classes in its registers: k rounds of "greatest that is left".  32 x 4 x 384 x 384 fp32 logits,
// the best 2: 170 MB in 32 us, 5.3 TB/s, bound by memory.
template <typename T, int CM, int VP>
__global__ __launch_bounds__(256) void top_pixels_kernel(const T* __restrict__ z, int64_t ld, int64_t s_c, int64_t s_p, int64_t inner, int V,
                                                         int k, float invT, T* __restrict__ values, int32_t* __restrict__ indices,
                                                         int64_t ts_c, int64_t ts_p, float* __restrict__ lse, int blocks_each) {
    const int64_t o = blockIdx.x / blocks_each;
    const int64_t i0 = ((int64_t)(blockIdx.x % blocks_each) * 256 + threadIdx.x) * VP;
    if (i0 >= inner) return;
    const float c = invT * kLog2e;
    z += o * ld;
    float x[CM][VP];
#pragma unroll
    for (int q = 0; q < CM; ++q) {
        if (q < V) {
            if constexpr (VP == 4) load_same4(z + q * s_c + i0, x[q]);
            else x[q][0] = load_same(z + q * s_c + i0 * s_p);
        } else {
#pragma unroll
            for (int v = 0; v < VP; ++v) x[q][v] = -INFINITY;
        }
    }
    uint32_t done[VP];
    float out[VP];
#pragma unroll
    for (int v = 0; v < VP; ++v) {
        done[v] = 0;
        float m = -INFINITY, s = 0.f;
#pragma unroll
        for (int q = 0; q < CM; ++q) m = fmaxf(m, x[q][v]);
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int q = 0; q < CM; ++q) s += exp_over(x[q][v], base, c);
        out[v] = (m == -INFINITY && s == 0.f) ? -INFINITY : base * invT + log2f(s) * kLn2;
    }
    if (lse) {
        if constexpr (VP == 4) Elem<float>::store4(lse + o * inner + i0, out);
        else lse[o * inner + i0] = out[0];
    }
    const int64_t t0 = o * k * inner;
    for (int j = 0; j < k; ++j) {
        int at[VP];
        float val[VP];
#pragma unroll
        for (int v = 0; v < VP; ++v) {
            uint32_t best = 0;
            at[v] = 0;
            val[v] = x[0][v];
            bool have = false;
#pragma unroll
            for (int q = 0; q < CM; ++q) {
                const uint32_t key = order_key(x[q][v]);
                const bool better = q < V && !((done[v] >> q) & 1u) && (!have || key > best);
                best = better ? key : best;
                at[v] = better ? q : at[v];
                val[v] = better ? x[q][v] : val[v];
                have = have || better;
            }
            done[v] |= 1u << at[v];
        }
        T* out_v = values + t0 + j * ts_c + i0 * ts_p;
        int32_t* out_i = indices + t0 + j * ts_c + i0 * ts_p;
        if constexpr (VP == 4) {
            store_same4(out_v, val);
            *reinterpret_cast<int4*>(out_i) = make_int4(at[0], at[1], at[2], at[3]);
        } else {
            store_same(out_v, val[0]);
            *out_i = at[0];
        }
    }
}

// Class planes of 33 to 256 classes, up to KM of them kept: a thread for a position reads them once and keeps a sorted list in registers,
// the keys of the logits and their classes; equal keys stay in the order of their classes.  8 x 80 x 256 x 256 fp32 logits, the best 1
// (8): 36 (70) us, 4.6 (2.4) TB/s; copied into rows first 354 (483).
template <typename T, int KM>
__global__ __launch_bounds__(256) void top_planes_kernel(const T* __restrict__ z, int64_t ld, int64_t inner, int V, int k, float invT, T* __restrict__ values,
                                                         int32_t* __restrict__ indices, float* __restrict__ lse, int blocks_each) {
    const int64_t o = blockIdx.x / blocks_each, i = (int64_t)(blockIdx.x % blocks_each) * 256 + threadIdx.x;
    if (i >= inner) return;
    const float c = invT * kLog2e;
    z += o * ld + i;
    const uint32_t none[kPlaneClasses / 32] = {};
    uint32_t key[KM];                          // 0: nothing yet, less than the key of any logit
    int cls[KM];
#pragma unroll
    for (int j = 0; j < KM; ++j) {
        key[j] = 0;
        cls[j] = 0;
    }
    float top = -INFINITY, s = 0.f;
    each_eight(z, inner, V, none, [&](int q0, float (&x)[8], uint32_t) {
        float m = top;
#pragma unroll
        for (int u = 0; u < 8; ++u) m = fmaxf(m, x[u]);
        s *= m > top ? rebase(top, m, c) : 1.f;
        top = m;
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            s += exp_over(x[u], base, c);
            uint32_t q = order_key(x[u]);
            if (q0 + u < V && q > key[KM - 1]) {
                int e = q0 + u;
                bool in = false;               // from its place on everything moves down
#pragma unroll
                for (int j = 0; j < KM; ++j) {
                    in = in || q > key[j];
                    const uint32_t kj = key[j];
                    const int cj = cls[j];
                    key[j] = in ? q : kj;
                    cls[j] = in ? e : cj;
                    q = in ? kj : q;
                    e = in ? cj : e;
                }
            }
        }
    });
    if (lse) lse[o * inner + i] = (top == -INFINITY && s == 0.f) ? -INFINITY : (top == -INFINITY ? 0.f : top) * invT + log2f(s) * kLn2;
    const int64_t t0 = o * k * inner + i;
#pragma unroll
    for (int j = 0; j < KM; ++j)
        if (j < k) {
            values[t0 + j * inner] = z[cls[j] * inner];
            indices[t0 + j * inner] = cls[j];
        }
}

// ------------------------------------------------------------------------------------------------ host
constexpr int kPixelClasses = 32;    // more classes than this: one workgroup (or wave) per row

// Threads of a row's workgroup and pieces in registers per thread, by the row's length.  Rows of 16 to 64 KB: 512 threads with 8
// pieces serve the loss, 256 with 16 the selection, whose search by the first wave leaves the others idle (4096 rows of 32000 bf16
// logits: loss and gradient 103 against 107 us, selection 66 against 56; six waves of the latter per SIMD instead of five: 67 -> 63).
template <typename T, bool TOP, typename F> static void row_tier(const void* z, int64_t rows, int64_t ld, int64_t V, int64_t k, F&& f) {
    constexpr int VEC = 16 / (int)sizeof(T);
    // Rows that begin between two pieces may touch one more.  (4096 rows of 16384 bf16 logits, 2048 pieces: selection 52 -> 39 us, loss with
    // gradient 83 -> 62 since they are not taken for 2049.)
    const int64_t pieces = (V + (aligned16(z) && ld % VEC == 0 ? VEC - 1 : 2 * (VEC - 1))) / VEC;
#define SEGK_TIER(nt, nch) if (pieces <= (int64_t)(nt) * (nch)) return f(std::integral_constant<int, nt>{}, std::integral_constant<int, nch>{})
    SEGK_TIER(64, 1);
    // The selection's bound lets few candidates through while k is well below the number of threads; a wave for each row still wins where its list
    // holds all that pass and the rows fill the chip.  64 / 256 threads, us: 20000 rows of 2000 bf16 logits, 24 kept 51/68, 32 kept 70/71,
    // 64 kept 517/111; of 1000, 32 kept 50/72, 40 kept 65/80, 48 kept 99/96; 8000 rows of 1000, 32 kept 32/34, 40 kept 37/37; 1000 rows
    // 20/13, 24/14.  fp32, 32 kept: 20000 rows of 1000 58/64, 8000 28/30, 4000 17/19, 2000 15/12.  20000 rows of 300, 64 kept: 71/114.
    if (!TOP || k <= 24 || V <= 512 || (V <= 1024 && k <= 40 && rows >= 6144)) {
        SEGK_TIER(64, 2);
        SEGK_TIER(64, 4);
        SEGK_TIER(64, 8);
    }
    SEGK_TIER(256, 4);
    SEGK_TIER(256, 8);
    if constexpr (TOP) {
        SEGK_TIER(256, 16);
    } else {
        SEGK_TIER(512, 8);
    }
    SEGK_TIER(1024, 8);
    SEGK_TIER(1024, 16);
#undef SEGK_TIER
    return f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 0>{});
}

static int check_logits(const char* who, const void* z, int dtype, int64_t outer, int64_t C, int64_t inner, int64_t ld, int64_t k,
                        float temperature, int most_planes) {
    SEGK_REQUIRE(z, SEGK_EINVAL, "%s: null pointer", who);
    SEGK_REQUIRE(dtype == SEGK_F32 || dtype == SEGK_BF16, SEGK_EINVAL, "%s: unknown dtype %d", who, dtype);
    SEGK_REQUIRE(outer > 0 && C > 0 && inner > 0 && outer < (1ll << 31) && C < (1ll << 30) && inner < (1ll << 31), SEGK_ESHAPE, "%s: bad shape", who);
    SEGK_REQUIRE(outer * inner < (1ll << 31), SEGK_ESHAPE, "%s: 2^31 positions and more", who);
    SEGK_REQUIRE(inner == 1 || C <= most_planes, SEGK_ESHAPE, "%s: more than %d classes have to be the innermost dimension", who, most_planes);
    SEGK_REQUIRE(ld >= C * inner, SEGK_ESHAPE, "%s: ld smaller than one row / image", who);
    SEGK_REQUIRE(k >= 1 && k <= kTopMax && k <= C, SEGK_ESHAPE, "%s: k must be between 1 and %d and at most the number of classes", who, kTopMax);
    // so that neither 1 / T nor T^2 leaves the range of fp32
    SEGK_REQUIRE(temperature >= 0x1p-40f && temperature <= 0x1p40f, SEGK_EINVAL, "%s: temperature must be between 2^-40 and 2^40", who);
    SEGK_REQUIRE(reinterpret_cast<uintptr_t>(z) % esize(dtype) == 0, SEGK_EALIGN, "%s: logits are not aligned to their type", who);
    return SEGK_OK;
}

// geometry of the thread-per-position kernels: rows of few classes count as the positions of one image, classes innermost
struct Pixels {
    int64_t outer, inner, s_c, s_p, ts_c, ts_p;
    int vp, blocks_each;
    int64_t blocks;
};
static Pixels pixels(int64_t outer, int64_t C, int64_t inner, int64_t ld, int64_t k, bool may_vec) {
    Pixels p;
    if (inner == 1) {
        p = {1, outer, 1, ld, 1, k, 1, 0, 0};
    } else {
        p = {outer, inner, inner, 1, inner, 1, 1, 0, 0};
        if (may_vec && C <= 8 && inner % 4 == 0 && ld % 4 == 0) p.vp = 4;
    }
    p.blocks_each = (int)((p.inner + 256 * p.vp - 1) / (256 * p.vp));
    p.blocks = p.outer * p.blocks_each;
    return p;
}
// One thread per position: class planes of up to 32 classes, and rows of so few classes.  Rows of 9 to 32 classes go to a wave each
// while they are too few to fill the chip with threads.  Thread / wave for each row, fp32, selection and loss with gradient, us: 8000
// rows of 4 classes 3.2/11.4, 8.7/15.2, of 16 6.3/7.5, 12.7/15.1, of 32 9.4/7.5, 18.6/15.3; 32000 of 32 9.6/18.4, 20.7/30.4; 1000 of 9
// 4.1/5.1, 9.9/9.5, of 32 9.3/5.1, 18.0/9.4.
static bool few(int64_t outer, int64_t C, int64_t inner) { return C <= kPixelClasses && (inner > 1 || C <= 8 || outer >= 512 * C); }

// f(first, n) for all units (rows, images) of so many threads each: a launch has to have fewer than 2^32 threads
template <typename F> static void by_launches(int64_t units, int64_t threads, F&& f) {
    const int64_t fit = (1ll << 31) / threads, most = fit < 1 ? 1 : fit;      // a single unit has at most 2^31 + 255 threads
    for (int64_t u = 0; u < units; u += most) f(u, units - u < most ? units - u : most);
}
template <typename T> static T* advance(T* p, int64_t elements) { return p ? p + elements : p; }
static const void* advance(const void* p, int64_t elements, size_t size) { return static_cast<const char*>(p) + elements * (int64_t)size; }

static bool planes(int64_t C, int64_t inner) { return inner > 1 && C > kPixelClasses; }

template <typename F> static void class_tier(int64_t C, int vp, F&& f) {
    if (C <= 4) return vp == 4 ? f(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{}) : f(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
    if (C <= 8) return vp == 4 ? f(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{}) : f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    if (C <= 16) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
}

}  // namespace segk

using namespace segk;

extern "C" int segk_top_logits(const void* logits, int dtype, int64_t outer, int64_t C, int64_t inner, int64_t ld, int64_t k, float temperature,
                               void* values, int32_t* indices, float* lse, int dev, void* stream) {
    if (const int rc = check_logits("top_logits", logits, dtype, outer, C, inner, ld, k, temperature, k <= kPlaneTop ? kPlaneClasses : kPixelClasses)) return rc;
    SEGK_REQUIRE(values && indices, SEGK_EINVAL, "top_logits: null output");
    SEGK_REQUIRE(aligned16(values) && aligned16(indices) && aligned16(lse), SEGK_EALIGN, "top_logits: outputs must be 16-byte aligned");
    const bool wide = planes(C, inner), pix = wide || few(outer, C, inner);
    const Pixels px = pixels(outer, C, inner, ld, k, aligned16(logits));
    SEGK_REQUIRE(!pix || px.blocks < (1ll << 31), SEGK_ESHAPE, "top_logits: too many positions");
    SEGK_USE_DEVICE(dev);
    hipStream_t st = (hipStream_t)stream;
    SEGK_DISPATCH_DTYPE(dtype, T, {
        const float inv_t = 1.f / temperature;
        if (pix) {
            by_launches(px.outer, px.blocks_each * 256ll, [&](int64_t o, int64_t n) {
                const dim3 grid((unsigned)(n * px.blocks_each));
                const int64_t kept = o * k * px.inner;
                if (wide) {
                    auto kernel = k <= 2 ? top_planes_kernel<T, 2> : top_planes_kernel<T, kPlaneTop>;
                    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, (const T*)logits + o * ld, ld, px.inner, (int)C, (int)k, inv_t, (T*)values + kept,
                                       indices + kept, advance(lse, o * px.inner), px.blocks_each);
                } else {
                    class_tier(C, px.vp, [&](auto cm, auto vp) {
                        hipLaunchKernelGGL((top_pixels_kernel<T, cm(), vp()>), grid, dim3(256), 0, st, (const T*)logits + o * ld, ld, px.s_c, px.s_p, px.inner, (int)C,
                                           (int)k, inv_t, (T*)values + kept, indices + kept, px.ts_c, px.ts_p, advance(lse, o * px.inner), px.blocks_each);
                    });
                }
            });
        } else {
            row_tier<T, true>(logits, outer, ld, C, k, [&](auto nt, auto nch) {
                constexpr int r = rows_per_group(nt(), nch());
                by_launches(outer, nt(), [&](int64_t o, int64_t n) {
                    hipLaunchKernelGGL((top_rows_kernel<T, nt(), nch()>), dim3((unsigned)((n + r - 1) / r)), dim3(nt(), r), 0, st, (const T*)logits + o * ld, n, ld, (int)C,
                                       (int)k, inv_t, (T*)values + o * k, indices + o * k, advance(lse, o));
                });
            });
        }
    });
    SEGK_LAUNCH_CHECK();
    return SEGK_OK;
}

// Workgroups that share a row (1: the row kernels).  The row kernels keep a row of up to 16384 pieces in registers and then read it
// once; longer ones they read twice, and a few of them leave most of the chip idle.  Whole call for 131000 fp32 classes, shared / not,
// forward and with gradient: 1 row 13/20, 17/34 us; 64 rows 17/30, 34/76; 128 rows 22/32, 54/82; 256 rows 35/35, 94/94.  For 131000
// bf16 classes, in registers of one CU: 16 rows 14/18, 20/27; 128 rows 18/21, 35/31.  Below 8192 pieces one CU is as fast: 32000 fp32
// classes, 16 rows 13/11, 19/15.
static int shares_of(int64_t rows, int64_t C, int dtype) {
    const int64_t pieces = C * (int64_t)esize(dtype) / 16;
    if (rows > (pieces > 16384 ? 128 : 16) || pieces <= 8192) return 1;
    int64_t s = pieces / 1024;
    if (s > 1024 / rows) s = 1024 / rows;
    return (int)(s > kShares ? kShares : s < 1 ? 1 : s);
}
static constexpr int kCollect = 256, kFinal = 16384;      // from more than kFinal values on the final sum has two levels
static_assert(kCollect == kCountBlocks);
// floats of the workspace: partial counts, level-1 sums, then one sum per row or workgroup
static size_t distill_partials(int64_t outer, int64_t C, int64_t inner) {
    if (!planes(C, inner) && !few(outer, C, inner)) return (size_t)outer * (outer <= 128 ? 1 + 2 * kShares + kRowFloats : 1) + 1;
    return (size_t)(pixels(outer, C, inner, C * inner, 1, false).blocks);      // an upper bound for either vector width
}
extern "C" size_t segk_distill_workspace(int64_t outer, int64_t C, int64_t inner) {
    if (outer <= 0 || C <= 0 || inner <= 0) return 0;
    return 4 * (kCountBlocks + kCollect + distill_partials(outer, C, inner));
}

extern "C" int segk_distill(const void* logits, int dtype, int64_t outer, int64_t C, int64_t inner, int64_t ld, const void* values, int values_dtype,
                            const void* indices, int index_bytes, const float* teacher_lse, int64_t k, float temperature, float weight, int flags,
                            const float* upstream, float* loss, float* position_loss, void* dlogits, int64_t ld_d, void* workspace,
                            size_t workspace_bytes, int dev, void* stream) {
    if (const int rc = check_logits("distill", logits, dtype, outer, C, inner, ld, k, temperature, kPlaneClasses)) return rc;
    const bool mean = flags & 1, each = flags & 2, skip = flags & 4;
    SEGK_REQUIRE(values && indices && workspace, SEGK_EINVAL, "distill: null pointer");
    SEGK_REQUIRE(values_dtype == SEGK_F32 || values_dtype == SEGK_BF16, SEGK_EINVAL, "distill: unknown dtype %d of the values", values_dtype);
    SEGK_REQUIRE(index_bytes == 4 || index_bytes == 8, SEGK_EINVAL, "distill: indices have 4 or 8 bytes, not %d", index_bytes);
    SEGK_REQUIRE(loss || position_loss || dlogits, SEGK_EINVAL, "distill: no output");
    SEGK_REQUIRE(!(mean && each), SEGK_EINVAL, "distill: a mean has one upstream gradient, not one for each position");
    SEGK_REQUIRE(!(each || skip) || (upstream && dlogits), SEGK_EINVAL, "distill: this flag needs an upstream gradient and dlogits");
    SEGK_REQUIRE(!(skip && (each || loss || position_loss)), SEGK_EINVAL, "distill: only the gradient of a scalar can be left as it is");
    SEGK_REQUIRE(!dlogits || (ld_d >= C * inner && reinterpret_cast<uintptr_t>(dlogits) % esize(dtype) == 0), SEGK_ESHAPE, "distill: bad dlogits");
    SEGK_REQUIRE(workspace_bytes >= segk_distill_workspace(outer, C, inner), SEGK_EWORKSPACE, "distill: workspace too small");
    SEGK_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 4 == 0, SEGK_EALIGN, "distill: workspace must be 4-byte aligned");
    const bool wide = planes(C, inner), pix = wide || few(outer, C, inner);
    const bool vec = aligned16(logits) && (!dlogits || (aligned16(dlogits) && ld_d % 4 == 0)) && aligned16(values) && aligned16(indices) && aligned16(teacher_lse);
    const Pixels px = pixels(outer, C, inner, ld, k, vec);
    SEGK_REQUIRE(!pix || px.blocks < (1ll << 31), SEGK_ESHAPE, "distill: too many positions");
    SEGK_USE_DEVICE(dev);
    hipStream_t st = (hipStream_t)stream;
    int* counts = static_cast<int*>(workspace);
    float* collected = reinterpret_cast<float*>(counts + kCountBlocks);
    float* partial = collected + kCollect;
    DistillArgs a = {};
    a.z = logits; a.ld = ld; a.V = (int)C; a.k = (int)k;
    a.t = values; a.t_bf16 = values_dtype == SEGK_BF16; a.idx = indices; a.idx64 = index_bytes == 8; a.tlse = teacher_lse;
    a.T = temperature; a.invT = 1.f / temperature; a.weight = weight;
    a.upstream = upstream; a.up_each = each; a.skip_if_one = skip;
    a.counts = mean ? counts : nullptr;
    a.dz = dlogits; a.ld_d = ld_d;
    if (pix) {
        a.inner = px.inner; a.s_c = px.s_c; a.s_p = px.s_p; a.ts_c = px.ts_c; a.ts_p = px.ts_p;
        a.d_c = px.s_c; a.d_p = inner == 1 ? ld_d : 1;
        a.row_loss = position_loss; a.partial = loss ? partial : nullptr;
    } else {
        a.inner = 1; a.ts_c = 1; a.ts_p = k;
        a.row_loss = position_loss ? position_loss : partial;
    }
    while ((1 << a.log_kp) < k) ++a.log_kp;
    // up to 1024 entries (16 loads of a wave, all in flight) are counted where the number is needed instead of in a launch of their own
    if (mean && inner == 1 && outer << a.log_kp <= 1024) a.count_here = (int)outer;
    if (mean && !dlogits && !pix) a.count_losses = outer > kFinal ? 2 : 1;
    if (a.count_losses) a.count_here = 0;
    if (mean && !skip && !a.count_here && !a.count_losses) {
        if (inner == 1) {
            hipLaunchKernelGGL(distill_count_rows_kernel, dim3(kCountBlocks), dim3(256), 0, st, a, outer, a.log_kp, counts);
        } else {
            if (!a.idx64 && inner % 4 == 0 && aligned16(indices)) hipLaunchKernelGGL(distill_count_planes4_kernel, dim3(kCountBlocks), dim3(1024), 0, st, a, outer * inner, counts);
            else if (a.idx64) hipLaunchKernelGGL(distill_count_planes_kernel<int64_t>, dim3(kCountBlocks), dim3(1024), 0, st, a, outer * inner, counts);
            else hipLaunchKernelGGL(distill_count_planes_kernel<int32_t>, dim3(kCountBlocks), dim3(1024), 0, st, a, outer * inner, counts);
        }
        SEGK_LAUNCH_CHECK();
    }
    // the arguments from image or row o on (rows counted in place need no second launch)
    auto from = [&](int64_t o) {
        DistillArgs b = a;
        const int64_t positions = o * a.inner;
        b.z = advance(a.z, o * ld, esize(dtype));
        b.t = advance(a.t, positions * k, esize(values_dtype));
        b.idx = advance(a.idx, positions * k, (size_t)index_bytes);
        b.tlse = advance(a.tlse, positions);
        if (each) b.upstream = advance(a.upstream, positions);
        b.row_loss = advance(a.row_loss, positions);
        b.partial = advance(a.partial, o * px.blocks_each);
        if (dlogits) b.dz = const_cast<void*>(advance(a.dz, o * ld_d, esize(dtype)));
        return b;
    };
    int64_t n = pix ? px.blocks : outer;
    bool summed = false;
    SEGK_DISPATCH_DTYPE(dtype, T, {
        if (pix) {
            by_launches(px.outer, px.blocks_each * 256ll, [&](int64_t o, int64_t images) {
                const DistillArgs b = from(o);
                const dim3 grid((unsigned)(images * px.blocks_each));
                if (wide) {
                    auto kernel = dlogits ? distill_planes_kernel<T, true> : distill_planes_kernel<T, false>;
                    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, b, px.blocks_each);
                } else {
                    class_tier(C, px.vp, [&](auto cm, auto vp) {
                        if (dlogits) hipLaunchKernelGGL((distill_pixels_kernel<T, cm(), vp(), true>), grid, dim3(256), 0, st, b, px.blocks_each);
                        else hipLaunchKernelGGL((distill_pixels_kernel<T, cm(), vp(), false>), grid, dim3(256), 0, st, b, px.blocks_each);
                    });
                }
            });
        } else if (const int shares = shares_of(outer, C, dtype); shares > 1) {
            float *parts = partial + outer, *joined = parts + outer * 2 * kShares;
            int* rows_done = loss ? reinterpret_cast<int*>(joined + outer * kRowFloats) : nullptr;
            summed = loss;
            hipLaunchKernelGGL((distill_share_kernel<T>), dim3(shares, (unsigned)outer), dim3(256), 0, st, a, parts, rows_done);
            hipLaunchKernelGGL((distill_join_kernel<T>), dim3((unsigned)outer), dim3(64), 0, st, a, parts, shares, dlogits ? joined : nullptr, rows_done, loss);
            if (dlogits) hipLaunchKernelGGL((distill_share_grad_kernel<T>), dim3(shares, (unsigned)outer), dim3(256), 0, st, a, joined);
        } else {
            row_tier<T, false>(logits, outer, ld, C, k, [&](auto nt, auto nch) {
                by_launches(outer, nt(), [&](int64_t o, int64_t rows) {
                    const DistillArgs b = from(o);
                    if (dlogits) hipLaunchKernelGGL((distill_rows_kernel<T, nt(), nch(), true>), dim3((unsigned)rows), dim3(nt()), 0, st, b);
                    else hipLaunchKernelGGL((distill_rows_kernel<T, nt(), nch(), false>), dim3((unsigned)rows), dim3(nt()), 0, st, b);
                });
            });
        }
    });
    SEGK_LAUNCH_CHECK();
    if (loss && !summed) {
        const float* v = pix ? partial : a.row_loss;
        if (n > kFinal) {
            hipLaunchKernelGGL(distill_collect_kernel, dim3(kCollect), dim3(1024), 0, st, a, v, n, collected);
            SEGK_LAUNCH_CHECK();
            v = collected;
            n = kCollect;
        }
        hipLaunchKernelGGL(distill_finalize_kernel, dim3(1), dim3(1024), 0, st, a, v, (int)n, loss);
        SEGK_LAUNCH_CHECK();
    }
    return SEGK_OK;
}
