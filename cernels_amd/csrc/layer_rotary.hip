// Rotary positions: the pair (a, b) of frequency f at position p becomes (a c - b s, b c + a s), c = scale cos(p f), s = scale sin(p f);
// the rest of the head is copied. Backward turns by -p f. With `append` the keys go to their slots in the pages, the values with them.
//
// Bound by memory: every element is read and written once. One workgroup has one token, so that a token's angles are computed once,
// in 64 bits up to the fraction of a turn (fp32 would lose 0.06 rad at position 2^20), and shared by its heads through LDS; the first
// vectors of the heads are loaded before the angles are needed.
// Measured: 8192 tokens of 72 heads of 64 in bf16 29 us each way, 5.2 TB/s, the rate of a large copy; 8 tokens of 36 heads of 128
// 3.9 us, append of 64 single tokens 5.9 us (latency); append of 4574 tokens of 40 heads of 128 22 us, 4.2 TB/s.
#include "layer_step.h"

namespace cmoe {

constexpr int kRotThreads = 256;


template <class T, int V>
__device__ __forceinline__ u32x4 unit_load(const typename T::raw* p) {
    if constexpr (V == 1) return u32x4{__float_as_uint(T::get(*p)), 0, 0, 0};
    else return load_vec<T>(p);
}
template <class T, int V>
__device__ __forceinline__ void unit_store(typename T::raw* p, const float* f) {
    if constexpr (V == 1) *p = T::put(f[0]);
    else store_vec<T>(p, T::pack(f));
}
template <class T, int V>
__device__ __forceinline__ void unit_unpack(const u32x4& r, float* f) {
    if constexpr (V == 1) f[0] = __uint_as_float(r[0]);
    else T::unpack(r, f);
}

// Where unit u of a head starts: its first element, and whether it holds pairs. Half layout: V pairs, the second elements `pairs`
// further; interleaved: V / 2 pairs (one pair, as two elements, for V = 1).
template <int V, bool INTER>
__device__ __forceinline__ int unit_at(int u, int pairs, bool& turned) {
    constexpr int W = INTER && V == 1 ? 2 : V;
    const int pu = INTER ? 2 * pairs / W : pairs / V;
    turned = u < pu;
    return turned ? u * W : 2 * pairs + (u - pu) * V;
}
template <int V, bool INTER>
__host__ __device__ __forceinline__ int units_of(int dim, int pairs) {
    constexpr int W = INTER && V == 1 ? 2 : V;
    return (INTER ? 2 * pairs / W : pairs / V) + (dim - 2 * pairs) / V;
}

template <class T, int V, bool INTER, bool APPEND>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotaryParams p) {
    typedef typename T::raw raw;
    extern __shared__ float2 turn[];  // [pairs] cos and sin, scaled
    const int t = blockIdx.x;
    const int units = units_of<V, INTER>(p.dim, p.pairs);
    const int hq = p.q.p ? p.q.heads : 0, hk = p.k.p ? p.k.heads : 0;
    const int vu = p.dim / V;  // a head's vectors of v
    const int n_turn = (hq + hk) * units, n = n_turn + (APPEND ? hk * vu : 0);

    // Work item w of the token: the units of q's heads, then of k's, then (append) v's vectors.
    auto item = [&](int w, int& head, int& u) {
        const bool is_v = APPEND && w >= n_turn;
        const int r = is_v ? w - n_turn : w, per = is_v ? vu : units;
        head = r / per;
        u = r - head * per;
        return is_v;
    };
    auto load = [&](int w, u32x4& a, u32x4& b) {
        int head, u;
        const bool is_v = item(w, head, u), is_q = !is_v && head < hq;
        const void* base = is_v ? p.v.p : is_q ? p.q.p : p.k.p;
        const long long st = is_v ? p.v.token : is_q ? p.q.token : p.k.token;
        const long long sh = is_v ? p.v.head : is_q ? p.q.head : p.k.head;
        const raw* x = static_cast<const raw*>(base) + t * st + (is_v || is_q ? head : head - hq) * sh;
        bool turned = false;
        const int at = is_v ? u * V : unit_at<V, INTER>(u, p.pairs, turned);
        a = unit_load<T, V>(x + at);
        if (turned && (!INTER || V == 1)) b = unit_load<T, V>(x + at + (INTER ? 1 : p.pairs));
    };

    long long pos;
    int page = -1, slot = 0;
    if constexpr (APPEND) {
        const int b = step_sequence(p.step, t);
        if (b >= p.step.seqs) return;  // behind the last sequence: its rows stay as they are
        int first, count;
        step_tokens(p.step, b, first, count);
        const int at = p.step.lengths[b] - count + (t - first);
        pos = at;
        if (at >= 0) {
            const int blk = at / p.step.page_size;
            page = step_page(p.step, b, blk);
            slot = at - blk * p.step.page_size;
        }
    } else {
        pos = p.position_i64 ? static_cast<const long long*>(p.positions)[t] : static_cast<const int*>(p.positions)[t];
    }
    u32x4 a{}, b{};
    int w = threadIdx.x;
    if (w < n) load(w, a, b);
    for (int i = threadIdx.x; i < p.pairs; i += kRotThreads) {
        const double f = p.freq_f64 ? static_cast<const double*>(p.inv_freq)[i] : (double)static_cast<const float*>(p.inv_freq)[i];
        const double turns = (double)pos * f * 0.15915494309189533577;  // 1 / (2 pi)
        const float part = (float)(turns - rint(turns));                // of a turn, in [-1/2, 1/2]
        float s, c;
        sincospif(2.0f * part, &s, &c);
        turn[i] = make_float2(c * p.scale, (p.backward ? -s : s) * p.scale);
    }
    __syncthreads();
    for (; w < n;) {
        int head, u;
        const bool is_v = item(w, head, u), is_q = !is_v && head < hq;
        bool turned = false;
        const int at = is_v ? u * V : unit_at<V, INTER>(u, p.pairs, turned);
        raw* out;
        if (is_q) {
            out = static_cast<raw*>(p.q_out) + ((long long)t * hq + head) * p.dim;
        } else if constexpr (APPEND) {
            void* base = is_v ? p.v_pages.p : p.k_pages.p;
            const long long sp = is_v ? p.v_pages.page : p.k_pages.page, ss = is_v ? p.v_pages.slot : p.k_pages.slot;
            const long long sh = is_v ? p.v_pages.head : p.k_pages.head;
            out = static_cast<raw*>(base) + page * sp + slot * ss + (is_v ? head : head - hq) * sh;
        } else {
            out = static_cast<raw*>(p.k_out) + ((long long)t * hk + head - hq) * p.dim;
        }
        const bool write = !APPEND || is_q || page >= 0;
        const u32x4 whole = a;
        float x[8], y[8];
        unit_unpack<T, V>(a, x);
        if (turned && (!INTER || V == 1)) unit_unpack<T, V>(b, y);
        const int next = w + kRotThreads;
        if (next < n) load(next, a, b);
        if (!turned) {
            if constexpr (V == 1) {
                if (write) *(out + at) = T::put(x[0]);
            } else if (write) {
                store_vec<T>(out + at, whole);
            }
        } else if constexpr (INTER && V > 1) {
            float z[8];
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float2 cs = turn[at / 2 + i];
                z[2 * i] = x[2 * i] * cs.x - x[2 * i + 1] * cs.y;
                z[2 * i + 1] = x[2 * i + 1] * cs.x + x[2 * i] * cs.y;
            }
            if (write) unit_store<T, V>(out + at, z);
        } else {
            float z[8], o[8];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 cs = turn[INTER ? at / 2 : at + i];
                z[i] = x[i] * cs.x - y[i] * cs.y;
                o[i] = y[i] * cs.x + x[i] * cs.y;
            }
            if (write) {
                unit_store<T, V>(out + at, z);
                unit_store<T, V>(out + at + (INTER ? 1 : p.pairs), o);
            }
        }
        w = next;
    }
}

template <class T, int V, bool INTER>
static void rotary_v(const RotaryParams& p, hipStream_t s) {
    const size_t lds = sizeof(float2) * (size_t)(p.pairs > 0 ? p.pairs : 1);
    if constexpr (sizeof(typename T::raw) == 2) {
        if (p.append) {
            hipLaunchKernelGGL((rotary_kernel<T, V, INTER, true>), dim3(p.tokens), dim3(kRotThreads), lds, s, p);
            return;
        }
    }
    hipLaunchKernelGGL((rotary_kernel<T, V, INTER, false>), dim3(p.tokens), dim3(kRotThreads), lds, s, p);
}

// Whole vectors where the turned part, its halves and the rest divide into them; single elements otherwise.
template <class T>
static void rotary_t(const RotaryParams& p, hipStream_t s) {
    constexpr int V = T::kVec;
    const bool whole = (p.interleaved ? 2 * p.pairs % V == 0 : p.pairs % V == 0) && (p.dim - 2 * p.pairs) % V == 0 && p.dim % V == 0;
    if (p.interleaved) {
        if (whole) rotary_v<T, V, true>(p, s);
        else rotary_v<T, 1, true>(p, s);
    } else {
        if (whole) rotary_v<T, V, false>(p, s);
        else rotary_v<T, 1, false>(p, s);
    }
}

hipError_t launch_rotary(const RotaryParams& p, hipStream_t s) {
    if (p.dtype == kDtBf16) rotary_t<TypeBf16>(p, s);
    else if (p.dtype == kDtF16) rotary_t<TypeF16>(p, s);
    else rotary_t<TypeF32>(p, s);
    return hipGetLastError();
}

}  // namespace cmoe
