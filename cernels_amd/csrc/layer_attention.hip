// Attention of a step's new tokens over a paged cache. Query head h of token i (position p) of sequence b sees keys j <= p of its
// sequence, with a window also j > p - window:
//   o = sum_j e_j v_j / (sum_j e_j + e_sink), e_j = exp(scale q k_j - M), e_sink = exp(sink_h - M)
// in one pass over the keys with a running M and sum (fp32). A row is one (token, query head of a key head's group); rows of one key
// head share its keys, so they are the columns of one matrix product S^T = K Q^T.
//
// Why S^T: in the matrix instructions' result layout a lane then owns one row of the softmax (a column here), and the values that it
// holds are exactly the elements that it has to supply as the second operand of O^T = V^T P^T, once the keys of a tile are numbered in
// the order in which the result registers hold them. The probabilities go from one product to the next without leaving the lane.
//
// Rows in sets of 16 (few) or 128 (tiles): see the two kernels. Launches: one or both of them, and a join where keys were split.
//
// M is raised only where a new score passes it by kSlack (a factor 2^kSlack in the exponentials, exact in fp32 and harmless in the
// 16-bit probabilities), so that most tiles need neither a reduction over lanes nor a rescaling of O.
#include "layer_step.h"
#include "moe_tile.h"

#include <type_traits>

namespace cmoe {

typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kSlack = 8.0f;
constexpr float kNone = -__builtin_inff();

struct MathBf16 {
    typedef TypeBf16 T;
    static constexpr uint32_t kExponent = 0x7f80;
    static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mma16_short(s16x4 a, u32x2 b, f32x4 c) {  // 16 x 16 x 16
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) { return cvt_bf16x2(a, b); }
    static __device__ __forceinline__ float add2(uint32_t pair, float sum) {  // sum + both values of the pair
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
    }
};
struct MathF16 {
    typedef TypeF16 T;
    static constexpr uint32_t kExponent = 0x7c00;
    static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mma16_short(s16x4 a, u32x2 b, f32x4 c) {
        typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) { return cvt_f16x2(a, b); }
    static __device__ __forceinline__ float add2(uint32_t pair, float sum) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), __builtin_bit_cast(f16x2, 0x3c003c00u), sum, false);
    }
};

// Values that are not finite, in tiles of which some rows do not see some keys: a key that a row does not see has probability 0 there,
// but 0 times an infinity is a NaN. Such tiles (the last ones of a row's keys and the first ones of its window) are looked through, and
// from one that holds such a value on, a wave goes through its keys one by one, adding to each row what it sees and nothing else.
template <class M>
__device__ __forceinline__ uint32_t not_finite(u32x4 v) {  // one of the two top bits is set if a value's exponent is all ones
    constexpr uint32_t kStep = (0x8000u - M::kExponent) * 0x10001u, kMask = M::kExponent * 0x10001u;
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) odd |= (v[i] & kMask) + kStep;  // carries into a half's own top bit, no further
    return odd & 0x80008000u;
}
// Part of q k: 8 elements.
template <class T>
__device__ __forceinline__ float dot8(const u32x4& a, const u32x4& b, float sum) {
    float x[8], y[8];
    T::unpack(a, x);
    T::unpack(b, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(x[i], y[i], sum);
    return sum;
}
// Raises the maximum to x; what the sums so far, and x, then weigh.
__device__ __forceinline__ void raise_to(float x, float& m, float& f, float& e) {
    const float m1 = fmaxf(m, x);
    f = m1 == kNone ? 1.0f : __builtin_amdgcn_exp2f(m - m1);
    e = __builtin_amdgcn_exp2f(x - (m1 == kNone ? 0.0f : m1));
    m = m1;
}

// What a launch works on beside the call's own parameters.
struct AttentionPlan {
    int splits;    // parts that a sequence's keys may be cut in; above 1 workgroups write partial results
    int few_rows;  // sequences of at most this many rows take the few-rows kernel, the others the tile kernel; -1: all take the former
    float* part;   // [tokens * heads][splits][dim] unnormalised O, then [tokens * heads][splits][2] M and sum
};

__device__ __forceinline__ float2* plan_stats(const AttentionPlan& a, const AttentionParams& p) {
    return reinterpret_cast<float2*>(a.part + (long long)p.step.tokens * p.q.heads * a.splits * p.dim);
}

// Part number `i` of `n` of the keys [begin, end): equal parts, whole multiples of `unit`.
__device__ __forceinline__ void split_range(int begin, int end, int i, int n, int unit, int& lo, int& hi) {
    const int keys = end > begin ? end - begin : 0;
    const int per = max(((keys + n - 1) / n + unit - 1) / unit * unit, unit);
    const long long at = (long long)per * i;
    lo = at < keys ? begin + (int)at : end;
    hi = end - lo < per ? end : lo + per;
}

constexpr int kTileRows = 128;  // of the tile kernel
// Workgroups that are on the card at once: as the rings in LDS (few rows) and the registers (tiles) let on a CU.
constexpr int card_slots(bool few, int dim) { return few ? 65536 / dim : dim <= 128 ? 512 : 256; }
constexpr int kLeastKeys = 256;

// A workgroup's work: one tile of rows of a sequence (all its rows: the few-rows kernel), and one of `parts` parts of their keys.
struct Piece {
    int b, first, count, rows, tile, split, parts;
};
// Piece number `i`, asked by whole waves; false behind the last one. Only the device knows the sequences' lengths, so the pieces are
// listed by every workgroup for itself: a sequence's keys are cut so that the card's slots get equal shares of all of them, of 256
// keys at least (128: 17 users with sinks 27.9 us, 256: 23.1), and workgroups without a piece, which hold a slot for some
// microseconds, are at most one per tile (a grid of 16 splits for each of 64 sequences of 4096 keys: 136 us, the list: 111).
template <bool FEW, int D>
__device__ __forceinline__ bool find_piece(const AttentionParams& p, const AttentionPlan& plan, int i, Piece& t) {
    constexpr int kSlots = card_slots(FEW, D);
    const int lane = threadIdx.x & 63, group = p.q.heads / p.kv_heads;
    int first = 0, count = 0, rows = 0, tiles = 0, keys = 0;
    auto look = [&](int b) __attribute__((always_inline)) {
        first = count = tiles = keys = 0;
        if (b < p.step.seqs) {
            step_tokens(p.step, b, first, count);
            const int length = p.step.lengths[b];
            keys = min(max(length, 0), p.step.blocks * p.step.page_size);
            if (p.window > 0) keys = (int)min((long long)keys, (long long)p.window + count);
        }
        rows = count * group;
        const bool few = plan.few_rows < 0 || rows <= plan.few_rows;
        tiles = rows == 0 || few != FEW ? 0 : FEW ? 1 : (rows + kTileRows - 1) / kTileRows;
    };
    auto cut = [&](float share) __attribute__((always_inline)) {
        return min(max((int)ceilf((float)keys / share - 0.05f), 1), plan.splits);  // a twentieth over a share is no part of its own
    };
    if (p.step.seqs == 1) {  // no list: the same in all lanes
        look(0);
        t.parts = cut(fmaxf((float)tiles * (float)keys * (float)p.kv_heads * (1.0f / kSlots), (float)kLeastKeys));
        if (tiles * p.kv_heads * t.parts > kSlots && t.parts > 1) t.parts = max(kSlots / (tiles * p.kv_heads), 1);
        t.b = 0, t.first = first, t.count = count, t.rows = rows;
        const int from_end = tiles * t.parts - 1 - i;
        t.tile = from_end / t.parts;
        t.split = from_end - t.tile * t.parts;
        return from_end >= 0;
    }
    look(lane);
    float share = 3.0e9f;
    if (plan.splits > 1) {
        float sum = 0.0f;
        for (int b = lane;;) {
            sum += (float)tiles * (float)keys;
            b += 64;
            if (b - lane >= p.step.seqs) break;
            look(b);
        }
        share = fmaxf(wave_sum(sum) * (float)p.kv_heads * (1.0f / kSlots), (float)kLeastKeys);
        if (p.step.seqs > 64) {
            look(lane);
        } else {  // equal sequences cut just over their share would be more pieces than slots, all of one size: a round more
            const float pieces = wave_sum((float)(tiles * cut(share))) * (float)p.kv_heads;
            if (pieces > kSlots) share *= fminf(pieces * (1.0f / kSlots), 1.5f);
        }
    }
    for (int b0 = 0; b0 < p.step.seqs; b0 += 64) {
        if (b0) look(b0 + lane);
        const int parts = cut(share);
        int sum = tiles * parts;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned long long has = __ballot(sum > i);
        if (has) {
            const int l = __builtin_ctzll(has);
            t.b = b0 + l;
            t.first = __builtin_amdgcn_readlane(first, l);
            t.count = __builtin_amdgcn_readlane(count, l);
            t.rows = __builtin_amdgcn_readlane(rows, l);
            t.parts = __builtin_amdgcn_readlane(parts, l);
            const int from_end = __builtin_amdgcn_readlane(sum, l) - 1 - i;
            t.tile = from_end / t.parts;  // the last tile first: it sees the most keys
            t.split = from_end - t.tile * t.parts;
            return true;
        }
        i -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// The splits that a sequence's parts leave unused saw nothing; the join reads that. Written by the workgroup of the first part.
__device__ __forceinline__ void unused_splits(const AttentionParams& p, const AttentionPlan& plan, const Piece& t, long long row) {
    if (t.split == 0)
        for (int i = t.parts; i < plan.splits; ++i) plan_stats(plan, p)[row * plan.splits + i] = make_float2(kNone, 0.0f);
}

// One row's result: normalised into the output, or as a partial result of its split.
template <class M>
__device__ __forceinline__ float row_scale(const AttentionParams& p, int head, float m, float l) {
    if (p.sinks) l += __builtin_amdgcn_exp2f(p.sinks[head] * kLog2e - (m == kNone ? 0.0f : m));
    return l > 0.0f || l != l ? 1.0f / l : 0.0f;  // a row that sees nothing is 0
}

__device__ const __align__(16) uint32_t kZeros[4] = {0, 0, 0, 0};

// ---- few rows: single tokens and short chunks ---------------------------------------------------------------------------------
// Bound by the stream of keys and values. The four waves of a workgroup share out its keys, and each runs alone: 16 keys at a time
// come through a ring of two stages of its own in LDS, sent there without passing through registers, so that a ring of 16 KB per
// wave (heads of 128) is on its way at any time however few registers the products leave (keys and values taken straight into
// operand registers: 64 users with mixed lengths 102 us, rings 87). Keys are read as operands as they lie, values turned
// (ds_read_b64_tr_b16: 4 keys of one column per lane).
// Measured: 64 users of 4096 keys (32 query, 4 key heads of 128) 111 us with the join, 4.8 TB/s, where a large copy moves 5.2; 64
// users with 195 to 8193 keys 70 us, 3.8 TB/s; one user behind 2168 keys 9 us and the join's 4.5, bound by latency.
constexpr int kFewWaves = 4;
constexpr int kFewKeys = 16;

template <class M, int D>
__global__ __launch_bounds__(64 * kFewWaves) void attend_few_kernel(AttentionParams p, AttentionPlan plan) {
    typedef typename M::T T;
    typedef typename T::raw raw;
    typedef __attribute__((address_space(3))) const u32x4* lds_vec;
    typedef __attribute__((address_space(3))) s16x4* lds_turned;
    constexpr int DS = D / 32;                                // steps of the first product
    constexpr int DJ = D / 16;                                // 16-row tiles of the second one's result
    constexpr int CH = D / 8, kMask = CH < 16 ? CH - 1 : 15;  // 16-byte vectors of a row; those that the banks' order permutes
    constexpr int kRowsPer = 64 / CH, kCopies = kFewKeys / kRowsPer;
    constexpr int kBytes = kFewKeys * D * 2, kWaveBytes = 4 * kBytes;  // a stage's keys; a wave's ring: [2][K | V]
    extern __shared__ __align__(1024) unsigned char lds[];             // the rings; afterwards the waves' results
    __shared__ float2 lds_ml[kFewWaves][16];
    float* lds_o = reinterpret_cast<float*>(lds);  // [wave][16 * D]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int kh = blockIdx.x % p.kv_heads, group = p.q.heads / p.kv_heads;
    Piece t;
    if (!find_piece<true, D>(p, plan, blockIdx.x / p.kv_heads, t)) return;
    const int b = t.b, first = t.first, count = t.count, rows = t.rows, split = t.split;
    const int length = p.step.lengths[b], page_size = p.step.page_size;
    const char* kbase = static_cast<const char*>(p.k.p) + 2 * kh * p.k.head;
    const char* vbase = static_cast<const char*>(p.v.p) + 2 * kh * p.v.head;
    const auto* table = (const __attribute__((address_space(4))) int32_t*)(p.step.table + b * p.step.table_stride);
    const float c = p.scale * kLog2e;
    // from a copy's first row: this lane's row, and the vector that belongs at its place
    const int crow = lane / CH, cpos = lane % CH;
    uint32_t koff[kCopies], voff[kCopies];
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
        const int r = i * kRowsPer + crow;
        koff[i] = (uint32_t)(2 * crow * p.k.slot) + 16 * (cpos ^ (r & kMask));
        voff[i] = (uint32_t)(2 * crow * p.v.slot) + 16 * (cpos ^ (2 * r & kMask));
    }
    const uint32_t ring = lds_u32(lds) + wave * kWaveBytes;
    uint32_t kaddr[DS], vaddr[DJ];
#pragma unroll
    for (int d = 0; d < DS; ++d) kaddr[d] = ring + col * D * 2 + 16 * ((4 * d + g) ^ (col & kMask));
#pragma unroll
    for (int j = 0; j < DJ; ++j) {
        const int r = 4 * g + col / 4, chunk = 2 * j + ((lane & 3) >> 1);
        vaddr[j] = ring + kBytes + r * D * 2 + 16 * (chunk ^ (2 * r & kMask)) + 8 * (lane & 1);
    }

    for (int r0 = 0; r0 < rows; r0 += 16) {
        // rows r0 .. r0 + 15: this lane's, its query and the keys that they see
        u32x4 q[DS];
        const int row = r0 + col, last = min(r0 + 15, rows - 1), before = length - count;
        const bool live = row < rows;
        const int token = live ? row / group : 0, head = kh * group + (live ? row - token * group : 0);
        const raw* src = static_cast<const raw*>(p.q.p) + (first + token) * p.q.token + head * p.q.head;
#pragma unroll
        for (int s = 0; s < DS; ++s) q[s] = live ? load_vec<T>(src + 8 * (g + 4 * s)) : u32x4{};
        // positions grow with the row: the first row sees the fewest later keys, the last one the fewest earlier ones
        auto low = [&](int tok) __attribute__((always_inline)) { return p.window > 0 && before + tok - p.window + 1 > 0 ? before + tok - p.window + 1 : 0; };
        const int hi = live ? before + token + 1 : 0, lo = low(token);
        const int all_hi = before + r0 / group + 1, least_lo = low(r0 / group), all_lo = low(last / group);
        const int most_hi = min(max(before + last / group + 1, 0), p.step.blocks * page_size);
        int begin, end;
        split_range(least_lo & ~(kFewKeys - 1), most_hi, split, t.parts, kFewKeys * kFewWaves, begin, end);
        // this wave's quarter of them; a stage lies inside one page (pages hold a multiple of 16 slots), and the pages are walked along
        // the table without a division
        const int quarter = (end - begin + kFewKeys * kFewWaves - 1) / (kFewKeys * kFewWaves) * kFewKeys;
        const int w_begin = min(begin + wave * quarter, end), w_end = min(w_begin + quarter, end);
        struct Run {
            int key, blk, slot, page;
        };
        auto look = [&](Run& r) __attribute__((always_inline)) {
            const int page = r.key < w_end ? table[r.blk] : -1;  // w_end is at most the table's
            r.page = (unsigned)page < (unsigned)p.step.pages ? page : -1;
        };
        auto walk = [&](Run& r) __attribute__((always_inline)) {
            r.key += kFewKeys;
            r.slot += kFewKeys;
            if (r.slot >= page_size) r.slot -= page_size, ++r.blk;
            look(r);
        };
        auto copy_keys = [&](const Run& r, int stage) __attribute__((always_inline)) {
            const char* kp = kbase + 2 * ((long long)max(r.page, 0) * p.k.page + r.slot * p.k.slot);  // without a page: page 0, dropped below
#pragma unroll
            for (int i = 0; i < kCopies; ++i) dma16_at(kp + 2 * i * kRowsPer * p.k.slot, koff[i], ring + stage * 2 * kBytes + i * 1024);
        };
        auto copy_values = [&](const Run& r, int stage) __attribute__((always_inline)) {
            const char* vp = vbase + 2 * ((long long)max(r.page, 0) * p.v.page + r.slot * p.v.slot);
            const uint32_t dst = ring + stage * 2 * kBytes + kBytes;
            if (r.page >= 0 && r.key >= least_lo && r.key + kFewKeys <= w_end) {
#pragma unroll
                for (int i = 0; i < kCopies; ++i) dma16_at(vp + 2 * i * kRowsPer * p.v.slot, voff[i], dst + i * 1024);
            } else {  // values that nobody sees may be anything, and 0 times anything is not always 0
#pragma unroll
                for (int i = 0; i < kCopies; ++i) {
                    const int key = r.key + i * kRowsPer + crow;
                    const bool zero = r.page < 0 || key >= w_end || key < least_lo;
                    dma16(zero ? reinterpret_cast<const char*>(kZeros) : vp + 2 * i * kRowsPer * p.v.slot + voff[i], dst + i * 1024);
                }
            }
        };

        float m = kNone, l = 0.0f;
        f32x4 o[DJ];
#pragma unroll
        for (int j = 0; j < DJ; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        // One stage: 16 keys from k0, `left` keys to come with them. K of the stage after next is sent once this stage's is read, V
        // likewise; a wait leaves in flight what was sent after what it waits for.
        auto step = [&](int k0, int left, bool bad, const Run& next, auto which) __attribute__((always_inline)) {
            constexpr int kBase = decltype(which)::value * 2 * kBytes;
            if (left > kFewKeys) wait_vmcnt<3 * kCopies>();
            else wait_vmcnt<kCopies>();
            f32x4 s{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < DS; ++d) {
                const u32x4 a = *(lds_vec)(kaddr[d] + kBase);
                s = M::mma16(a, q[d], s);
            }
            if ((k0 < all_lo || k0 + kFewKeys > all_hi)) {  // some row does not see some key
                wait_vmcnt<0>();
                uint32_t odd = 0;
#pragma unroll
                for (int at = 0; at < kBytes; at += 1024) odd |= not_finite<M>(*(lds_vec)(ring + kBase + kBytes + at + 16 * lane));
                if (__ballot(odd != 0) != 0) return true;
            }
            const bool sent = left > 2 * kFewKeys;
            if (sent) copy_keys(next, decltype(which)::value);
            const bool whole = !bad && k0 >= all_lo && k0 + kFewKeys <= all_hi && left >= kFewKeys;
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = k0 + 4 * g + i;
                    const bool sees = !bad & (key < hi) & (key >= lo) & (key < w_end);
                    s[i] = sees ? s[i] : kNone;
                }
            }
            float t = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])) * c;
            if (__ballot(t > m + kSlack) != 0) {
                t = fmaxf(t, __shfl_xor(t, 16));
                t = fmaxf(t, __shfl_xor(t, 32));
                const float m1 = fmaxf(m, t);
                const float f = m1 == kNone ? 1.0f : __builtin_amdgcn_exp2f(m - m1);
                m = m1;
                l *= f;
#pragma unroll
                for (int j = 0; j < DJ; ++j) o[j] *= f;
            }
            const float sub = m == kNone ? 0.0f : m;
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -sub));
            // rounded to the values' type for the product; the sum takes the rounded ones too (as in the tile kernel)
            const u32x2 pr{M::pack2(e[0], e[1]), M::pack2(e[2], e[3])};
            l = M::add2(pr[1], M::add2(pr[0], l));
            if (sent) wait_vmcnt<3 * kCopies>();
            else if (left > kFewKeys) wait_vmcnt<2 * kCopies>();
            else wait_vmcnt<0>();
#pragma unroll
            for (int j = 0; j < DJ; ++j) {
                const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_turned)(vaddr[j] + kBase));
                o[j] = M::mma16_short(a, pr, o[j]);
            }
            if (sent) copy_values(next, decltype(which)::value);
            return false;
        };
        int resume = w_end;  // the keys from here on are gone through one by one
        __syncthreads();  // the rings held the waves' results of the rows before
        if (w_begin < w_end) {
            Run r{w_begin, w_begin / page_size, 0, -1};
            r.slot = w_begin - r.blk * page_size;
            look(r);
            copy_keys(r, 0);
            copy_values(r, 0);
            bool bad0 = r.page < 0, bad1 = true;
            walk(r);
            if (r.key < w_end) {
                copy_keys(r, 1);
                copy_values(r, 1);
                bad1 = r.page < 0;
                walk(r);
            }
            wait_all_loads();  // the queries too: the waits in the loop count copies only
            for (int k0 = w_begin; k0 < w_end; k0 += 2 * kFewKeys) {
                if (step(k0, w_end - k0, bad0, r, std::integral_constant<int, 0>{})) {
                    resume = k0;
                    break;
                }
                bad0 = r.page < 0;
                walk(r);
                if (k0 + kFewKeys >= w_end) break;
                if (step(k0 + kFewKeys, w_end - k0 - kFewKeys, bad1, r, std::integral_constant<int, 1>{})) {
                    resume = k0 + kFewKeys;
                    break;
                }
                bad1 = r.page < 0;
                walk(r);
            }
        }
#pragma unroll 1
        for (int key = resume; key < w_end; ++key) {
            Run at{key, key / page_size, 0, -1};
            at.slot = key - at.blk * page_size;
            look(at);
            if (at.page < 0) continue;
            const char* kp = kbase + 2 * ((long long)at.page * p.k.page + at.slot * p.k.slot);
            const char* vp = vbase + 2 * ((long long)at.page * p.v.page + at.slot * p.v.slot);
            float x = 0.0f;
#pragma unroll
            for (int d = 0; d < DS; ++d) x = dot8<T>(*reinterpret_cast<const u32x4*>(kp + 64 * d + 16 * g), q[d], x);
            x += __shfl_xor(x, 16);
            x = (x + __shfl_xor(x, 32)) * c;
            if (key < hi && key >= lo) {
                float f, e;
                raise_to(x, m, f, e);
                l = l * f + (g == 0 ? e : 0.0f);
#pragma unroll
                for (int j = 0; j < DJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[j][i] = o[j][i] * f + e * T::get(reinterpret_cast<const raw*>(vp)[16 * j + 4 * g + i]);
            }
        }
        // the waves' results
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        __syncthreads();
        if (g == 0) lds_ml[wave][col] = make_float2(m, l);
#pragma unroll
        for (int j = 0; j < DJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 16 * j + 4 * g + r;
                lds_o[wave * 16 * D + col * D + (d ^ (col & 7) * 4)] = o[j][r];
            }
        __syncthreads();
        constexpr int kPer = 64 * kFewWaves / 16;  // threads that share a row
        const int my = threadIdx.x / kPer, part = threadIdx.x % kPer, mine = r0 + my;
        if (mine < rows) {
            float mx = kNone, sum = 0.0f, f[kFewWaves];
#pragma unroll
            for (int w = 0; w < kFewWaves; ++w) mx = fmaxf(mx, lds_ml[w][my].x);
#pragma unroll
            for (int w = 0; w < kFewWaves; ++w) {
                f[w] = lds_ml[w][my].x == kNone ? 0.0f : __builtin_amdgcn_exp2f(lds_ml[w][my].x - mx);
                sum += f[w] * lds_ml[w][my].y;
            }
            const int token = mine / group, head = kh * group + mine - token * group;
            const long long at = (long long)(first + token) * p.q.heads + head;
            const float k = plan.splits > 1 ? 1.0f : row_scale<M>(p, head, mx, sum);
            for (int d = 4 * part; d < D; d += 4 * kPer) {
                f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kFewWaves; ++w)
                    v += f[w] * *reinterpret_cast<const f32x4*>(&lds_o[w * 16 * D + my * D + (d ^ (my & 7) * 4)]);
                if (plan.splits > 1)
                    *reinterpret_cast<f32x4*>(plan.part + (at * plan.splits + split) * D + d) = v;
                else
                    *reinterpret_cast<u32x2*>(static_cast<raw*>(p.out) + at * D + d) =
                        u32x2{M::pack2(v[0] * k, v[1] * k), M::pack2(v[2] * k, v[3] * k)};
            }
            if (plan.splits > 1 && part == 0) {
                plan_stats(plan, p)[at * plan.splits + split] = make_float2(mx, sum);
                unused_splits(p, plan, t, at);
            }
        }
    }
}

// ---- many rows: chunks and prompts --------------------------------------------------------------------------------------------
// Bound by the matrix instructions. Four waves of 32 rows each share tiles of keys and values in LDS, the next tile on its way there
// while one is worked on. K's 16-byte vectors are read as operands as they are; V's operands are columns, which LDS hands out turned
// (ds_read_b64_tr_b16: 4 keys of one column per lane). Two workgroups to a CU (256 registers a lane): the one's exponentials run
// beside the other's products, and within a wave beside the next tile's first product.
// Measured: 509 tokens behind 32003 keys (32 query, 4 key heads of 128) 275 us and the join's 10, 0.98 PFLOP/s in the kernel, where a
// large bf16 product reaches 1.38; three prompts of 5092 tokens 107 us, 0.70 PFLOP/s with its ramp and tail. Sequences of 17 to 32
// rows are better off here than as two sets of the kernel above: 64 users of 4 tokens behind 2048 keys 68 us, there 109.
constexpr int kTileWaves = 4;
static_assert(kTileRows == 32 * kTileWaves, "a wave has 32 rows");

template <int D>
struct TileSize {
    static constexpr int kKeys = D <= 128 ? 64 : 32;
    static constexpr int kBytes = kKeys * D * 2;
};

template <class M, int D>
__global__ __launch_bounds__(64 * kTileWaves, D <= 128 ? 2 : 1) void attend_tile_kernel(AttentionParams p, AttentionPlan plan) {
    typedef typename M::T T;
    typedef typename T::raw raw;
    typedef __attribute__((address_space(3))) const u32x4* lds_vec;
    typedef __attribute__((address_space(3))) s16x4* lds_turned;
    constexpr int KT = TileSize<D>::kKeys, kBytes = TileSize<D>::kBytes;
    constexpr int CH = D / 8, kMask = CH < 16 ? CH - 1 : 15;  // 16-byte vectors of a row; those that the banks' order permutes
    constexpr int kRowsPer = 64 / CH;                         // rows that one copy instruction of a wave moves
    constexpr int kRun = KT / kTileWaves, kCopies = kRun / kRowsPer;  // keys that a wave copies, all of one page
    constexpr int DS = D / 16, DT = D / 32, KU = KT / 32;
    extern __shared__ __align__(1024) unsigned char lds[];  // [2][K | V]
    __shared__ __align__(16) uint32_t missing[4][kTileWaves];  // per tile and wave's run of keys: without a page
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    const int kh = blockIdx.x % p.kv_heads, group = p.q.heads / p.kv_heads;
    Piece t;
    if (!find_piece<false, D>(p, plan, blockIdx.x / p.kv_heads, t)) return;
    const int row0 = t.tile * kTileRows;
    const int length = p.step.lengths[t.b];
    const char* kbase = static_cast<const char*>(p.k.p) + 2 * kh * p.k.head;
    const char* vbase = static_cast<const char*>(p.v.p) + 2 * kh * p.v.head;
    const float c = p.scale * kLog2e;

    const int row = row0 + 32 * wave + col;
    const bool live = row < t.rows;
    const int token = live ? row / group : 0, head = kh * group + (live ? row - token * group : 0);
    u32x4 q[DS];
    {
        const raw* src = static_cast<const raw*>(p.q.p) + (t.first + token) * p.q.token + head * p.q.head;
#pragma unroll
        for (int s = 0; s < DS; ++s) q[s] = live ? load_vec<T>(src + 16 * s + 8 * h) : u32x4{};
    }
    // keys that the row, the wave's rows and the tile's rows see; positions grow with the row
    const int page_size = p.step.page_size, cap = p.step.blocks * page_size, before = length - t.count;
    auto low = [&](int tok) __attribute__((always_inline)) { return p.window > 0 && before + tok - p.window + 1 > 0 ? before + tok - p.window + 1 : 0; };
    const int hi = live ? before + token + 1 : 0, lo = low(token);
    const int last_row = min(row0 + kTileRows, t.rows) - 1;
    const int w_first = min(row0 + 32 * wave, last_row) / group, w_last = min(row0 + 32 * wave + 31, last_row) / group;
    bool idle = row0 + 32 * wave >= t.rows;
    const int w_hi = before + w_last + 1, w_all_hi = before + w_first + 1, w_lo = low(w_first), w_all_lo = low(w_last);
    const int tile_lo = low(row0 / group);
    int begin, end;
    split_range(tile_lo / KT * KT, min(before + last_row / group + 1, cap), t.split, t.parts, KT, begin, end);

    // This wave's run of the next tile to copy: its page and first slot, walked along the table without a division. Keys are sent one
    // tile ahead of the values, so the values' run is the one that the keys had before.
    struct Run {
        int key, blk, slot, page;
    };
    const auto* table = (const __attribute__((address_space(4))) int32_t*)(p.step.table + t.b * p.step.table_stride);
    auto page_of = [&](int key, int block) __attribute__((always_inline)) {
        const int page = key < end ? table[block] : -1;  // end is at most the table's
        return (unsigned)page < (unsigned)p.step.pages ? page : -1;
    };
    Run kr, vr;
    kr.key = begin + kRun * wave;
    kr.blk = kr.key / page_size;
    kr.slot = kr.key - kr.blk * page_size;
    kr.page = page_of(kr.key, kr.blk);
    vr = kr;
    const int crow = lane / CH, cpos = lane % CH;
    uint32_t koff[kCopies], voff[kCopies];  // from a copy's first row: this lane's row, and the vector that belongs at its place
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
        const int r = wave * kRun + i * kRowsPer + crow;
        koff[i] = (uint32_t)(2 * crow * p.k.slot) + 16 * (cpos ^ (r & kMask));
        voff[i] = (uint32_t)(2 * crow * p.v.slot) + 16 * (cpos ^ (2 * r & kMask));
    }
    const uint32_t mine = lds_u32(lds) + wave * kRun * D * 2;
    auto copy_keys = [&](int tile) __attribute__((always_inline)) {
        const uint32_t dst = mine + (tile & 1) * 2 * kBytes;
        const long long at = kr.page < 0 ? 0 : kr.page;  // keys without a page are read from page 0 and dropped below
        const char* kp = kbase + 2 * (at * p.k.page + kr.slot * p.k.slot);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) dma16_at(kp + 2 * i * kRowsPer * p.k.slot, koff[i], dst + i * 1024);
        if (lane == 0) missing[tile & 3][wave] = kr.page < 0;
        kr.key += KT;
        kr.slot += KT;
        while (kr.slot >= page_size) kr.slot -= page_size, ++kr.blk;
        kr.page = page_of(kr.key, kr.blk);
    };
    auto copy_values = [&](int tile, const Run& r) __attribute__((always_inline)) {
        const uint32_t dst = mine + (tile & 1) * 2 * kBytes + kBytes;
        const long long at = r.page < 0 ? 0 : r.page;
        const char* vp = vbase + 2 * (at * p.v.page + r.slot * p.v.slot);
        if (r.page >= 0 && r.key >= tile_lo && r.key + kRun <= end) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) dma16_at(vp + 2 * i * kRowsPer * p.v.slot, voff[i], dst + i * 1024);
        } else {  // values that nobody sees may be anything, and 0 times anything is not always 0
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int key = r.key + i * kRowsPer + crow;
                const bool zero = r.page < 0 || key >= end || key < tile_lo;
                dma16(zero ? reinterpret_cast<const char*>(kZeros) : vp + 2 * i * kRowsPer * p.v.slot + voff[i], dst + i * 1024);
            }
        }
    };

    float m = kNone, l = 0.0f;
    f32x16 o[DT];
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[j][i] = 0.0f;
    // Where this lane reads its operands: K's row `col`, vector 2 d + h; V's 4 keys x 16 columns for each 16 lanes, of which lane n
    // addresses 4 columns of key n / 4 and gets column n.
    uint32_t kaddr[DS], vaddr[DT];
#pragma unroll
    for (int d = 0; d < DS; ++d) kaddr[d] = lds_u32(lds) + col * D * 2 + 16 * ((2 * d + h) ^ (col & kMask));
#pragma unroll
    for (int j = 0; j < DT; ++j) {
        const int r = 4 * h + (lane & 15) / 4, chunk = 4 * j + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        vaddr[j] = lds_u32(lds) + kBytes + r * D * 2 + 16 * (chunk ^ (2 * r & kMask)) + 8 * (lane & 1);
    }

    f32x16 s[KU];
    auto scores = [&](auto which) __attribute__((always_inline)) {  // of the tile whose keys lie in buffer `which`
        constexpr int kBase = decltype(which)::value * 2 * kBytes;
        f32x16 r[KU];
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) r[u][i] = 0.0f;
#pragma unroll
        for (int d = 0; d < DS; ++d)
#pragma unroll
            for (int u = 0; u < KU; ++u) r[u] = M::mma32(*(lds_vec)(kaddr[d] + kBase + u * 32 * D * 2), q[d], r[u]);
#pragma unroll
        for (int u = 0; u < KU; ++u) s[u] = r[u];
    };
    // The running maximum over s, the scores of the tile at k0; hidden ones become -inf.
    auto raise = [&](int k0, int tile) __attribute__((always_inline)) {
        uint32_t gone[kTileWaves], any = 0;
#pragma unroll
        for (int w = 0; w < kTileWaves; ++w) any |= gone[w] = missing[tile & 3][w];
        const bool whole = k0 >= w_all_lo && k0 + KT <= w_all_hi && k0 + KT <= end && !__builtin_amdgcn_readfirstlane(any);
        if (!whole) {
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 32 * u + 8 * (i >> 2) + 4 * h + (i & 3), key = k0 + r;
                    const bool sees = (key < hi) & (key >= lo) & (key < end) & (gone[(32 * u + 8 * (i >> 2)) / kRun] == 0);
                    s[u][i] = sees ? s[u][i] : kNone;
                }
        }
        float x = s[0][0];
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) x = fmaxf(x, s[u][i]);
        x *= c;
        if (__ballot(x > m + kSlack) != 0) {
            const float m1 = fmaxf(m, max_halves(x));
            const float f = m1 == kNone ? 1.0f : __builtin_amdgcn_exp2f(m - m1);
            m = m1;
            l *= f;
#pragma unroll
            for (int j = 0; j < DT; ++j) o[j] *= f;
        }
    };
    // The probabilities of s and their product with the values in buffer `which`; between them the next tile's scores.
    auto weigh = [&](auto which, auto more) __attribute__((always_inline)) {
        constexpr int kBase = decltype(which)::value * 2 * kBytes;
        const float sub = m == kNone ? 0.0f : m;
        f32x16 t[KU];
#pragma unroll
        for (int u = 0; u < KU; ++u) t[u] = s[u];
        if constexpr (decltype(more)::value) scores(std::integral_constant<int, 1 - decltype(which)::value>{});
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[u][8 * k + i], c, -sub));
                // Rounded to the values' type for the product. The sum takes the rounded ones too: what rounding does to a row's
                // weights as a whole then cancels.
                const u32x4 pr{M::pack2(e[0], e[1]), M::pack2(e[2], e[3]), M::pack2(e[4], e[5]), M::pack2(e[6], e[7])};
#pragma unroll
                for (int i = 0; i < 4; ++i) l = M::add2(pr[i], l);
#pragma unroll
                for (int j = 0; j < DT; ++j) {
                    u32x4 a;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_turned)(vaddr[j] + kBase + (32 * u + 16 * k + 8 * i) * D * 2));
                        const u32x2 w = __builtin_bit_cast(u32x2, v);
                        a[2 * i] = w[0], a[2 * i + 1] = w[1];
                    }
                    o[j] = M::mma32(a, pr, o[j]);
                }
            }
        // The order: six operands of the first product ahead, then each of its instructions with two exponentials and their company; the
        // second product's operands one instruction ahead. Left to itself 297 us (509 tokens behind 32003), in this order 264; operands
        // read just ahead of each instruction 360.
        if constexpr (decltype(more)::value && D <= 128) {
            __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
            for (int i = 0; i < KU * DS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
#pragma unroll
            for (int i = 0; i < 2 * KU * DT; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
        }
    };
    auto odd_values = [&](auto which) __attribute__((always_inline)) {
        uint32_t odd = 0;
#pragma unroll 4
        for (int at = 16 * lane; at < kBytes; at += 1024) odd |= not_finite<M>(*(lds_vec)(lds_u32(lds) + decltype(which)::value * 2 * kBytes + kBytes + at));
        return __ballot(odd != 0) != 0;
    };
    int resume = end;  // the keys from here on are gone through one by one
    // One tile. What was sent a tile ago has landed (its values, the next one's keys); the keys of the tile after that and the next
    // values are sent into the buffers that no wave reads any more.
    auto step = [&](int k0, int tile, auto which) __attribute__((always_inline)) {
        const bool more = k0 + KT < end;
        wait_vmcnt<0>();
        __syncthreads();
        if (more) {
            const Run next = kr;
            if (k0 + 2 * KT < end) copy_keys(tile + 2);
            copy_values(tile + 1, vr);
            vr = next;
        }
        if (idle) return;
        if ((k0 < w_all_lo || k0 + KT > w_all_hi) && odd_values(which)) {
            resume = k0;
            idle = true;  // of the tiles; the wave still sends its copies
            return;
        }
        raise(k0, tile);
        if (more) weigh(which, std::true_type{});
        else weigh(which, std::false_type{});
    };
    if (begin < end) {
        copy_keys(0);
        copy_values(0, vr);
        vr = kr;
        wait_all_loads();  // the queries too: a wait for them inside the loop would be one for the copies sent there
        __syncthreads();
        if (begin + KT < end) copy_keys(1);
        if (!idle) scores(std::integral_constant<int, 0>{});
    }
    for (int k0 = begin, tile = 0; k0 < end; k0 += 2 * KT, tile += 2) {
        step(k0, tile, std::integral_constant<int, 0>{});
        if (k0 + KT >= end) break;
        step(k0 + KT, tile + 1, std::integral_constant<int, 1>{});
    }
    auto halves = [](float v) __attribute__((always_inline)) {
        uint32_t a = __float_as_uint(v), b = a;
        swap_halves(a, b);
        return __uint_as_float(a) + __uint_as_float(b);
    };
#pragma unroll 1
    for (int key = resume; key < end; ++key) {
        const int at = key / page_size, page = page_of(key, at), in = key - at * page_size;
        if (page < 0) continue;
        const char* kp = kbase + 2 * ((long long)page * p.k.page + in * p.k.slot);
        const char* vp = vbase + 2 * ((long long)page * p.v.page + in * p.v.slot);
        float x = 0.0f;
#pragma unroll
        for (int d = 0; d < DS; ++d) x = dot8<T>(*reinterpret_cast<const u32x4*>(kp + 32 * d + 16 * h), q[d], x);
        x = halves(x) * c;
        if (key < hi && key >= lo) {
            float f, e;
            raise_to(x, m, f, e);
            l = l * f + (h == 0 ? e : 0.0f);
#pragma unroll
            for (int j = 0; j < DT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const raw* v = reinterpret_cast<const raw*>(vp) + 32 * j + 8 * i + 4 * h;
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[j][4 * i + r] = o[j][4 * i + r] * f + e * T::get(v[r]);
                }
        }
    }
    l = halves(l);
    if (!live) return;
    const long long at = (long long)(t.first + token) * p.q.heads + head;
    if (plan.splits > 1) {
        if (h == 0) {
            plan_stats(plan, p)[at * plan.splits + t.split] = make_float2(m, l);
            unused_splits(p, plan, t, at);
        }
        float* part = plan.part + (at * plan.splits + t.split) * D;
        if (l == 0.0f) return;  // nobody reads it
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(part + 32 * j + 8 * i + 4 * h) =
                    f32x4{o[j][4 * i], o[j][4 * i + 1], o[j][4 * i + 2], o[j][4 * i + 3]};
        return;
    }
    const float k = row_scale<M>(p, head, m, l);
    raw* out = static_cast<raw*>(p.out) + at * D;
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<u32x2*>(out + 32 * j + 8 * i + 4 * h) = u32x2{M::pack2(o[j][4 * i] * k, o[j][4 * i + 1] * k),
                                                                            M::pack2(o[j][4 * i + 2] * k, o[j][4 * i + 3] * k)};
}

// ---- joining the splits ---------------------------------------------------------------------------------------------------------
// One wave per row: the splits' M and sums by lane, then the O of those that saw a key, in their order.
template <class M, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(AttentionParams p, AttentionPlan plan) {
    typedef typename M::T::raw raw;
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= (long long)p.step.tokens * p.q.heads) return;
    const int token = (int)at / p.q.heads, head = (int)at - token * p.q.heads;  // fewer than 2^31 rows
    // what the row needs is on its way before it is known to be one: every row has its place in the workspace
    const float2* st = plan_stats(plan, p) + at * plan.splits;
    const float2 mine = lane < plan.splits ? st[lane] : make_float2(kNone, 0.0f);
    const float* part = plan.part + at * plan.splits * D + E * lane;
    float v[4][E];
    auto fetch = [&](int i, int n) __attribute__((always_inline)) {  // four splits at a time
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) v[u][e] = part[(long long)min(i + u, n - 1) * D + e];
    };
    fetch(0, plan.splits);
    if (step_sequence(p.step, token) >= p.step.seqs) return;
    const float mx = wave_max(mine.y == 0.0f ? kNone : mine.x);
    const float f = mine.y == 0.0f || mine.x == kNone ? 0.0f : __builtin_amdgcn_exp2f(mine.x - mx);
    const float sum = wave_sum(f * mine.y);
    const unsigned long long used = __ballot(mine.y != 0.0f);
    const int n = used ? 64 - __builtin_clzll(used) : 0;  // splits that saw nothing come last, as a rule
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    for (int i = 0; i < n; i += 4) {
        if (i) fetch(i, n);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float w = i + u < n ? __shfl(f, i + u) : 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = w != 0.0f ? o[e] + w * v[u][e] : o[e];  // what a split that saw nothing holds is never read as a number
        }
    }
    const float k = row_scale<M>(p, head, mx, sum);
    raw* out = static_cast<raw*>(p.out) + at * D + E * lane;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = M::T::put(o[e] * k);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------

bool attention_dim_ok(int dim) { return dim == 64 || dim == 128 || dim == 256; }

constexpr int kMostSplits = 64;  // the join kernel holds a split's statistics per lane
// Rows of a sequence that take the few-rows kernel: one set of 16.
constexpr int kFewRows = 16;

struct Forms {
    bool few, tile;
    int splits;
    long long few_pieces, tile_pieces;  // at most, for each key head
};

static Forms attention_forms(const AttentionParams& p) {
    const int group = p.q.heads / p.kv_heads, seqs = p.step.seqs;
    const long long rows = (long long)p.step.tokens * group;
    const int even = (p.step.tokens + seqs - 1) / seqs;  // some sequence has at least that many tokens
    const long long most = (long long)(p.max_new > p.step.tokens ? p.step.tokens : p.max_new < even ? even : p.max_new) * group;
    Forms f{};
    f.tile = most > kFewRows;
    // as many tokens as the longest sequence's for each: all are alike, and one kernel takes them all, whatever they hold in truth
    f.few = !f.tile || most * seqs != rows;
    // many-row sequences: at most one partly filled tile each
    const long long part = rows / (kFewRows + 1);
    const long long tiles = f.tile ? (rows + kTileRows - 1) / kTileRows + (seqs == 1 ? 0 : seqs < part ? seqs : part) : 0;
    // Room for partial results: one sequence's tiles are cut alike; among several a long one is cut in more parts than the average, up
    // to twice as many (tiles) or eight times (sets of 16 rows).
    const long long groups = (f.tile ? tiles : seqs) * p.kv_heads;
    const long long slots = card_slots(!f.tile, p.dim);
    const long long want = seqs == 1 ? slots / groups : ((f.tile ? 2 : 8) * slots + groups / 2) / groups;
    const long long useful = ((long long)p.step.blocks * p.step.page_size + kLeastKeys - 1) / kLeastKeys;
    const long long n = want < useful ? want : useful;
    f.splits = (int)(n < 1 ? 1 : n > kMostSplits ? kMostSplits : n);
    auto cuts = [&](bool few) { return f.splits > 1 ? (card_slots(few, p.dim) + p.kv_heads - 1) / p.kv_heads : 0; };
    f.few_pieces = f.few ? seqs + cuts(true) : 0;
    f.tile_pieces = f.tile ? tiles + cuts(false) : 0;
    return f;
}

size_t attention_workspace_bytes(const AttentionParams& p) {
    const Forms f = attention_forms(p);
    if (f.splits <= 1) return 16;
    return (size_t)p.step.tokens * p.q.heads * f.splits * (p.dim + 2) * sizeof(float);
}

template <class M, int D>
static hipError_t attention_d(const AttentionParams& p, hipStream_t s) {
    const Forms f = attention_forms(p);
    const AttentionPlan plan{f.splits, f.tile ? (f.few ? kFewRows : 0) : -1, p.ws};
    if (f.tile)
        hipLaunchKernelGGL((attend_tile_kernel<M, D>), dim3((unsigned)(f.tile_pieces * p.kv_heads)), dim3(64 * kTileWaves),
                           4 * TileSize<D>::kBytes, s, p, plan);
    if (f.few)  // the rings; the results of 16 rows take half of them
        hipLaunchKernelGGL((attend_few_kernel<M, D>), dim3((unsigned)(f.few_pieces * p.kv_heads)), dim3(64 * kFewWaves),
                           kFewWaves * 4 * kFewKeys * D * 2, s, p, plan);
    if (f.splits > 1) {
        const long long rows = (long long)p.step.tokens * p.q.heads;
        hipLaunchKernelGGL((attend_join_kernel<M, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, p, plan);
    }
    return hipGetLastError();
}

template <class M>
static hipError_t attention_m(const AttentionParams& p, hipStream_t s) {
    if (p.dim == 64) return attention_d<M, 64>(p, s);
    if (p.dim == 128) return attention_d<M, 128>(p, s);
    return attention_d<M, 256>(p, s);
}

hipError_t launch_attention(const AttentionParams& p, hipStream_t s) {
    return p.dtype == kDtBf16 ? attention_m<MathBf16>(p, s) : attention_m<MathF16>(p, s);
}

}  // namespace cmoe
