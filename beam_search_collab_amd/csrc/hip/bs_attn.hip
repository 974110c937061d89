// Attention over packed sequences (include/bs_embed.h).
//
// One pass over the keys with the running maximum and sum of the softmax.  The rows of a tile are
// (query token, head of the group) pairs of one sequence and key/value head, so grouped heads share the
// keys in LDS whatever the number of tokens.  Scores are formed transposed, S^T = K Q^T: a lane then holds
// one row of the tile and its scores stay in its registers -- maximum, sum and rescaling are per lane
// (plus one exchange between the wave's halves), and the weights are the second operand of O^T = V^T P^T
// as they stand, once V's keys are taken in the order in which the result of the first product has them.
#include "bs_embed.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {
using namespace bse;

template <typename T>
struct Mma;
template <>
struct Mma<f16> {
    __device__ static f32x16 go(Vec<f16, 8> a, Vec<f16, 8> b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mma<bf16> {
    __device__ static f32x16 go(Vec<bf16, 8> a, Vec<bf16, 8> b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

constexpr int BN = 64;  // keys of a tile
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;
constexpr float NONE = -INFINITY;

// n / d for n < 2^31 and one d: floor(n m / 2^(31 + s)) with s = ceil(log2 d), m = ceil(2^(31 + s) / d) < 2^32.  (m d -
// 2^(31 + s) < d <= 2^s, so the quotient is off by less than n / 2^31 / d and never reaches the next integer.)
struct Divisor {
    uint32_t m, s;
    Divisor(uint32_t d = 1) : m(0), s(0) {
        while ((1ull << s) < d) ++s;
        m = static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d);
    }
    __device__ uint32_t quotient(uint32_t n) const { return __umulhi(n << 1, m) >> s; }
};

struct Params {
    bs_attention_args a;
    uint32_t group;    // heads per key/value head
    Divisor by_group, by_kv;
    uint32_t splits;   // pieces of the keys; > 1: parts go to the workspace
    uint32_t piece;    // keys of a piece, a multiple of BN
    float* part_out;   // splits x q_tokens x heads x head_dim: sums of p v, unscaled
    float2* part_stat; // splits x q_tokens x heads: maximum (in units of log2) and sum
};

struct Sequence {
    uint32_t q0, nq, k0, nk;
};

__device__ inline Sequence sequence(const bs_attention_args& a, uint32_t s) {
    Sequence r{0, a.q_tokens, 0, a.k_tokens};
    if (a.q_offsets) {  // whatever the offsets hold, the tokens lie inside the buffers
        const uint32_t b = static_cast<uint32_t>(max(a.q_offsets[s], 0)), e = static_cast<uint32_t>(max(a.q_offsets[s + 1], 0));
        r.q0 = min(b, a.q_tokens);
        r.nq = min(e, a.q_tokens) - min(r.q0, min(e, a.q_tokens));
    }
    if (a.k_offsets) {
        const uint32_t b = static_cast<uint32_t>(max(a.k_offsets[s], 0)), e = static_cast<uint32_t>(max(a.k_offsets[s + 1], 0));
        r.k0 = min(b, a.k_tokens);
        r.nk = min(e, a.k_tokens) - min(r.k0, min(e, a.k_tokens));
    }
    return Sequence{uniform(r.q0), uniform(r.nq), uniform(r.k0), uniform(r.nk)};
}

// The tiles of all sequences are counted without a list of them: sequence s gets the tile numbers from
// offset(s) * group / rows + s on.  That leaves room for its own tiles and at most one unused number per sequence.
__device__ inline uint64_t first_tile(const int32_t* off, uint32_t s, uint32_t group, uint32_t rows) {
    return static_cast<uint64_t>(max(off[s], 0)) * group / rows + s;
}
// The last of n ascending values that `below` holds for (the first one if for none), the same for all lanes: 256
// candidates a step, so one round of loads for up to 256 sequences.
template <typename F>
__device__ inline uint32_t last_below(uint32_t n, F below) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 255) / 256, at = lo + (threadIdx.x & 63) * step;
        int k = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = at + i * 64 * step;
            k += __popcll(__ballot(x < hi && below(x)));
        }
        lo += (k > 0 ? k - 1 : 0) * step;
        hi = min(lo + step, hi);
    }
    return uniform(lo);
}
// the sequence that a tile number belongs to
__device__ inline uint32_t find(const int32_t* off, uint32_t n, uint64_t tile, uint32_t group, uint32_t rows) {
    return last_below(n, [&](uint32_t s) { return first_tile(off, s, group, rows) <= tile; });
}
// the last sequence that starts at or before the token
__device__ inline uint32_t holder(const int32_t* off, uint32_t n, uint32_t tok) {
    return last_below(n, [&](uint32_t s) { return static_cast<uint32_t>(max(off[s], 0)) <= tok; });
}

// chunk c of 16 bytes in row r of an LDS tile of S bytes per row (64, 128 or 256).  16 rows read at one
// chunk (a quarter wave's operand of K) lie in 16 different chunks of the 256 bytes that all banks span,
// and the 4 rows x 64 bytes of a transposed read of V in 4 different quarters of them.
template <int S>
__device__ inline int place(int r, int c) {
    const int f = S == 256 ? ((r & 3) << 2 | ((r >> 2) & 3)) : S == 128 ? (((r >> 1) & 1) << 2 | ((r >> 2) & 3)) : ((r >> 2) & 3);
    return r * S + ((c ^ f) << 4);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ inline s16x4 read_transposed(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4*>(
        reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)p)));
}

// waits until all but the wave's N youngest moves to LDS are done, and its reads of LDS
template <int N>
__device__ inline void landed() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);  // vmcnt(N) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// the same for all of them, and meets the workgroup's other waves
__device__ inline void meet() {
    landed<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// meets the workgroup's other waves with this wave's reads and writes of LDS done; moves stay on their way
__device__ inline void settle() {
    landed<63>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

__device__ inline uint32_t keys_of(const bs_attention_args& a, const Sequence& sq, uint32_t t) {  // visible keys of query t
    const int64_t e = a.causal ? min(static_cast<int64_t>(sq.nk), static_cast<int64_t>(sq.nk) - sq.nq + t + 1) : static_cast<int64_t>(sq.nk);
    return static_cast<uint32_t>(e < 0 ? 0 : e);
}

// the values of lanes l and l + 32, to both
__device__ inline float2 halves(float v) {
    const uint32_t b = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The maximum that keeps NaN: three operands an instruction, and none of them is multiplied by 1 first, as fmaxf has it
// done to quiet NaN.
__device__ inline float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

template <int DP>
constexpr int ROW = DP <= 32 ? 64 : DP <= 64 ? 128 : 256;  // bytes of a key or value in LDS

// The rows of one wave: 32 of them, lanes l and l + 32 (half h) hold row l.
template <typename T, int DP>
struct Rows {
    static constexpr int S = ROW<DP>;
    Vec<T, 8> q[DP / 16];
    f32x16 o[DP / 32];
    float top, sum;  // what the weights are taken against, in units of log2, and their sum over this half's keys
    // The weights are rounded to the values' type for their product (the sum takes them as they are), since two 16-bit
    // products a score, of a weight's upper and lower bits, would double the matrix work.  float16 has nothing below 2^-24,
    // where many small weights beside a large one would be lost: there the largest weight stands at 2^7, and may grow to
    // 2^11 before the row is rescaled.  (Its largest value is 2^16; the rest is for scores so large that float32 has them
    // in steps of up to 4.)  A weight is then off by 2^-32 of the row's largest at most.
    // A weight is exp2(score * scale - top) with one rounding, while the top is rounded too: where float32 has steps of 8 and
    // more, the largest weight could be anything up to 2^4 and more off.  Rows so `far` have scores and top rounded alike
    // and subtracted first, in the branch that rescales (in a branch of its own: documents 1124 us instead of 1006).
    bool far;  // some row of the wave is
    __device__ static bool is_far(float top) { return fabsf(top) >= 0x1p26f && fabsf(top) < INFINITY; }
    static constexpr float ROOM = std::is_same<T, f16>::value ? 7.0f : 0.0f, LAG = std::is_same<T, f16>::value ? 4.0f : 8.0f;

    __device__ void clear() {
        top = NONE;
        sum = 0.0f;
        far = false;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[d] = f32x16{};
    }
    // scores are taken times a scale > 0: a negative one turns the sign of the query, for 0 the query is 0
    __device__ void load(const T* p, uint32_t head_dim, float scale, int h) {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const uint32_t d = s * 16 + h * 8;
            q[s] = Vec<T, 8>{};
            if (d < head_dim && scale != 0.0f) q[s] = *reinterpret_cast<const Vec<T, 8>*>(p + d);
            if (scale < 0.0f) q[s] = -q[s];
        }
    }
    __device__ bool odd() const {  // some result is not finite
        uint32_t most = 0;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) most = max(most, __float_as_uint(o[d][r]) & 0x7FFFFFFFu);
        return most >= 0x7F800000u;
    }
    // What a step over KB x 32 keys holds besides.  Operands are read a part ahead of their products: parts of 32
    // elements of the keys, then of 16 of the values, the first of which comes in under the exponentials.  (Two
    // ahead cost 16 registers more and spill at 128.)
    static constexpr int PARTS = DP / 32;
    template <int KB>
    struct Work {
        f32x16 z[KB];  // scores; register r of block b: key b * 32 + r % 4 + 8 (r / 4) + 4 h
        Vec<T, 8> w[2 * KB], k[2][2][KB], v[2][PARTS];
    };
    template <int KB>
    __device__ static void read_keys(Work<KB>& x, const char* tk, int i, int lane) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int b = 0; b < KB; ++b)
                x.k[i & 1][s][b] = *reinterpret_cast<const Vec<T, 8>*>(tk + place<S>(b * 32 + (lane & 31), i * 4 + s * 2 + (lane >> 5)));
    }
    template <int KB>
    __device__ static void read_values(Work<KB>& x, const char* tv, int s, int lane) {
#pragma unroll
        for (int d = 0; d < PARTS; ++d) {
            // lanes 16g .. 16g + 15 read 4 keys x 16 elements and get an element's 4 keys each
            const int key = s * 16 + (lane >> 5) * 4 + ((lane & 15) >> 2), e = d * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
            const s16x4 lo = read_transposed(tv + place<S>(key, e >> 3) + (e & 7) * 2);
            const s16x4 hi = read_transposed(tv + place<S>(key + 8, e >> 3) + (e & 7) * 2);
            x.v[s & 1][d] = __builtin_bit_cast(Vec<T, 8>, Vec<short, 8>{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
        }
    }
    // scores of the keys, whose first part has been read
    template <int KB>
    __device__ void scores(Work<KB>& x, const char* tk, int lane) const {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            if (i + 1 < PARTS) read_keys(x, tk, i + 1, lane);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int b = 0; b < KB; ++b) x.z[b] = Mma<T>::go(x.k[i & 1][s][b], q[i * 2 + s], i + s ? x.z[b] : f32x16{});
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // weights of the scores.  Masked: only keys below `mine` count.
    template <bool Masked, int KB>
    __device__ void weights(Work<KB>& x, uint32_t j0, uint32_t mine, float scale, int lane) {
        // Keys that this lane's row sees: register r of block b has key b * 32 + r % 4 + 8 (r / 4) + 4 h.  Opaque, and the
        // scores after it, so that a comparison with a constant and a selection per score are all that is left of it.
        int left = static_cast<int>(min(mine, j0 + 64u) - min(mine, j0)) - (lane >> 5) * 4;
        if (Masked) asm volatile("" : "+v"(left));
        float high[4] = {NONE, NONE, NONE, NONE};
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (Masked) {
                    float z = b * 32 + (r & 3) + 8 * (r >> 2) >= left ? NONE : x.z[b][r];
                    asm volatile("" : "+v"(z));
                    x.z[b][r] = z;
                }
                high[r >> 2] = larger(high[r >> 2], x.z[b][r]);
            }
        const float2 two = halves(larger(larger(high[0], high[1]), larger(high[2], high[3])));
        const float most = larger(two.x, two.y) * scale;  // scale > 0; NaN if some score is, as the row's sum will be
        // The weights may stand against an older maximum while they stay below 2^(ROOM + LAG): sums and results lose
        // nothing by that, and the results are rescaled seldom.  A row's own scores alone decide about it, so that no
        // other row's keys show in its bits.
        const bool grows = most - top > ROOM + LAG;
        float base = top;
        if (__any(grows) || far) {
            const float now = most - ROOM, fade = grows ? __builtin_amdgcn_exp2f(top - now) : 1.0f;
            top = grows ? now : top;
            sum *= fade;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= fade;
            far = __any(is_far(top));
            base = top;
            if (far) {
                const float by = is_far(top) ? scale : 1.0f, off = is_far(top) ? top : 0.0f, back = 1.0f / by;
                base = is_far(top) ? 0.0f : top;
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) x.z[b][r] = (x.z[b][r] * by - off) * back;
            }
        }
        base = base == NONE ? 0.0f : base;  // nothing visible yet: every weight is exp2(-inf) = 0
        float add[4] = {};
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = __builtin_amdgcn_exp2f(fmaf(x.z[b][r], scale, -base));
                add[r & 3] += e;
                x.w[b * 2 + (r >> 3)][r & 7] = static_cast<T>(e);
            }
        sum += (add[0] + add[1]) + (add[2] + add[3]);
    }
    // the weighted values, whose first part has been read: products that follow each other are of different
    // elements, for one that waits for its predecessor's result takes twice as long
    template <int KB>
    __device__ void results(Work<KB>& x, const char* tv, int lane) {
#pragma unroll
        for (int s = 0; s < 2 * KB; ++s) {
            __builtin_amdgcn_sched_barrier(0);
            if (s + 1 < 2 * KB) read_values(x, tv, s + 1, lane);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < PARTS; ++d) o[d] = Mma<T>::go(x.v[s & 1][d], x.w[s], o[d]);
        }
    }
    // all of it for the keys from j0 on, in LDS
    template <int KB, bool Masked>
    __device__ void step(const char* tk, const char* tv, uint32_t j0, uint32_t mine, float scale, int lane) {
        Work<KB> x;
        read_keys(x, tk, 0, lane);
        scores(x, tk, lane);
        read_values(x, tv, 0, lane);
        __builtin_amdgcn_sched_barrier(0);
        weights<Masked>(x, j0, mine, scale, lane);
        results(x, tv, lane);
    }
    __device__ void join_halves() {
        const float2 two = halves(sum);
        sum = two.x + two.y;
    }
};

// A weight of 0 times NaN or an infinity is NaN, so a row would be touched by values that it does not see.  Where
// the tiles that some row does not see whole give a result that is not finite, they are taken five times:
// as they are, with 1 for every NaN (+infinity, -infinity) and 0 for the rest, and with 0 for what is not
// finite.  The last pass gives the sums; NaN and infinities are added where their passes gave more than 0.  Those passes take
// every key that is seen about alike, for its weight may be too small for its type.
enum { PLAIN = 0, NANS = 1, HIGH = 2, LOW = 3, FINITE = 4 };
__device__ inline float scale_of(int pass, float scale) { return pass == PLAIN || pass == FINITE ? scale : 0x1p-126f; }

// the values of keys that no row of the tile sees -- later ones of the sequence, and what lies past its end, for which the
// moves repeat its last one: no weight of 0 meets NaN there
template <int S>
__device__ inline void blank(char* tv, uint32_t first, uint32_t rows, int thread, int threads) {
    for (uint32_t i = first * (S / 16) + thread; i < rows * (S / 16); i += threads) reinterpret_cast<Vec<float, 4>*>(tv)[i] = Vec<float, 4>{};
}
// the values of a tile for a pass: 16 bytes at a time, by THREADS threads
template <typename T>
__device__ inline void sift(char* tv, int bytes, int pass, int thread, int threads) {
    for (int i = thread; i < bytes / 16; i += threads) {
        Vec<T, 8>* p = reinterpret_cast<Vec<T, 8>*>(tv) + i;
        Vec<T, 8> x = *p;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = static_cast<float>(x[j]);
            const int is = f != f ? NANS : f == INFINITY ? HIGH : f == NONE ? LOW : FINITE;
            x[j] = static_cast<T>(pass == FINITE ? (is == FINITE ? f : 0.0f) : is == pass ? 1.0f : 0.0f);
        }
        *p = x;
    }
}
template <int N>
struct Found {  // results with such values: a bit each, NaN and +infinity in one word, -infinity in the other
    uint32_t one[N], two[N];
    __device__ void clear() {
#pragma unroll
        for (int d = 0; d < N; ++d) one[d] = two[d] = 0;
    }
    __device__ void take(const f32x16 (&o)[N], int pass) {
#pragma unroll
        for (int d = 0; d < N; ++d) {
            uint32_t bits = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) bits |= o[d][r] > 0.0f ? 1u << r : 0u;
            one[d] |= pass == NANS ? bits : pass == HIGH ? bits << 16 : 0u;
            two[d] |= pass == LOW ? bits : 0u;
        }
    }
    __device__ void give(f32x16 (&o)[N]) const {
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (one[d] >> r & 1) o[d][r] = NAN;
                if (one[d] >> (r + 16) & 1) o[d][r] += INFINITY;
                if (two[d] >> r & 1) o[d][r] += NONE;
            }
    }
};

__device__ inline float reciprocal_of(float sum) { return sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum; }
__device__ inline float log_of(float top, float sum) { return sum == 0.0f ? NONE : (top + log2f(sum)) * LN2; }

// Moves KEYS rows of keys and of values to LDS, 16 bytes a lane; THREADS threads (whole waves) share them.
template <int S, int KEYS, int THREADS>
struct Mover {
    static constexpr int CH = S / 16, N = THREADS / CH, MOVES = KEYS / N;  // rows of a move; moves of each kind
    const char *k, *v;
    int64_t khop, vhop;   // bytes between rows
    uint32_t kat, vat;    // this thread's row of a move, if rows lie within 32 bits (near)
    uint32_t nk, chunks, first;
    int row, wave;

    __device__ Mover(const bs_attention_args& a, const Sequence& sq, uint32_t kvh, int thread)
        : khop(a.k_stride * 2), vhop(a.v_stride * 2), nk(sq.nk), chunks(a.head_dim / 8), row(thread / CH),
          wave(uniform(static_cast<uint32_t>(thread >> 6))) {
        k = static_cast<const char*>(a.k) + static_cast<int64_t>(sq.k0) * khop + static_cast<int64_t>(kvh) * a.k_head_stride * 2;
        v = static_cast<const char*>(a.v) + static_cast<int64_t>(sq.k0) * vhop + static_cast<int64_t>(kvh) * a.v_head_stride * 2;
        kat = row * static_cast<uint32_t>(khop);
        vat = row * static_cast<uint32_t>(vhop);
        first = (place<S>(row, thread % CH) - row * S) >> 4;
    }
    // the chunk whose place this thread's slot is in move i
    __device__ uint32_t chunk(int i) const { return first ^ static_cast<uint32_t>((place<S>(i * N, 0) - i * N * S) >> 4); }
    // rows j0 .. j0 + KEYS - 1 of the sequence, near
    __device__ void near(const char* from, int64_t hop, uint32_t at, uint32_t j0, char* to) const {
        const char* p = from + static_cast<int64_t>(j0) * hop;
#pragma unroll
        for (int i = 0; i < MOVES; ++i)
            if (chunk(i) < chunks) move16(p + i * (N * hop), at + chunk(i) * 16, to + i * N * S + wave * 1024);
    }
    // any rows; those past the sequence's end repeat its last one, and no row sees them
    __device__ void any(const char* from, int64_t hop, uint32_t j0, char* to) const {
#pragma unroll
        for (int i = 0; i < MOVES; ++i) {
            const char* p = from + static_cast<int64_t>(min(j0 + i * N + row, nk - 1)) * hop;
            if (chunk(i) < chunks)
                __builtin_amdgcn_global_load_lds((global_ptr)(p + chunk(i) * 16), (lds_ptr)(to + i * N * S + wave * 1024), 16, 0, 0);
        }
    }
    // the values lie after the keys
    __device__ void near(uint32_t j0, char* to) const {
        near(k, khop, kat, j0, to);
        near(v, vhop, vat, j0, to + KEYS * S);
    }
    __device__ void any(uint32_t j0, char* to) const {
        any(k, khop, j0, to);
        any(v, vhop, j0, to + KEYS * S);
    }
};

struct Place {  // of a row: its query token in the sequence, its head, the keys that it sees
    uint32_t tok, head, keys;
    bool live;
};
// row of a sequence's (token, head of the group) pairs; past the end the last one, not live
__device__ inline Place place_of(const Params& p, const Sequence& sq, uint32_t kvh, uint32_t row, uint32_t rows) {
    Place x;
    x.live = row < rows;
    const uint32_t r = x.live ? row : rows - 1;
    x.tok = p.by_group.quotient(r);
    x.head = kvh * p.group + (r - x.tok * p.group);
    x.keys = keys_of(p.a, sq, x.tok);
    return x;
}

// a row's results: parts to the workspace, or the output
template <typename T, int DP>
__device__ inline void write_rows(const Params& p, const Sequence& sq, const Place& me, const Rows<T, DP>& r, int h) {
    if (!me.live) return;
    const bs_attention_args& a = p.a;
    const int64_t at = static_cast<int64_t>(sq.q0 + me.tok) * a.heads + me.head;
    if (p.splits > 1) {
        const int64_t slot = static_cast<int64_t>(blockIdx.y) * a.q_tokens * a.heads + at;
        if (h == 0) p.part_stat[slot] = make_float2(r.top, r.sum);
        float* out = p.part_out + slot * a.head_dim;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t e = d * 32 + i * 8 + h * 4;
                const f32x4 v = {r.o[d][i * 4], r.o[d][i * 4 + 1], r.o[d][i * 4 + 2], r.o[d][i * 4 + 3]};
                if (e < a.head_dim) *reinterpret_cast<f32x4*>(out + e) = v;
            }
        return;
    }
    const float over = reciprocal_of(r.sum);
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(sq.q0 + me.tok) * a.out_stride + static_cast<int64_t>(me.head) * a.out_head_stride;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t e = d * 32 + i * 8 + h * 4;
            Vec<T, 4> v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = static_cast<T>(r.o[d][i * 4 + j] * over);
            if (e < a.head_dim) *reinterpret_cast<Vec<T, 4>*>(out + e) = v;
        }
    if (a.lse && h == 0) a.lse[at] = log_of(r.top, r.sum);
}

// Whole prompts.  Four waves of 32 rows share the tiles of 64 keys in LDS, two of them: the next tile's moves
// run under a tile's products.  Two workgroups per compute unit (three for heads up to 64): one's matrix
// instructions run under the other's exponentials.  (Three for heads of 64: passages below 90 to 83 us; four spill: 144.)
//
// Two causal documents of 8192 and 7500 tokens, 32 heads of 128, 8 key/value heads, bf16: 973 us (992 TFLOP/s), the
// vector and matrix pipes half busy each (0.50, 0.47): a wave's exponentials and its products do not overlap, only two
// waves' do.  96 passages of 37..512 tokens, 16 heads of 64: 69 us, the vector pipe busy for 0.43 of the time (170
// instructions beside 16 matrix instructions a tile, 270 with masks) and waves waiting for 0.40 of theirs, on the four
// dependent rounds of loads with which each of the 3864 short workgroups starts.  Other orders that were slower for
// the documents: two groups of waves half a step apart, meeting between their phases (1244 against 1175), moves between
// the products and exponentials instead of before them (1246 against 1142).
template <typename T, int DP>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : 2) void attention_kernel(Params p) {
    constexpr int ROWS = 128, S = ROW<DP>, TILE = BN * S;
    // blocks of 32 keys at a time in the tiles that some row does not see whole: one where heads are short, for its code
    // is short too and half of a short prompt's tiles are such (passages: 74 us, 80 with two); two for heads of 128
    // (documents: 989 us, 1001 with one)
    constexpr int KB = DP <= 64 ? 1 : 2;
    __shared__ __attribute__((aligned(16))) char lds[2][2 * TILE];
    __shared__ int flag;
    const bs_attention_args& a = p.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 31, h = lane >> 5;
    const uint32_t tile = p.by_kv.quotient(blockIdx.x), kvh = blockIdx.x - tile * a.kv_heads;
    const uint32_t seq = a.q_offsets ? find(a.q_offsets, a.sequences, tile, p.group, ROWS) : 0;
    const uint64_t first = a.q_offsets ? first_tile(a.q_offsets, seq, p.group, ROWS) : 0;
    const Sequence sq = sequence(a, seq);
    const uint32_t rows = sq.nq * p.group;  // < 2^31, as q_tokens x heads
    if (tile < first || (tile - first) * ROWS >= rows) return;
    // the tiles that see most keys start first
    const uint32_t row0 = ((rows - 1) / ROWS - static_cast<uint32_t>(tile - first)) * ROWS;
    const uint32_t all = keys_of(a, sq, p.by_group.quotient(min(rows, row0 + ROWS) - 1));  // of the tile's last row: the most
    uint32_t kb = 0, ke = all;
    if (p.splits > 1) {
        kb = min(all, blockIdx.y * p.piece);
        if (blockIdx.y + 1 < p.splits) ke = min(all, kb + p.piece);
        if (kb >= ke && blockIdx.y > 0) return;  // the join does not read it
    }
    // The tiles that some row does not see whole come first, on a state of zeros, so that they can be taken again.
    const uint32_t seen = keys_of(a, sq, p.by_group.quotient(row0));  // by every row of the tile
    const uint32_t full = max(kb, min(ke, seen) / BN * BN);          // kb and pieces are multiples of BN
    const uint32_t parts = (ke - full + BN - 1) / BN, tiles = parts + (full - kb) / BN;
    auto start = [&](uint32_t t) { return t < parts ? full + t * BN : kb + (t - parts) * BN; };
    if (a.head_dim != DP) {  // the padding of the heads is never moved to
        for (int i = threadIdx.x; i < 2 * 2 * TILE / 16; i += 256) reinterpret_cast<Vec<float, 4>*>(lds[0])[i] = Vec<float, 4>{};
    }
    if (threadIdx.x == 0) flag = 0;
    settle();
    const Mover<S, BN, 256> mover(a, sq, kvh, threadIdx.x);
    if (tiles) mover.any(start(0), lds[0]);
    const Place me = place_of(p, sq, kvh, row0 + wave * 32 + l, rows);
    Rows<T, DP> me_;
    me_.load(static_cast<const T*>(a.q) + static_cast<int64_t>(sq.q0 + me.tok) * a.q_stride + static_cast<int64_t>(me.head) * a.q_head_stride,
             a.head_dim, a.scale, h);
    me_.clear();
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * LOG2E;
    const uint32_t mine = min(me.keys, ke);
    // keys up to which this wave's last row sees; a wave past the last row has nothing to do but its moves
    const uint32_t wave0 = row0 + wave * 32;
    const uint32_t reach = wave0 < rows ? min(ke, keys_of(a, sq, p.by_group.quotient(min(rows, wave0 + 32) - 1))) : 0;
    Found<DP / 32> found;
    for (int pass = PLAIN; parts; ++pass) {
        for (uint32_t t = 0; t < parts; ++t) {
            char* tk = lds[t & 1];
            meet();  // tile t is in LDS, and nobody reads tile t - 1 any more
            if (t + 1 < tiles) mover.any(start(t + 1), lds[~t & 1]);
            if (start(t) + BN > all || pass != PLAIN) {
                if (start(t) + BN > all) blank<S>(tk + TILE, all - start(t), BN, threadIdx.x, 256);  // start(t) < ke <= all
                settle();
                if (pass != PLAIN) sift<T>(tk + TILE, TILE, pass, threadIdx.x, 256);
                settle();
            }
#pragma unroll 1
            for (int b = 0; b < BN; b += KB * 32)
                if (reach > start(t) + b) me_.template step<KB, true>(tk + b * S, tk + TILE + b * S, start(t) + b, mine, scale_of(pass, scale), lane);
        }
        if (pass == PLAIN) {
            if (seen == all) break;  // all rows see the same keys, and the others' values are blank
            if (me_.odd()) flag = 1;
            settle();
            if (!uniform(static_cast<uint32_t>(flag))) break;
            meet();
            found.clear();
        } else if (pass == FINITE) {
            found.give(me_.o);
            break;
        } else {
            found.take(me_.o, pass);
            meet();
        }
        me_.clear();
        mover.any(start(0), lds[0]);  // tile `parts` has landed, and is moved again
    }
    for (uint32_t t = parts; t < tiles; ++t) {
        const char* tk = lds[t & 1];
        meet();
        if (t + 1 < tiles) mover.near(kb + (t + 1 - parts) * BN, lds[~t & 1]);
        if (reach) {
            // a loop of one turn: as a block of its own the step is scheduled apart from the moves (documents: 989 us, 1004
            // in one block with them)
#pragma unroll 1
            for (int b = 0; b < BN; b += 64) me_.template step<2, false>(tk + b * S, tk + TILE + b * S, 0, 0, scale, lane);
        }
    }
    me_.join_halves();
    write_rows<T, DP>(p, sq, me, me_, h);
}

// Few rows per sequence (single tokens): the keys' bytes bound the time.  A tile has at most 32 rows, and the
// FEW_WAVES waves of a workgroup take turns at its tiles of 32 keys, through LDS of their own, without meeting;
// their results are joined at the end.  16 tokens over 16 sequences of 1.4k..16k keys, 8 heads of 128: 135 us, 4.7 TB/s
// (a copy reaches 5.1), and 5 us for the join of the pieces; four waves, of which fewer fit: 155 against 146 then.
constexpr int FEW_WAVES = 2;

// Near: rows of keys that a move takes lie within 32 bits of each other, of values too
template <typename T, int DP, bool Near>
__global__ __launch_bounds__(FEW_WAVES * 64, 1) void attention_few_kernel(Params p) {
    constexpr int ROWS = 32, KN = 32, S = ROW<DP>, TILE = KN * S, NB = 32768 / (2 * TILE);  // NB tiles of a wave in LDS
    constexpr int W = FEW_WAVES;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const bs_attention_args& a = p.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 31, h = lane >> 5;
    const uint32_t tile = p.by_kv.quotient(blockIdx.x), kvh = blockIdx.x - tile * a.kv_heads;
    const uint32_t seq = a.q_offsets ? find(a.q_offsets, a.sequences, tile, p.group, ROWS) : 0;
    const uint64_t first = a.q_offsets ? first_tile(a.q_offsets, seq, p.group, ROWS) : 0;
    const Sequence sq = sequence(a, seq);
    const uint32_t rows = sq.nq * p.group;  // < 2^31, as q_tokens x heads
    if (tile < first || (tile - first) * ROWS >= rows) return;
    const uint32_t row0 = static_cast<uint32_t>(tile - first) * ROWS;
    const Place me = place_of(p, sq, kvh, row0 + l, rows);
    const uint32_t here = min(rows - row0, static_cast<uint32_t>(ROWS));  // rows of the tile
    const uint32_t all = keys_of(a, sq, p.by_group.quotient(row0 + here - 1));
    const uint32_t kb = min(all, blockIdx.y * p.piece), ke = blockIdx.y + 1 < p.splits ? min(all, kb + p.piece) : all;
    if (kb >= ke && blockIdx.y > 0) return;  // the join does not read it
    Rows<T, DP> me_;
    me_.load(static_cast<const T*>(a.q) + static_cast<int64_t>(sq.q0 + me.tok) * a.q_stride + static_cast<int64_t>(me.head) * a.q_head_stride,
             a.head_dim, a.scale, h);
    me_.clear();
    char* mem = lds + wave * 32768;
    if (a.head_dim != DP) {  // the padding of the heads is never moved to
        for (int i = lane; i < 32768 / 16; i += 64) reinterpret_cast<Vec<float, 4>*>(mem)[i] = Vec<float, 4>{};
    }
    const Mover<S, KN, 64> mover(a, sq, kvh, lane);
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * LOG2E;
    const uint32_t mine = min(me.keys, ke), seen = keys_of(a, sq, p.by_group.quotient(row0));
    // tiles from the last to the first: of those that some row does not see whole (at most 2 in a row: a
    // tile of rows has at most 32 tokens) a wave has at most one, its first
    const uint32_t tiles = (ke - kb + KN - 1) / KN, n = tiles > static_cast<uint32_t>(wave) ? (tiles - wave + W - 1) / W : 0;
    auto start = [&](uint32_t u) { return kb + (tiles - 1 - wave - W * u) * KN; };
    auto buffer = [&](uint32_t u) { return mem + u % NB * (2 * TILE); };
    constexpr int MOVES = 2 * Mover<S, KN, 64>::MOVES;  // of a tile
    static_assert(NB * MOVES < 64, "counted by vmcnt");
    landed<0>();
#pragma unroll
    for (int u = 0; u < NB; ++u)
        if (static_cast<uint32_t>(u) < n) mover.any(start(u), buffer(u));
    auto arrive = [&](uint32_t u) {  // the moves of tiles u + 1 .. u + NB - 1 may be on their way
        if (u + NB <= n)
            landed<(NB - 1) * MOVES>();
        else
            landed<0>();
        return buffer(u);
    };
    auto follow = [&](uint32_t u) {
        if (u + NB < n) {
            landed<63>();  // this tile's reads are done
            if (Near)  // whole: only a wave's first tile may pass the end
                mover.near(start(u + NB), buffer(u));
            else
                mover.any(start(u + NB), buffer(u));
        }
    };
    uint32_t u = 0;
    if (n && start(0) + KN > min(seen, ke)) {
        char* tk = arrive(0);
        const uint32_t j0 = start(0);
        Found<DP / 32> found;
        for (int pass = PLAIN;; ++pass) {
            if (j0 + KN > all) blank<S>(tk + TILE, all - j0, KN, lane, 64);  // j0 < ke <= all
            landed<63>();
            if (pass != PLAIN) {
                sift<T>(tk + TILE, TILE, pass, lane, 64);
                landed<63>();
            }
            me_.template step<1, true>(tk, tk + TILE, j0, mine, scale_of(pass, scale), lane);
            if (pass == PLAIN) {
                // all rows see the same keys, and the others' values are blank; or nothing is there to touch them
                if (seen == all || !__any(me_.odd())) break;
                found.clear();
            } else if (pass == FINITE) {
                found.give(me_.o);
                break;
            } else {
                found.take(me_.o, pass);
            }
            me_.clear();
            landed<63>();
            mover.any(j0, tk);
            landed<0>();
        }
        follow(0);
        u = 1;
    }
    for (; u < n; ++u) {
        const char* tk = arrive(u);
        me_.template step<1, false>(tk, tk + TILE, start(u), mine, scale, lane);
        follow(u);
    }
    me_.join_halves();
    // joins the waves: every wave's results against the largest of their maxima, then a sum in wave order
    __shared__ float2 stat[W][32];
    landed<0>();
    __syncthreads();  // nobody reads tiles any more
    if (h == 0) stat[wave][l] = make_float2(me_.top, me_.sum);
    float* all_o = reinterpret_cast<float*>(lds);  // W x 32 x (DP + 4)
    __syncthreads();
    float top = NONE;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, stat[w][l].x);
    const float gain = __builtin_amdgcn_exp2f(me_.top - (top == NONE ? 0.0f : top));
    if (static_cast<uint32_t>(l) < here) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<f32x4*>(all_o + (wave * 32 + l) * (DP + 4) + d * 32 + r * 8 + h * 4) =
                    f32x4{me_.o[d][r * 4] * gain, me_.o[d][r * 4 + 1] * gain, me_.o[d][r * 4 + 2] * gain, me_.o[d][r * 4 + 3] * gain};
    }
    __syncthreads();
    const uint32_t quads = a.head_dim / 4;
    for (uint32_t i = threadIdx.x; i < here * quads; i += W * 64) {
        const uint32_t r = i / quads, e = i % quads * 4;
        float t = NONE, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) t = fmaxf(t, stat[w][r].x);
        f32x4 v = {};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            sum += stat[w][r].y * __builtin_amdgcn_exp2f(stat[w][r].x - (t == NONE ? 0.0f : t));
            v += *reinterpret_cast<const f32x4*>(all_o + (w * 32 + r) * (DP + 4) + e);
        }
        const Place x = place_of(p, sq, kvh, row0 + r, rows);
        const int64_t at = static_cast<int64_t>(sq.q0 + x.tok) * a.heads + x.head;
        if (p.splits > 1) {
            const int64_t slot = static_cast<int64_t>(blockIdx.y) * a.q_tokens * a.heads + at;
            *reinterpret_cast<f32x4*>(p.part_out + slot * a.head_dim + e) = v;
            if (e == 0) p.part_stat[slot] = make_float2(t, sum);
        } else {
            const float over = reciprocal_of(sum);
            const Vec<T, 4> y = {static_cast<T>(v[0] * over), static_cast<T>(v[1] * over), static_cast<T>(v[2] * over), static_cast<T>(v[3] * over)};
            *reinterpret_cast<Vec<T, 4>*>(static_cast<T*>(a.out) + static_cast<int64_t>(sq.q0 + x.tok) * a.out_stride +
                                          static_cast<int64_t>(x.head) * a.out_head_stride + e) = y;
            if (a.lse && e == 0) a.lse[at] = log_of(t, sum);
        }
    }
}

// Joins the pieces of a row (query token, head), W waves a row.  First the maximum of all pieces and the sum against it, a
// piece per lane; then the results, the pieces in W contiguous runs, one per wave.
template <typename T, int W>
__global__ __launch_bounds__(256) void join_kernel(Params p) {
    static_assert(W == 1 || W == 4, "a workgroup has four waves");
    __shared__ float2 half[4][64];
    const bs_attention_args& a = p.a;
    const int lane = threadIdx.x & 63, wave = static_cast<int>(uniform(threadIdx.x >> 6)), part = W == 1 ? 0 : wave;
    const uint64_t rows = static_cast<uint64_t>(a.q_tokens) * a.heads;
    const uint32_t at = W == 1 ? blockIdx.x * 4 + wave : blockIdx.x;  // < 2^31 + 4
    if (at >= rows) return;
    const uint32_t tok = at / a.heads, head = at % a.heads;
    const uint32_t seq = a.q_offsets ? holder(a.q_offsets, a.sequences, tok) : 0;
    const Sequence sq = sequence(a, seq);
    if (tok < sq.q0 || tok - sq.q0 >= sq.nq) return;
    const uint32_t keys = keys_of(a, sq, tok - sq.q0);
    const uint32_t n = max(1u, min(p.splits, (keys + p.piece - 1) / p.piece));
    float top = NONE, sum = 0.0f;
    for (uint32_t s = lane; s < n; s += 64) top = fmaxf(top, p.part_stat[s * rows + at].x);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    const float base = top == NONE ? 0.0f : top;
    for (uint32_t s = lane; s < n; s += 64) {
        const float2 st = p.part_stat[s * rows + at];
        sum += st.y * __builtin_amdgcn_exp2f(st.x - base);
    }
    sum = wave_sum(sum);
    const uint32_t d = lane * 2, run = (n + W - 1) / W, begin = part * run, end = min(begin + run, n);
    float2 o = make_float2(0.0f, 0.0f);
    if (d < a.head_dim) {
#pragma unroll 4
        for (uint32_t s = begin; s < end; ++s) {
            const uint64_t slot = s * rows + at;
            const float gain = __builtin_amdgcn_exp2f(p.part_stat[slot].x - base);
            const float2 v = *reinterpret_cast<const float2*>(p.part_out + slot * a.head_dim + d);
            o.x = fmaf(v.x, gain, o.x);
            o.y = fmaf(v.y, gain, o.y);
        }
    }
    if (W > 1) {
        half[wave][lane] = o;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 1; w < W; ++w) o.x += half[w][lane].x, o.y += half[w][lane].y;
    }
    const float over = reciprocal_of(sum);
    if (d < a.head_dim) {
        T* out = static_cast<T*>(a.out) + static_cast<int64_t>(tok) * a.out_stride + static_cast<int64_t>(head) * a.out_head_stride;
        *reinterpret_cast<Vec<T, 2>*>(out + d) = Vec<T, 2>{static_cast<T>(o.x * over), static_cast<T>(o.y * over)};
    }
    if (a.lse && lane == 0) a.lse[at] = log_of(top, sum);
}

uint64_t tiles_of(const bs_attention_args& a, uint32_t rows) {
    const uint64_t t = static_cast<uint64_t>(a.q_tokens) * (a.heads / a.kv_heads);
    return t / rows + a.sequences;
}

// Whether the rows of a move lie within 32 bits of each other, so that its addresses are a scalar and an offset per lane
// (documents above: 1118 us, 1173 with 64 bits per lane).  Rows farther apart go to the few rows' kernel, which has both.
bool near_of(const bs_attention_args& a) { return a.k_stride < (1 << 22) && a.v_stride < (1 << 22); }

// Single tokens of groups up to 8, by the longest sequence where it is given, else by the mean.  Against whole prompts'
// kernel: 16 tokens over 1.4k..16k keys of 8 heads of 128, groups of 4: 141 and 162 us, of 16 heads of 64: 147 and 210;
// but two tokens each over 4096 keys, groups of 4: 38 and 36, eight 68 and 40; one token over 16384 keys, group of 32:
// 16.7 and 15.4.
bool few_of(const bs_attention_args& a) {
    const uint64_t tokens = a.longest_q ? a.longest_q : (a.q_tokens + a.sequences - 1) / a.sequences;
    return tokens <= 1 && a.heads / a.kv_heads <= 8;
}

// Pieces of the keys, multiples of the keys that a workgroup takes at a time.  The last one takes what is left,
// should a sequence be longer than longest_k said.
void split(const bs_attention_args& a, uint32_t& splits, uint32_t& piece) {
    const uint32_t longest = a.longest_k ? std::min(a.longest_k, a.k_tokens) : a.k_tokens;
    const uint64_t rows = static_cast<uint64_t>(a.q_tokens) * a.heads;
    uint64_t want;
    if (few_of(a)) {
        // About six workgroups per compute unit, so that sequences of different lengths even out: 16 tokens over 1.4k..16k
        // keys take 141 us, with two 161, with twelve 140.  Pieces of 256 keys at least (one token over 16384 keys 20.2 us,
        // 25.9 with 128, 21.4 with 512), of 512 where there is a workgroup for every compute unit without (64 over 1024
        // keys, 4 heads of 64: 20.8, with 256 24.5).
        const uint64_t keys = static_cast<uint64_t>(a.k_tokens) * a.kv_heads;
        const uint64_t least = static_cast<uint64_t>(a.sequences) * a.kv_heads >= CUS ? 512 : 256;
        want = std::max<uint64_t>(keys / (6 * CUS), least);
    } else {
        // Two workgroups per compute unit, where the keys are long enough for the parts of the rows to be written and joined.
        // With and without: 200 tokens over 4096 keys, 32 heads of 128 35 and 101 us, 768 over 8192 117 and 204; 900 over 900
        // 34 and 25, 600 over 1200 34 and 31, 1024 over 1024, 16 heads of 64 26 and 20.
        const uint64_t groups = tiles_of(a, 128) * a.kv_heads;
        const bool whole = groups >= 2 * CUS || static_cast<uint64_t>(longest) * 16 <= rows + 8192;
        want = whole ? longest : std::max<uint64_t>(longest * groups / (2 * CUS), 256);
    }
    piece = static_cast<uint32_t>(std::min<uint64_t>((want + 127) / 128 * 128, (static_cast<uint64_t>(longest) + 127) / 128 * 128));
    if (piece == 0) piece = 128;
    // at most 256 MB of parts: with many sequences the pieces are for their different lengths alone
    const uint64_t row = rows * (a.head_dim + 2) * sizeof(float);
    const uint64_t most = std::max<uint64_t>(1, std::min<uint64_t>(65535, (1ull << 28) / std::max<uint64_t>(row, 1)));
    if ((longest + piece - 1) / piece > most) piece = static_cast<uint32_t>((longest + most - 1) / most + 127) / 128 * 128;
    splits = std::max(1u, (longest + piece - 1) / piece);
}

uint64_t workspace_of(const bs_attention_args& a) {
    uint32_t splits, piece;
    split(a, splits, piece);
    if (splits <= 1) return 0;
    return static_cast<uint64_t>(splits) * a.q_tokens * a.heads * (a.head_dim + 2) * sizeof(float);
}

int check(const char* what, const bs_attention_args* a) {
    const std::string w = what;
    if (!a) return refuse(w + ": args is null");
    if (a->type != BS_F16 && a->type != BS_BF16) return refuse(w + ": type must be BS_F16 or BS_BF16");
    if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8) return refuse(w + ": head_dim must be a multiple of 8 in 8..128");
    if (a->heads == 0 || a->heads > 1024 || a->kv_heads == 0 || a->heads % a->kv_heads)
        return refuse(w + ": heads must be in 1..1024 and a multiple of kv_heads");
    if (a->q_tokens > 0x7FFFFFFFu || a->k_tokens > 0x7FFFFFFFu) return refuse(w + ": q_tokens and k_tokens must be < 2^31");
    if (a->sequences == 0 || a->sequences > 0x7FFFFFFu) return refuse(w + ": sequences must be in 1..2^27");
    if (!(std::fabs(a->scale) <= 1e30f)) return refuse(w + ": scale must be finite, at most 1e30");
    // threads of a launch are counted in 32 bits
    if (tiles_of(*a, 32) * a->kv_heads * 256 > 0xFFFFFFFFull || static_cast<uint64_t>(a->q_tokens) * a->heads > 0x7FFFFFFFull) return refuse(w + ": too many tiles for one launch");
    return BS_OK;
}

template <typename T, int DP, bool Near>
int start_few(const Params& p, hipStream_t s) {
    constexpr int LDS = FEW_WAVES * 32768;
    auto* k = attention_few_kernel<T, DP, Near>;
    static std::atomic<uint64_t> done{0};
    if (const int rc = allow_lds(reinterpret_cast<const void*>(k), LDS, done)) return rc;
    k<<<dim3(static_cast<uint32_t>(tiles_of(p.a, 32) * p.a.kv_heads), p.splits), FEW_WAVES * 64, LDS, s>>>(p);
    return BS_OK;
}
template <typename T, int DP>
int start(const Params& p, hipStream_t s) {
    if (!near_of(p.a)) return start_few<T, DP, false>(p, s);  // rows too far apart for the other kernel's moves
    if (few_of(p.a)) return start_few<T, DP, true>(p, s);
    attention_kernel<T, DP><<<dim3(static_cast<uint32_t>(tiles_of(p.a, 128) * p.a.kv_heads), p.splits), 256, 0, s>>>(p);
    return BS_OK;
}

template <typename T>
int launch(const Params& p, hipStream_t s) {
    const uint32_t d = p.a.head_dim;
    const int rc = d <= 32 ? start<T, 32>(p, s) : d <= 64 ? start<T, 64>(p, s) : d <= 96 ? start<T, 96>(p, s) : start<T, 128>(p, s);
    if (rc) return rc;
    if (p.splits > 1) {
        // Four waves a row where rows are few and their latency counts, one where there are many.  One and four: 1000 tokens
        // over 4096 keys, 16 heads of 64 38 and 54 us, 768 over 8192, 32 heads of 128 117 and 137, 8 x 8 over 4096 (2048
        // rows) 38.5 and 39.2; but 40 over 8192 (1280 rows) 26.4 and 25.5, one token over 16384 24.0 and 20.3.
        const uint32_t rows = p.a.q_tokens * p.a.heads;
        if (rows >= 8 * CUS)
            join_kernel<T, 1><<<(rows + 3) / 4, 256, 0, s>>>(p);
        else
            join_kernel<T, 4><<<rows, 256, 0, s>>>(p);
    }
    return launched("bs_attention");
}

}  // namespace

extern "C" int bs_attention_workspace(const bs_attention_args* args, uint64_t* bytes) try {
    if (!bytes) return refuse("bs_attention_workspace: bytes is null");
    if (const int rc = check("bs_attention_workspace", args)) return rc;
    *bytes = workspace_of(*args);
    return BS_OK;
} catch (...) {
    return bs_internal_exception();
}

extern "C" int bs_attention(const bs_attention_args* args, void* workspace, uint64_t workspace_bytes, void* stream) try {
    if (const int rc = check("bs_attention", args)) return rc;
    const bs_attention_args& a = *args;
    if (a.sequences > 1 && (!a.q_offsets || !a.k_offsets)) return refuse("bs_attention: several sequences need q_offsets and k_offsets");
    if (a.q_tokens == 0) return BS_OK;
    if (!a.q || !a.out || (a.k_tokens && (!a.k || !a.v))) return refuse("bs_attention: q, k, v and out must be given");
    auto stride_ok = [&](const void* p, int64_t s, int64_t hs, uint32_t heads, uint32_t tokens) {
        return aligned16(p) && (tokens <= 1 || (s >= a.head_dim && s % 8 == 0)) && (heads <= 1 || (hs >= a.head_dim && hs % 8 == 0));
    };
    if (!stride_ok(a.q, a.q_stride, a.q_head_stride, a.heads, a.q_tokens) || !stride_ok(a.out, a.out_stride, a.out_head_stride, a.heads, a.q_tokens) ||
        (a.k_tokens && (!stride_ok(a.k, a.k_stride, a.k_head_stride, a.kv_heads, a.k_tokens) || !stride_ok(a.v, a.v_stride, a.v_head_stride, a.kv_heads, a.k_tokens))))
        return refuse("bs_attention: base addresses must be multiples of 16 bytes, strides multiples of 8 and >= head_dim");
    Params p{};
    p.a = a;
    p.group = a.heads / a.kv_heads;
    p.by_group = Divisor(p.group);
    p.by_kv = Divisor(a.kv_heads);
    split(a, p.splits, p.piece);
    if (p.splits > 1) {
        const uint64_t need = workspace_of(a);
        if (!workspace || workspace_bytes < need) return refuse("bs_attention: the workspace must hold " + std::to_string(need) + " bytes");
        if (!aligned16(workspace)) return refuse("bs_attention: the workspace must be 16-byte aligned");
        p.part_out = static_cast<float*>(workspace);
        p.part_stat = reinterpret_cast<float2*>(p.part_out + static_cast<uint64_t>(p.splits) * a.q_tokens * a.heads * a.head_dim);
    }
    return a.type == BS_F16 ? launch<f16>(p, static_cast<hipStream_t>(stream)) : launch<bf16>(p, static_cast<hipStream_t>(stream));
} catch (...) {
    return bs_internal_exception();
}
