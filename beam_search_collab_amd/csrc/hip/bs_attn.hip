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

struct Params {
    bs_attention_args a;
    uint32_t group;    // heads per key/value head
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
    return r;
}

// The tiles of all sequences are counted without a list of them: sequence s gets the tile numbers from
// offset(s) * group / rows + s on.  That leaves room for its own tiles and at most one unused number per sequence.
__device__ inline uint64_t first_tile(const int32_t* off, uint32_t s, uint32_t group, uint32_t rows) {
    return static_cast<uint64_t>(max(off[s], 0)) * group / rows + s;
}
// the last sequence whose first tile is <= tile: 64 candidates a step, the same for all lanes
__device__ inline uint32_t find(const int32_t* off, uint32_t n, uint64_t tile, uint32_t group, uint32_t rows) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 63) / 64, at = lo + (threadIdx.x & 63) * step;
        const bool below = at < hi && first_tile(off, at, group, rows) <= tile;
        const int k = __popcll(__ballot(below));
        lo += (k > 0 ? k - 1 : 0) * step;
        hi = min(lo + step, hi);
    }
    return lo;
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

// DP: head_dim rounded up to 32.  Four waves of 32 rows.
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void attention_kernel(Params p) {
    constexpr int ROWS = 128, S = DP <= 32 ? 64 : DP <= 64 ? 128 : 256, CH = DP / 8;
    __shared__ __attribute__((aligned(16))) char tk[BN * S], tv[BN * S];
    const bs_attention_args& a = p.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 31, h = lane >> 5;
    const uint32_t kvh = blockIdx.x % a.kv_heads, tile = blockIdx.x / a.kv_heads;
    const uint32_t seq = a.q_offsets ? find(a.q_offsets, a.sequences, tile, p.group, ROWS) : 0;
    const uint64_t first = a.q_offsets ? first_tile(a.q_offsets, seq, p.group, ROWS) : 0;
    const Sequence sq = sequence(a, seq);
    const uint64_t rows = static_cast<uint64_t>(sq.nq) * p.group;
    if (tile < first || (tile - first) * ROWS >= rows) return;
    const uint64_t row0 = (tile - first) * ROWS;
    const int64_t shift = static_cast<int64_t>(sq.nk) - sq.nq;  // query i sees the keys up to i + shift

    // this lane's row
    const uint64_t row = row0 + wave * 32 + l;
    const bool live = row < rows;
    const uint32_t tok = static_cast<uint32_t>((live ? row : rows - 1) / p.group);
    const uint32_t head = kvh * p.group + static_cast<uint32_t>((live ? row : rows - 1) - static_cast<uint64_t>(tok) * p.group);
    auto keys_of = [&](uint32_t t) {  // visible keys of query t
        const int64_t e = a.causal ? min(static_cast<int64_t>(sq.nk), t + shift + 1) : static_cast<int64_t>(sq.nk);
        return static_cast<uint32_t>(e < 0 ? 0 : e);
    };
    const uint32_t mine = keys_of(tok);
    const uint64_t last_row = min(rows, row0 + ROWS) - 1;
    const uint32_t all = keys_of(static_cast<uint32_t>(last_row / p.group));  // of the tile's last row: the most
    uint32_t kb = 0, ke = all;
    if (p.splits > 1) {
        kb = min(all, blockIdx.y * p.piece);
        if (blockIdx.y + 1 < p.splits) ke = min(all, kb + p.piece);
        if (kb >= ke && blockIdx.y > 0) return;  // the join does not read it
    }

    Vec<T, 8> q[DP / 16];
    const T* qp = static_cast<const T*>(a.q) + static_cast<int64_t>(sq.q0 + tok) * a.q_stride + static_cast<int64_t>(head) * a.q_head_stride;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const uint32_t d = s * 16 + h * 8;
        q[s] = Vec<T, 8>{};
        if (d < a.head_dim) q[s] = *reinterpret_cast<const Vec<T, 8>*>(qp + d);
    }
    const T* kp = static_cast<const T*>(a.k) + static_cast<int64_t>(sq.k0) * a.k_stride + static_cast<int64_t>(kvh) * a.k_head_stride;
    const T* vp = static_cast<const T*>(a.v) + static_cast<int64_t>(sq.k0) * a.v_stride + static_cast<int64_t>(kvh) * a.v_head_stride;

    f32x16 o[DP / 32];
    float top, sum;
    auto clear = [&] {
        top = NONE;
        sum = 0.0f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[d] = f32x16{};
    };
    const float scale = a.scale * LOG2E;
    // one tile of keys; Masked: some row of the workgroup does not see all of them
    auto step = [&](uint32_t j0, auto Masked, auto Careful) {
        constexpr bool masked = decltype(Masked)::value, careful = decltype(Careful)::value;
        __syncthreads();
        for (int at = threadIdx.x; at < BN * CH; at += 256) {
            const int r = at / CH, c = at % CH;
            Vec<T, 8> x = {}, y = {};
            if (j0 + r < sq.nk && static_cast<uint32_t>(c * 8) < a.head_dim) {
                x = *reinterpret_cast<const Vec<T, 8>*>(kp + static_cast<int64_t>(j0 + r) * a.k_stride + c * 8);
                y = *reinterpret_cast<const Vec<T, 8>*>(vp + static_cast<int64_t>(j0 + r) * a.v_stride + c * 8);
            }
            *reinterpret_cast<Vec<T, 8>*>(tk + place<S>(r, c)) = x;
            *reinterpret_cast<Vec<T, 8>*>(tv + place<S>(r, c)) = y;
        }
        __syncthreads();
        f32x16 z[2] = {};
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const Vec<T, 8> k = *reinterpret_cast<const Vec<T, 8>*>(tk + place<S>(b * 32 + l, s * 2 + h));
                z[b] = Mma<T>::go(k, q[s], z[b]);
            }
        // result register r of block b: key b * 32 + r % 4 + 8 (r / 4) + 4 h
        float most = NONE;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t j = j0 + b * 32 + (r & 3) + 8 * (r >> 2) + 4 * h;
                z[b][r] *= scale;
                if (masked && (j >= mine || j >= ke)) z[b][r] = NONE;
                most = fmaxf(most, z[b][r]);
            }
        most = fmaxf(most, __shfl_xor(most, 32));
        const float now = fmaxf(top, most);
        const float base = now == NONE ? 0.0f : now;  // nothing visible yet: every weight is exp2(-inf) = 0
        const float fade = exp2f(top - base);
        float add = 0.0f;
        Vec<T, 8> w[4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = exp2f(z[b][r] - base);
                add += e;
                w[b * 2 + (r >> 3)][r & 7] = static_cast<T>(e);
            }
        add += __shfl_xor(add, 32);
        sum = fmaf(sum, fade, add);
        top = now;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] *= fade;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
            Vec<T, 8> v[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                // lanes 16g .. 16g + 15 read 4 keys x 16 elements and get an element's 4 keys each
                const int key = s * 16 + h * 4 + ((lane & 15) >> 2), e = d * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
                const s16x4 lo = read_transposed(tv + place<S>(key, e >> 3) + (e & 7) * 2);
                const s16x4 hi = read_transposed(tv + place<S>(key + 8, e >> 3) + (e & 7) * 2);
                v[s] = __builtin_bit_cast(Vec<T, 8>, Vec<short, 8>{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
                if (!careful) o[d] = Mma<T>::go(v[s], w[s], o[d]);
            }
            if (careful) {
                // a weight of 0 times NaN or an infinity is NaN: what is not finite is left out of the product and
                // its kind brought in where the weights of such values sum to more than 0
                for (int kind = 0; kind < 4; ++kind) {
                    f32x16 c = {};
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        Vec<T, 8> x;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float f = static_cast<float>(v[s][i]);
                            const int is = f != f ? 1 : f == INFINITY ? 2 : f == NONE ? 3 : 0;
                            x[i] = static_cast<T>(kind == 0 ? (is ? 0.0f : f) : is == kind ? 1.0f : 0.0f);
                        }
                        c = Mma<T>::go(x, w[s], c);
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        o[d][r] += kind == 0 ? c[r] : !(c[r] > 0.0f) ? 0.0f : kind == 1 ? NAN : kind == 2 ? INFINITY : NONE;
                }
            }
        }
    };
    // The tiles that some row does not see whole come first, on a state of zeros: if a result is then not
    // finite, they are taken again with care, so that a row is never touched by a value it does not see.
    const uint32_t seen = keys_of(static_cast<uint32_t>(row0 / p.group));  // by every row of the tile
    const uint32_t full = max(kb, min(ke, seen) / BN * BN);                // kb and pieces are multiples of BN
    clear();
    for (uint32_t j0 = full; j0 < ke; j0 += BN) step(j0, std::true_type(), std::false_type());
    if (full < ke) {
        bool odd = false;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) odd |= !(fabsf(o[d][r]) < INFINITY);
        if (__syncthreads_or(odd)) {
            clear();
            for (uint32_t j0 = full; j0 < ke; j0 += BN) step(j0, std::true_type(), std::true_type());
        }
    }
    for (uint32_t j0 = kb; j0 < full; j0 += BN) step(j0, std::false_type(), std::false_type());
    if (!live) return;
    const int64_t at = static_cast<int64_t>(sq.q0 + tok) * a.heads + head;
    if (p.splits > 1) {
        const int64_t slot = static_cast<int64_t>(blockIdx.y) * a.q_tokens * a.heads + at;
        if (h == 0) p.part_stat[slot] = make_float2(top, sum);
        float* out = p.part_out + slot * a.head_dim;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t e = d * 32 + r * 8 + h * 4;
                if (e < a.head_dim) *reinterpret_cast<f32x4*>(out + e) = f32x4{o[d][r * 4], o[d][r * 4 + 1], o[d][r * 4 + 2], o[d][r * 4 + 3]};
            }
        return;
    }
    const float over = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(sq.q0 + tok) * a.out_stride + static_cast<int64_t>(head) * a.out_head_stride;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t e = d * 32 + r * 8 + h * 4;
            Vec<T, 4> v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = static_cast<T>(o[d][r * 4 + i] * over);
            if (e < a.head_dim) *reinterpret_cast<Vec<T, 4>*>(out + e) = v;
        }
    if (a.lse && h == 0) a.lse[at] = sum == 0.0f ? NONE : (top + log2f(sum)) * LN2;
}

// joins the pieces of a row: a wave per (query token, head)
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Params p) {
    const bs_attention_args& a = p.a;
    const int lane = threadIdx.x & 63;
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6), rows = static_cast<uint64_t>(a.q_tokens) * a.heads;
    if (at >= rows) return;
    const uint32_t tok = static_cast<uint32_t>(at / a.heads), head = static_cast<uint32_t>(at % a.heads);
    uint32_t seq = 0;
    if (a.q_offsets) {
        // the last sequence that starts at or before the token and holds it
        uint32_t lo = 0, hi = a.sequences;
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo + 63) / 64, x = lo + lane * step;
            const int k = __popcll(__ballot(x < hi && static_cast<uint32_t>(max(a.q_offsets[x], 0)) <= tok));
            lo += (k > 0 ? k - 1 : 0) * step;
            hi = min(lo + step, hi);
        }
        seq = lo;
    }
    const Sequence sq = sequence(a, seq);
    if (tok < sq.q0 || tok - sq.q0 >= sq.nq) return;
    int64_t e = a.causal ? min(static_cast<int64_t>(sq.nk), static_cast<int64_t>(tok - sq.q0) + sq.nk - sq.nq + 1) : static_cast<int64_t>(sq.nk);
    const uint32_t keys = e < 0 ? 0 : static_cast<uint32_t>(e);
    const uint32_t n = max(1u, min(p.splits, (keys + p.piece - 1) / p.piece));
    float top = NONE, sum = 0.0f, o[2] = {0.0f, 0.0f};
    const uint32_t d = lane * 2;
    for (uint32_t s = 0; s < n; ++s) {
        const uint64_t slot = s * rows + at;
        const float2 st = p.part_stat[slot];
        const float now = fmaxf(top, st.x), base = now == NONE ? 0.0f : now;
        const float fade = exp2f(top - base), gain = exp2f(st.x - base);
        sum = sum * fade + st.y * gain;
        top = now;
        if (d < a.head_dim) {
            const float2 v = *reinterpret_cast<const float2*>(p.part_out + slot * a.head_dim + d);
            o[0] = o[0] * fade + v.x * gain;
            o[1] = o[1] * fade + v.y * gain;
        }
    }
    const float over = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(tok) * a.out_stride + static_cast<int64_t>(head) * a.out_head_stride;
    if (d < a.head_dim) {
        const Vec<T, 2> v = {static_cast<T>(o[0] * over), static_cast<T>(o[1] * over)};
        *reinterpret_cast<Vec<T, 2>*>(out + d) = v;
    }
    if (a.lse && lane == 0) a.lse[at] = sum == 0.0f ? NONE : (top + log2f(sum)) * LN2;
}

uint64_t tiles_of(const bs_attention_args& a, uint32_t rows) {
    const uint64_t t = static_cast<uint64_t>(a.q_tokens) * (a.heads / a.kv_heads);
    return t / rows + a.sequences;
}

// pieces of the keys: enough workgroups for the chip, pieces of 256 keys at least
void split(const bs_attention_args& a, uint32_t& splits, uint32_t& piece) {
    const uint64_t groups = tiles_of(a, 128) * a.kv_heads;
    const uint32_t longest = a.longest_k ? std::min(a.longest_k, a.k_tokens) : a.k_tokens;
    splits = 1;
    piece = 0;
    if (groups >= 2 * CUS || longest <= 512) return;
    const uint64_t want = std::min<uint64_t>((4 * CUS + groups - 1) / groups, (longest + 255) / 256);
    piece = static_cast<uint32_t>(((longest + want - 1) / want + BN - 1) / BN * BN);
    splits = (longest + piece - 1) / piece;
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
    if (!(std::fabs(a->scale) < INFINITY)) return refuse(w + ": scale must be finite");
    if (tiles_of(*a, 128) * a->kv_heads > 0x7FFFFFFFull) return refuse(w + ": too many tiles for one launch");
    return BS_OK;
}

template <typename T>
void launch(const Params& p, hipStream_t s) {
    const dim3 grid(static_cast<uint32_t>(tiles_of(p.a, 128) * p.a.kv_heads), p.splits);
    if (p.a.head_dim <= 32)
        attention_kernel<T, 32><<<grid, 256, 0, s>>>(p);
    else if (p.a.head_dim <= 64)
        attention_kernel<T, 64><<<grid, 256, 0, s>>>(p);
    else if (p.a.head_dim <= 96)
        attention_kernel<T, 96><<<grid, 256, 0, s>>>(p);
    else
        attention_kernel<T, 128><<<grid, 256, 0, s>>>(p);
    if (p.splits > 1) {
        const uint64_t rows = static_cast<uint64_t>(p.a.q_tokens) * p.a.heads;
        join_kernel<T><<<static_cast<uint32_t>((rows + 3) / 4), 256, 0, s>>>(p);
    }
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
    split(a, p.splits, p.piece);
    if (p.splits > 1) {
        const uint64_t need = workspace_of(a);
        if (!workspace || workspace_bytes < need) return refuse("bs_attention: the workspace must hold " + std::to_string(need) + " bytes");
        if (!aligned16(workspace)) return refuse("bs_attention: the workspace must be 16-byte aligned");
        p.part_out = static_cast<float*>(workspace);
        p.part_stat = reinterpret_cast<float2*>(p.part_out + static_cast<uint64_t>(p.splits) * a.q_tokens * a.heads * a.head_dim);
    }
    a.type == BS_F16 ? launch<f16>(p, static_cast<hipStream_t>(stream)) : launch<bf16>(p, static_cast<hipStream_t>(stream));
    return launched("bs_attention");
} catch (...) {
    return bs_internal_exception();
}
