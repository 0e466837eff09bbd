// ns_attn.hip -- attention over the paged key/value cache (ns_kv.hpp), for single tokens, prompts
// and batches of both, and for batches whose sequences share a prefix.
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(scale q_r.k_j - m_r),  over the keys j that row r sees
//
// in one pass over the keys with a running maximum m and sum l per row (fp32).  A row is one query
// head of one new token; the G = q_heads / kv_heads heads that share a key head and all new tokens of
// a sequence are rows of one product, so a key is read once for all of them.
//
// All kernels form S^T = K Q^T and O^T = V^T P^T on the matrix cores.  A lane then holds one row r
// (a column of S^T) and several keys; the rows of the K operand are permuted so that these keys are
// the consecutive ones which the same lane feeds back as the P^T operand of the second product: P
// never leaves its lane, and the statistics of a row need one or two lane exchanges.
//
// Work that is split over the keys leaves parts (O unnormalised, m as a score before the scale, l) in the
// workspace.  Parts are joined in part order, so results do not depend on the order of arrival, by the last
// workgroup of a sequence and key head to arrive (few rows) or by a launch of its own (tiles).  No
// workgroup waits for another.
#include <algorithm>

#include "ns_internal.hpp"
#include "ns_kv.hpp"

namespace ns {
namespace {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.44269504088896340736f;
// P is held times a power of two, and the maximum that a row's scores are taken against may lag behind the true one by
// kLag powers of two: O and l are then rescaled a few times in a row's run instead of whenever its maximum
// creeps up.  P <= 2^(bias + lag) has to stay below fp16's 65504.  As two fp16 P keeps 22 bits down to 2^-28 of the
// maximum, and what falls below is less than fp32's own rounding over any number of keys that fits the cache;
// as one it keeps its 11 bits down to 2^-22, and 2^18 keys below 2^-33 come to 2^-15 of the sum, against 2^-11 of
// the output's own rounding.  One fp16 is taken by the row tiles of fp16 outputs, those of a shared prefix among them, also
// where each sequence has few rows of its own: as two, 64 sequences on a prefix of 32,768 take 135 us instead of 107
// (128-dim heads, 4 tokens each: 207 instead of 159).
template <bool HILO>
constexpr float kBias = HILO ? 14.0f : 9.0f;
template <bool HILO>
constexpr float kLag = HILO ? 1.5f : 6.0f;
template <bool HILO>
constexpr float kUnbias = HILO ? 0x1p-14f : 0x1p-9f;  // parts are kept without the bias: both kinds may meet in a join
// P = 2^(c1 s - (c1 m - bias)) is one operation a score.  What is in brackets is rounded, by 2^-15 while c1 |m| is at most
// kFar; far above it the rounding would move P by whole powers of two (past 65504, or to nothing).  There s - m is
// formed first, exact for the scores that weigh: a wave with such a row, or with one that has seen nothing yet (m = -inf, its
// scores as well: 0 is subtracted), takes the branch of a raised maximum for every tile.  Parts are compared by m
// itself for the same reason.  (2,048 tokens at 32,768 keys 1,028 -> 1,034 us, 157 tokens 22.4 -> 22.7, against always the
// one operation.)  The step stands in each kernel: as a function over their scores and O it takes 10 to 20 registers
// more, and the 256-dim instances spill 60 bytes a lane and more.
constexpr float kFar = 1024.0f;
// The |m| from which a row is far.  Formed in the kernel: a launch argument more costs each of them some .2 us.
__device__ __forceinline__ float far_max(float c1) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, kFar * __builtin_amdgcn_rcpf(c1))));
}
constexpr uint32_t kRowsMax = 16;  // rows of a sequence and key head up to which the few-row kernel takes them

struct AttnArgs {
    KvArgs kv;
    const uint16_t *q;
    void *out;
    float *rows;   // parts: row i's O at rows[i * D]
    float *stats;  // and its (m, l) at stats[2 * i]
    uint32_t *counters;
    uint32_t q_heads, group, window, prefix;
    float c1, v_scale;  // c1 = scale * k_scale * log2(e)
    int half_out;
    uint32_t target, min_tiles;  // few-row kernel: parts of the batch per key head, least key tiles of a part
    uint32_t row_cap;            // rows a part has room for
    uint32_t parts;              // tile kernel: key parts of a row tile
    int skip_small;              // tile kernel: sequences of at most kRowsMax rows are the few-row kernel's
    uint4 *tokens;               // separate join of the few-row kernel's parts: what it left for each token
    uint32_t row_slots;
    uint64_t pre_row;            // first row of the prefix's parts; its part p, head h, row r is
    uint32_t pre_parts, pre_rows;  //   pre_row + (p * kv_heads + h) * pre_rows + r
};

// All LDS of a workgroup: its size is a launch's choice, and one launch may hold workgroups of two kinds.
extern __shared__ __align__(16) uint8_t smem[];

__device__ __forceinline__ float exp2f_fast(float x) { return __builtin_amdgcn_exp2f(x); }

template <bool STREAM>
__device__ __forceinline__ u32x4 load16(const uint8_t *p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
    else return *reinterpret_cast<const u32x4 *>(p);
}

// Eight fp16 from a 16-byte chunk: the chunk itself, or half `u` of 16 e4m3 values (exact).
template <bool E4M3>
__device__ __forceinline__ half8_t chunk_half(const u32x4 &c, int u) {
    if constexpr (!E4M3) {
        return __builtin_bit_cast(half8_t, c);
    } else {
        const uint32_t a = c[2 * u], b = c[2 * u + 1];
        const half2_t v0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false), v1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
        const half2_t v2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false), v3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
        return half8_t{v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
    }
}

// Used inside an `if` on a value that it changes: keeps the branch (the compiler would otherwise do the work
// always and select).
template <class T>
__device__ __forceinline__ void keep_branch(T &v) {
    asm volatile("" : "+v"(v));
}

// Parts are written through to memory and read from there: the workgroup that joins them may run on
// another XCD, whose L2 does not see this one's.
__device__ __forceinline__ void store2(float *p, float a, float b) {
    const uint64_t v = uint64_t(__builtin_bit_cast(uint32_t, a)) | (uint64_t(__builtin_bit_cast(uint32_t, b)) << 32);
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load2(const float *p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return float2{__builtin_bit_cast(float, uint32_t(v)), __builtin_bit_cast(float, uint32_t(v >> 32))};
}

// Four consecutive dims of one row of the output.
template <int D>
__device__ __forceinline__ void write_out(const AttnArgs &a, uint32_t token, uint32_t head, uint32_t dim, const float4 &v) {
    const uint64_t at = (uint64_t(token) * a.q_heads + head) * D + dim;
    if (a.half_out)
        *reinterpret_cast<half4_t *>(static_cast<_Float16 *>(a.out) + at) = half4_t{_Float16(v.x), _Float16(v.y), _Float16(v.z), _Float16(v.w)};
    else
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) = v;
}

// The parts of one row of (sequence, key head): part p < own has it at own_row + p * own_step, the prefix's follow.
struct Parts {
    uint32_t own, n;
    uint64_t own_row, own_step, pre_row, pre_step;
    __device__ __forceinline__ uint64_t at(uint32_t p) const { return p < own ? own_row + p * own_step : pre_row + (p - own) * pre_step; }
};

constexpr uint32_t kPartsMax = 512;  // parts of a row that a plan makes at most

// Joins the parts of a sequence's `rows` rows by one workgroup of 256: a thread adds four dims of a row over the
// parts, or over every ng-th of them where the rows leave threads over (red: 256 float4, red_ml: 16 pairs of
// LDS).  Sixteen parts' statistics and values are in flight at once: the parts come from memory, some 2 us away.
template <int D>
__device__ void join_rows(const AttnArgs &a, const Parts &ps, uint32_t rows, uint32_t token0, uint32_t kv_head, float4 *red, float2 *red_ml) {
    constexpr int B = 16;
    const uint32_t tid = threadIdx.x, cols = rows * (D / 4), ng = max(1u, 256 / cols);
    for (uint32_t c = tid; c < cols * ng; c += 256) {
        const uint32_t gi = c / cols, it = c % cols, r = it / (D / 4), d = it % (D / 4) * 4;
        float M = -__builtin_inff(), l = 0.f;
        float4 o{0.f, 0.f, 0.f, 0.f};
        for (uint32_t p0 = gi; p0 < ps.n; p0 += B * ng) {
            float2 st[B], x[B], y[B];
#pragma unroll
            for (int u = 0; u < B; ++u) {
                const uint32_t p = p0 + u * ng;
                st[u] = float2{-__builtin_inff(), 0.f};
                x[u] = y[u] = float2{0.f, 0.f};
                if (p < ps.n) {
                    const uint64_t at = ps.at(p) + r;
                    st[u] = load2(a.stats + 2 * at);
                    x[u] = load2(a.rows + at * D + d);
                    y[u] = load2(a.rows + at * D + d + 2);
                }
            }
            float top = M;
#pragma unroll
            for (int u = 0; u < B; ++u) top = __builtin_fmaxf(top, st[u].x);
            const float zero = top == -__builtin_inff() ? 0.f : top;  // parts that see nothing of this row
            const float f = exp2f_fast((M - zero) * a.c1);
            M = top;
            l *= f;
            o = float4{o.x * f, o.y * f, o.z * f, o.w * f};
#pragma unroll
            for (int u = 0; u < B; ++u) {
                const float w = exp2f_fast((st[u].x - zero) * a.c1);
                l = __builtin_fmaf(w, st[u].y, l);
                o.x = __builtin_fmaf(w, x[u].x, o.x);
                o.y = __builtin_fmaf(w, x[u].y, o.y);
                o.z = __builtin_fmaf(w, y[u].x, o.z);
                o.w = __builtin_fmaf(w, y[u].y, o.w);
            }
        }
        if (ng > 1) {
            red[c] = o;
            if (d == 0) red_ml[gi * rows + r] = float2{M, l};
        } else {
            const float f = a.v_scale / l;
            write_out<D>(a, token0 + r / a.group, kv_head * a.group + r % a.group, d, float4{o.x * f, o.y * f, o.z * f, o.w * f});
        }
    }
    if (ng == 1) return;
    __syncthreads();
    if (tid < cols) {
        const uint32_t r = tid / (D / 4);
        float M = -__builtin_inff(), l = 0.f;
        for (uint32_t i = 0; i < ng; ++i) M = __builtin_fmaxf(M, red_ml[i * rows + r].x);
        float4 o{0.f, 0.f, 0.f, 0.f};
        for (uint32_t i = 0; i < ng; ++i) {
            const float2 s = red_ml[i * rows + r];
            const float4 x = red[i * cols + tid];
            const float w = exp2f_fast((s.x - M) * a.c1);
            l = __builtin_fmaf(w, s.y, l);
            o = float4{__builtin_fmaf(w, x.x, o.x), __builtin_fmaf(w, x.y, o.y), __builtin_fmaf(w, x.z, o.z), __builtin_fmaf(w, x.w, o.w)};
        }
        const float f = a.v_scale / l;
        write_out<D>(a, token0 + r / a.group, kv_head * a.group + r % a.group, tid % (D / 4) * 4, float4{o.x * f, o.y * f, o.z * f, o.w * f});
    }
}

// Four dims of a row over its parts, in part order, by one thread: eight parts in flight, their maximum, their sums.
template <int D>
__device__ __forceinline__ void join_row(const AttnArgs &a, const Parts &ps, uint32_t r, uint32_t d, uint32_t token, uint32_t qhead) {
    float M = -__builtin_inff(), l = 0.f;
    float4 o{0.f, 0.f, 0.f, 0.f};
    for (uint32_t p0 = 0; p0 < ps.n; p0 += 8) {  // eight parts in flight, their maximum, then their sums
        float2 st[8];
        float4 x[8];
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u) {
            st[u] = float2{-__builtin_inff(), 0.f};
            x[u] = float4{0.f, 0.f, 0.f, 0.f};
            if (p0 + u < ps.n) {
                const uint64_t i = ps.at(p0 + u) + r;
                st[u] = *reinterpret_cast<const float2 *>(a.stats + 2 * i);
                x[u] = *reinterpret_cast<const float4 *>(a.rows + i * D + d);
            }
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < 8; ++u) top = __builtin_fmaxf(top, st[u].x);
        const float zero = top == -__builtin_inff() ? 0.f : top;  // parts that see nothing of this row: M stays -inf
        const float f = exp2f_fast((M - zero) * a.c1);
        l *= f;
        o = float4{o.x * f, o.y * f, o.z * f, o.w * f};
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float w = exp2f_fast((st[u].x - zero) * a.c1);
            l = __builtin_fmaf(w, st[u].y, l);
            o.x = __builtin_fmaf(w, x[u].x, o.x);
            o.y = __builtin_fmaf(w, x[u].y, o.y);
            o.z = __builtin_fmaf(w, x[u].z, o.z);
            o.w = __builtin_fmaf(w, x[u].w, o.w);
        }
        M = top;
    }
    const float f = a.v_scale / l;
    write_out<D>(a, token, qhead, d, float4{o.x * f, o.y * f, o.z * f, o.w * f});
}

// True in the workgroup that arrives last of `parts`; its parts and everyone's are then in memory.
__device__ __forceinline__ bool last_arrival(uint32_t *counter, uint32_t parts, uint32_t *flag) {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t prev = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = prev == parts - 1;
        if (prev == parts - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *flag != 0;
}

// NaN rows of a sequence whose description does not hold.
template <int D>
__device__ void write_nan(const AttnArgs &a, uint32_t row0, uint32_t rows, uint32_t token0, uint32_t kv_head) {
    const float nan = __builtin_nanf("");
    for (uint32_t it = threadIdx.x; it < rows * (D / 4); it += blockDim.x) {
        const uint32_t gr = row0 + it / (D / 4);
        write_out<D>(a, token0 + gr / a.group, kv_head * a.group + gr % a.group, it % (D / 4) * 4, float4{nan, nan, nan, nan});
    }
}

// Inclusive sum over the lanes of a wave (data-parallel primitives: a fifth of the latency of shuffles).
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    int v = int(x);
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return uint32_t(v);
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return uint32_t(__builtin_amdgcn_readlane(int(v), lane)); }

// ---- few rows: at most 16 rows (new tokens times heads of the group) of a sequence -----------------------
//
// v_mfma_f32_16x16x32_f16.  A wave takes key tiles of 4 c keys (c a chunk's elements: 32 fp16 keys, 64
// e4m3) straight from memory into registers: lane l holds row l % 16 of the operand and the chunk of
// group g = l / 16.  Row m of K row tile t is key c (m / 4) + 4 t + m % 4, so lane l's scores are those of
// keys c g ... c g + c - 1, the chunk of V that it reads.  The next tile's K loads are issued before
// the softmax of this one.  Bound by the bytes of K and V: fp16, 256 dims, 8 key heads, one token at 262,144 keys
// 319-336 us a call on different boxes (6.4-6.7 TB/s; 320 us the shortest launch in a trace of the 319 us one), 32
// sequences up to 8,192 keys 197 us (5.6 TB/s).  Short calls are bound by a chain of
// dependent steps: one token at 2,206 keys 9.2 us, of which 2.5 until the first K is asked for (lengths, scan over the
// sequences, table entry), 1.8 for loads and products, .9 to join the waves, 1.8 for the parts' way to memory and
// the count, 2.2 for the join.
// The four waves of a workgroup take a part's tiles in turn and join their O in LDS.
// UNI: pages hold whole key tiles, so a tile's page is one scalar and its loads take a scalar base.
// JOIN: the last workgroup of a sequence and key head joins its parts; otherwise they are left to attn_shared_join_kernel.
template <int D>
struct RowsLds {
    static constexpr uint32_t kQueries = kRowsMax * (D + 8) * 2, kRed = kQueries + 256 * 16, kRedMl = kRed + 16 * 8, kStats = kRedMl + 2 * 4 * kRowsMax * 4,
                              kFixed = kStats + 16;
    static constexpr uint32_t bytes(uint32_t row_cap) { return kFixed + 4 * row_cap * (D + 4) * 4; }
};
// STREAM: K and V are loaded as data that is not used again, which a single sequence's are (262,144 keys: 374 -> 336 us on
// one box, 360 -> 319 on another).
// Sequences may share pages, and find each other's in the caches (64 of them on a prefix of 32,768: 756 us, 1,787
// with such loads).
template <int D, bool E4M3, bool UNI, bool STREAM, bool JOIN>
__device__ __forceinline__ void attn_rows(const AttnArgs &a, uint32_t block) {
    constexpr int C = E4M3 ? 16 : 8, KT = 4 * C, NT = C / 4, U = C / 8, JS = D / (4 * C), DT = D / 16;
    using Lds = RowsLds<D>;
    uint16_t(&qs)[kRowsMax][D + 8] = *reinterpret_cast<uint16_t(*)[kRowsMax][D + 8]>(smem);  // rows 16 bytes apart in the banks
    float4 *red = reinterpret_cast<float4 *>(smem + Lds::kQueries);
    float2 *red_ml = reinterpret_cast<float2 *>(smem + Lds::kRed);
    float(&wm)[4][kRowsMax] = *reinterpret_cast<float(*)[4][kRowsMax]>(smem + Lds::kRedMl);
    float(&wl)[4][kRowsMax] = *reinterpret_cast<float(*)[4][kRowsMax]>(smem + Lds::kRedMl + 4 * kRowsMax * 4);
    uint32_t *flag = reinterpret_cast<uint32_t *>(smem + Lds::kStats);
    float *lds = reinterpret_cast<float *>(smem + Lds::kFixed);
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15u, g = lane >> 4;
    const uint32_t head = block % a.kv.kv_heads, slot = block / a.kv.kv_heads;

    // Key tiles of sequence s that its rows see.
    auto span = [&](const KvSeq &q, uint32_t &lo) {
        lo = a.prefix;
        if (a.window && q.kv - q.n + 1 > a.window) lo = q.kv - q.n + 1 - a.window;
        return (q.kv + KT - 1) / KT - lo / KT;
    };
    KvSeq q{};  // of sequence b + lane, then of the workgroup's
    auto tiles_of = [&](uint32_t i) -> uint32_t {
        if (i >= a.kv.seqs) return 0;
        q = kv_seq(a.kv, i, a.prefix);
        if (q.n == 0 || (q.ok && q.n * a.group > kRowsMax)) return 0;
        uint32_t lo;
        return q.ok ? span(q, lo) : 1;  // a contradicting one's rows are NaN, however many
    };
    // The batch's tiles are cut into parts of `chunk` tiles, about `target` parts whatever the lengths
    // are; workgroup `slot` finds its sequence and part by a scan over the sequences.
    uint32_t t = 0, total = 0;
    for (uint32_t b = 0; b < a.kv.seqs; b += 64) {
        t = tiles_of(b + lane);
        total += lane_value(wave_scan(t), 63);
    }
    const uint32_t chunk = max(a.min_tiles, (total + a.target - 1) / a.target);
    uint32_t s = 0, base = 0, parts = 0;
    bool found = false;
    for (uint32_t b = 0; b < a.kv.seqs && !found; b += 64) {
        if (a.kv.seqs > 64) t = tiles_of(b + lane);
        const uint32_t p = (t + chunk - 1) / chunk, incl = wave_scan(p);
        const uint64_t over = __ballot(base + incl > slot);
        if (over) {
            const int at = __builtin_ctzll(over);
            found = true;
            s = b + at;
            parts = lane_value(p, at);
            base += lane_value(incl, at) - parts;
            q.q0 = lane_value(q.q0, at);
            q.n = lane_value(q.n, at);
            q.kv = lane_value(q.kv, at);
            q.ok = lane_value(q.ok ? 1u : 0u, at) != 0;
        } else {
            base += lane_value(incl, 63);
        }
    }
    if (!found) return;
    const uint32_t part = slot - base;
    const uint32_t rows = q.n * a.group;
    if (!JOIN && part == 0 && head == 0)
        for (uint32_t i = tid; i < q.n; i += 256) a.tokens[q.q0 + i] = uint4{base, q.ok ? parts : 0u, q.q0 * a.group, 0u};
    if (!q.ok) {
        write_nan<D>(a, 0, rows, q.q0, head);
        return;
    }
    uint32_t lo;
    const uint32_t ntile = span(q, lo), tile0 = lo / KT;
    const uint32_t first = tile0 + part * chunk, end = tile0 + min(ntile, (part + 1) * chunk);

    const uint32_t limit = q.kv - q.n + min(col, rows - 1) / a.group;  // this lane's row sees keys up to here
    const uint32_t least = a.window && limit + 1 > a.window ? max(limit + 1 - a.window, a.prefix) : a.prefix;

    const int32_t *table = a.kv.table + uint64_t(s) * a.kv.stride;
    const uint32_t smask = (1u << a.kv.page_shift) - 1;
    bool bad = false;
    // A tile's page (UNI), or that of the 4-key run that this lane reads of K (group col / 4) and of its chunk of
    // V (group g).  Past the sequence's ends the nearest page is taken: those keys are masked.
    auto page_of = [&](uint32_t key) {
        const uint32_t e = min(max(key, lo), q.kv - 1) >> a.kv.page_shift;
        if constexpr (UNI) return uint32_t(((const __attribute__((address_space(4))) int32_t *)table)[__builtin_amdgcn_readfirstlane(e)]);
        else return uint32_t(table[e]);
    };
    auto checked = [&](uint32_t p) {
        bad |= p >= a.kv.pages;
        return p < a.kv.pages ? p : 0u;
    };

    float4_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = float4_t{0.f, 0.f, 0.f, 0.f};
    const float far_m = far_max(a.c1);
    float m = -__builtin_inff(), l = 0.f;
    u32x4 kf[NT][JS], vf[DT];

    // Slots of the lane's K rows and V chunk inside the tile's page
    const uint32_t kslot = C * (col / 4) + col % 4, vslot = C * g;
    auto load_k = [&](uint32_t tile, uint32_t page) {
        const uint64_t at = kv_offset<D, E4M3>(a.kv, page, head);
        if constexpr (UNI) {
            const uint8_t *p = a.kv.k + at + ((tile * KT) & smask) * 16;  // scalar
            const uint32_t off = ((g << a.kv.page_shift) + kslot) * 16;
#pragma unroll
            for (int j = 0; j < JS; ++j)
#pragma unroll
                for (int i = 0; i < NT; ++i)
                    kf[i][j] = load16<STREAM>(p + ((uint64_t(4 * j) << a.kv.page_shift) + 4 * i) * 16 + off);
        } else {
            const uint32_t sl = (tile * KT + kslot) & smask;
            const uint8_t *p = a.kv.k + at + sl * 16 + (uint64_t(g) << a.kv.page_shift) * 16;
#pragma unroll
            for (int j = 0; j < JS; ++j)
#pragma unroll
                for (int i = 0; i < NT; ++i)
                    kf[i][j] = load16<STREAM>(p + ((uint64_t(4 * j) << a.kv.page_shift) + 4 * i) * 16);
        }
    };
    auto load_v = [&](uint32_t tile, uint32_t page) {
        const uint64_t at = kv_offset<D, E4M3>(a.kv, page, head);
        if constexpr (UNI) {
            const uint8_t *p = a.kv.v + at + ((tile * KT) & smask) * (D * 16 / C);  // scalar
            const uint32_t off = (g * D + col) * 16;
#pragma unroll
            for (int d = 0; d < DT; ++d) vf[d] = load16<STREAM>(p + off + d * 256);
        } else {
            const uint32_t sl = (tile * KT + vslot) & smask;
            const uint8_t *p = a.kv.v + at + (uint64_t(sl / C) * D + col) * 16;
#pragma unroll
            for (int d = 0; d < DT; ++d) vf[d] = load16<STREAM>(p + d * 256);
        }
    };

    // Table entries are loaded two tiles ahead: vector loads return in order, so an entry asked for after V
    // would hold the next K back until all of V is there.
    uint32_t tile = first + wave;
    auto k_entry = [&](uint32_t i) { return page_of(i * KT + (UNI ? 0 : C * (col / 4))); };
    auto v_entry = [&](uint32_t i) { return page_of(i * KT + (UNI ? 0 : C * g)); };
    const uint32_t pk0 = k_entry(tile);  // any tile's entry is one inside the sequence's
    uint32_t pv = v_entry(tile), pk = k_entry(tile + 4), pv1 = v_entry(tile + 4);
    // The queries wait in LDS: read again for every tile, they leave their registers to loads in flight.
    u32x4 qv[(kRowsMax * D / 8 + 255) / 256];
#pragma unroll
    for (uint32_t i = 0; i < kRowsMax * D / 8; i += 256) {
        const uint32_t it = min(i + tid, rows * (D / 8) - 1), r = it / (D / 8), d = it % (D / 8) * 8;
        qv[i / 256] = *reinterpret_cast<const u32x4 *>(a.q + (uint64_t(q.q0 + r / a.group) * a.q_heads + head * a.group + r % a.group) * D + d);
    }
    if (tile < end) load_k(tile, checked(pk0));
#pragma unroll
    for (uint32_t i = 0; i < kRowsMax * D / 8; i += 256) {
        const uint32_t it = i + tid, r = it / (D / 8), d = it % (D / 8) * 8;
        if (r < rows) *reinterpret_cast<u32x4 *>(&qs[r][d]) = qv[i / 256];
    }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the LDS writes; K stays in flight
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    uint32_t qat = min(col, rows - 1) * (D + 8);  // Q^T operand: lane holds row col
    for (; tile < end; tile += 4) {
        const uint32_t next = tile + 4;
        const uint32_t pk2 = k_entry(tile + 8), pv2 = v_entry(tile + 8);
        load_v(tile, checked(pv));
        // an opaque offset keeps the queries' loads in the loop, out of registers
        asm volatile("" : "+v"(qat));
        const uint16_t *qrow = &qs[0][0] + qat;
        float4_t sc[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) sc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < JS; ++j)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const half8_t qf = __builtin_bit_cast(half8_t, *reinterpret_cast<const u32x4 *>(qrow + (4 * j + g) * C + 8 * u));
#pragma unroll
                for (int i = 0; i < NT; ++i) sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(chunk_half<E4M3>(kf[i][j], u), qf, sc[i], 0, 0, 0);
            }
        if (next < end) load_k(next, checked(pk));
        pk = pk2;
        pv = pv1;
        pv1 = pv2;

        // lane's scores: keys key0 + 4 i + e of row col
        const uint32_t key0 = tile * KT + C * g;
        const bool edge = tile * KT < lo || tile * KT + KT > q.kv - q.n + 1 || (a.window && tile * KT + a.window < q.kv);
        if (edge) {
#pragma unroll
            for (int i = 0; i < NT; ++i) keep_branch(sc[i]);
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t key = key0 + 4 * i + e;
                    if (key > limit || key < least) sc[i][e] = -__builtin_inff();
                }
        }
        float top = sc[0][0];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = __builtin_fmaxf(top, sc[i][e]);
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float mn = __builtin_fmaxf(m, top);
        bool far = false;
        if (__ballot((mn - m) * a.c1 > kLag<true> || __builtin_fabsf(m) > far_m)) {  // some row's maximum left the lag (from -inf: infinitely)
            const float f = mn == m ? 1.f : exp2f_fast((m - mn) * a.c1);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
            m = mn;
            if (__ballot(__builtin_fabsf(m) > far_m)) {
                const float zero = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    keep_branch(sc[i]);
                    sc[i] -= zero;
                }
                far = true;
            }
        }
        const float mc = far ? -kBias<true> : __builtin_fmaf(m, a.c1, -kBias<true>);
        half8_t hi[U], lw[U];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = exp2f_fast(__builtin_fmaf(sc[i][e], a.c1, -mc));
                l += p;
                // P as the sum of two fp16 (22 bits): the second product adds less than fp32's own sums do,
                // and the matrix cores idle behind the loads here
                const _Float16 h = _Float16(p);
                hi[i / 2][(i % 2) * 4 + e] = h;
                lw[i / 2][(i % 2) * 4 + e] = _Float16(p - float(h));
            }
        if (edge) {  // slots outside the sequence may hold anything: 0 * NaN would reach the sums
#pragma unroll
            for (int d = 0; d < DT; ++d) keep_branch(vf[d]);
            uint32_t mask[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                mask[w] = 0;
#pragma unroll
                for (int e = 0; e < C / 4; ++e) {
                    const uint32_t key = key0 + w * (C / 4) + e;
                    if (key >= lo && key < q.kv) mask[w] |= (E4M3 ? 0xffu : 0xffffu) << (e * (E4M3 ? 8 : 16));
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int w = 0; w < 4; ++w) vf[d][w] &= mask[w];
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const half8_t v = chunk_half<E4M3>(vf[d], u);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi[u], o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lw[u], o[d], 0, 0, 0);
            }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (__ballot(bad)) l = __builtin_nanf("");  // a page outside the cache

    // ---- the waves' parts: common maximum, then the sum in wave order
    const uint32_t pitch = D + 4;
    if (g == 0) {
        wm[wave][col] = m;
        wl[wave][col] = l;
    }
    if (col < rows) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
            *reinterpret_cast<float4_t *>(&lds[(wave * a.row_cap + col) * pitch + d * 16 + 4 * g]) = o[d];
    }
    __syncthreads();
    const uint64_t own_row = (uint64_t(base) * a.kv.kv_heads + head) * a.row_cap, own_step = uint64_t(a.kv.kv_heads) * a.row_cap;
    const uint64_t my_row = own_row + part * own_step;
    const bool whole = JOIN && parts == 1 && a.pre_parts == 0;
    for (uint32_t it = tid; it < rows * (D / 4); it += 256) {
        const uint32_t r = it / (D / 4), d = it % (D / 4) * 4;
        const float M = __builtin_fmaxf(__builtin_fmaxf(wm[0][r], wm[1][r]), __builtin_fmaxf(wm[2][r], wm[3][r]));
        float L = 0.f;
        float4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = M == -__builtin_inff() ? 1.f : exp2f_fast(__builtin_fmaf(wm[w][r] - M, a.c1, -kBias<true>));
            const float4_t x = *reinterpret_cast<const float4_t *>(&lds[(w * a.row_cap + r) * pitch + d]);
            L = __builtin_fmaf(f, wl[w][r], L);
            acc.x = __builtin_fmaf(f, x[0], acc.x);
            acc.y = __builtin_fmaf(f, x[1], acc.y);
            acc.z = __builtin_fmaf(f, x[2], acc.z);
            acc.w = __builtin_fmaf(f, x[3], acc.w);
        }
        if (whole) {
            const float f = a.v_scale / L;
            write_out<D>(a, q.q0 + r / a.group, head * a.group + r % a.group, d, float4{acc.x * f, acc.y * f, acc.z * f, acc.w * f});
        } else {
            float *dst = a.rows + (my_row + r) * D + d;
            if constexpr (JOIN) {
                store2(dst, acc.x, acc.y);
                store2(dst + 2, acc.z, acc.w);
                if (d == 0) store2(a.stats + 2 * (my_row + r), M, L);
            } else {
                *reinterpret_cast<float4 *>(dst) = acc;
                if (d == 0) *reinterpret_cast<float2 *>(a.stats + 2 * (my_row + r)) = float2{M, L};
            }
        }
    }
    if (!JOIN || whole) return;
    if (!last_arrival(&a.counters[s * a.kv.kv_heads + head], parts, flag)) return;
    join_rows<D>(a, Parts{parts, parts + a.pre_parts, own_row, own_step, a.pre_row + uint64_t(head) * a.pre_rows + uint64_t(q.q0) * a.group,
                          uint64_t(a.kv.kv_heads) * a.pre_rows}, rows, q.q0, head, red, red_ml);
}
template <int D, bool E4M3, bool UNI, bool STREAM>
__global__ __launch_bounds__(256, 2) void attn_rows_kernel(AttnArgs a) {
    attn_rows<D, E4M3, UNI, STREAM, true>(a, blockIdx.x);
}

// A direct load of 16 bytes per lane into the 1 KiB of LDS at byte `lds`.  The builtin for it makes the compiler wait
// for every such load before it reads any LDS that it cannot tell apart, so the next tile's loads would never
// overlap this one's products; here the kernel's own waits order them.  (No destination registers; m0 needs a
// wait state before its use.)
__device__ __forceinline__ void dma16(const uint8_t *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}

// N of them (1, 2 or 4) from one scalar base: the i-th takes 16 bytes at base + off[i] + 1024 i to LDS byte lds + 1024 i +
// 16 lane (the instruction's offset counts on both sides, so m0 is set once).
template <int N>
__device__ __forceinline__ void dma16_run(const uint8_t *base, const uint32_t *off, uint32_t lds) {
    static_assert(N == 1 || N == 2 || N == 4, "");
    if constexpr (N == 1)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off[0]), "s"(base) : "memory", "m0");
    else if constexpr (N == 2)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024" ::"s"(lds),
                     "v"(off[0]), "v"(off[1]), "s"(base)
                     : "memory", "m0");
    else
        asm volatile(
            "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\tglobal_load_lds_dwordx4 %2, %5 offset:1024\n\t"
            "global_load_lds_dwordx4 %3, %5 offset:1024*2\n\tglobal_load_lds_dwordx4 %4, %5 offset:1024*3" ::"s"(lds),
            "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base)
            : "memory", "m0");
}

// l plus the sum of a lane's 16 P values as they enter the product, in fp32, two a step.  The dot product takes fp16's
// subnormals as they are (16,384 sums of them were exact); of 49,152 sums of other sizes 4.5% were not the nearest fp32, the
// worst off by 1.5 units in the last place, and chains of 4,096 by 5e-6 at most.
__device__ __forceinline__ float add_halves(const half8_t (&p)[2], float l) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 8; e += 2) l = __builtin_amdgcn_fdot2(half2_t{p[i][e], p[i][e + 1]}, half2_t{_Float16(1.f), _Float16(1.f)}, l, false);
    return l;
}

// The larger of this lane's and lane ^ 32's value.
__device__ __forceinline__ float max_halves(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __builtin_fmaxf(__builtin_bit_cast(float, uint32_t(r[0])), __builtin_bit_cast(float, uint32_t(r[1])));
}

// What a workgroup of the tile kernels works on: rows [row0, row_end) of sequence s (its first TM of them are the
// workgroup's), keys [lo, hi).
struct TileSpan {
    uint32_t s, row0, row_end, token0, lo, hi;
    uint32_t before;  // the position of the sequence's first row
};
// Finds row tile `slot` of TM rows; false where there is none, or its rows are done.  PREFIX: the rows of the whole
// batch against the shared prefix.
template <int D, int TM, bool PREFIX>
__device__ __forceinline__ bool tile_span(const AttnArgs &a, uint32_t slot, uint32_t part, uint32_t head, TileSpan &t) {
    if constexpr (PREFIX) {
        t = TileSpan{0, slot * TM, a.kv.tokens * a.group, 0, 0, a.prefix, 0};
        return true;
    } else {
        // Sequence s owns the row tiles from q_start[s] * G / TM + s on: room for each one's last, ragged tile.
        auto first_tile = [&](uint32_t i) {
            return uint32_t(uint64_t(min(uint32_t(max(a.kv.q_start[i], 0)), a.kv.tokens)) * a.group / TM) + i;
        };
        t.s = find_seq(a.kv.seqs, slot, first_tile);
        const KvSeq q = kv_seq(a.kv, t.s, a.prefix);
        t.row_end = q.n * a.group;
        const uint32_t at = slot - first_tile(t.s), tiles = (t.row_end + TM - 1) / TM;
        if (at >= tiles || (a.skip_small && (t.row_end <= kRowsMax || !q.ok))) return false;
        t.row0 = (tiles - 1 - at) * TM;  // the tiles with the most keys first
        t.token0 = q.q0;
        if (!q.ok) {
            if (part == 0) write_nan<D>(a, t.row0, min(uint32_t(TM), t.row_end - t.row0), t.token0, head);
            return false;
        }
        t.before = q.kv - q.n;
        t.hi = t.before + min(t.row0 + TM - 1, t.row_end - 1) / a.group + 1;
        t.lo = a.prefix;
        const uint32_t p0 = t.before + t.row0 / a.group;
        if (a.window && p0 + 1 > a.window) t.lo = max(t.lo, p0 + 1 - a.window);
        return true;
    }
}

// ---- some rows: one tile of 32 rows a workgroup ----------------------------------------------------------
//
// The tile kernel's products (v_mfma_f32_32x32x16_f16, the same operand orders) with the few-row kernel's loads: the
// four waves of a workgroup take a part's key tiles in turn, straight into registers, and join their O in LDS.
// For calls whose row tiles of 128 are too few to fill the chip: the keys are split four ways without parts in
// memory.  A wave of 256 dims holds 128 O, 128 K and V registers: one workgroup a CU.  Bound by the latency of its
// loads: 157 tokens on 2,205 keys, 16 heads on 8 of 256 dims, 17 us and 4 for the join (32 in row tiles of
// 128); the matrix pipe is busy 16% of the time.
template <int D>
struct MidLds {
    static constexpr uint32_t kQueries = 32 * (D + 8) * 2, kFixed = kQueries + 2 * 4 * 32 * 4, kBytes = kFixed + 4 * 32 * (D + 4) * 4;
};
template <int D, bool E4M3, bool UNI, bool HILO, bool PREFIX>
__device__ __forceinline__ void attn_mid(const AttnArgs &a, uint32_t block, uint32_t n_parts) {
    constexpr int C = E4M3 ? 16 : 8, U = C / 8, KT = 32, TM = 32, KL = D / (2 * C), DT = D / 32, NV = 2 / U;
    uint16_t(&qs)[TM][D + 8] = *reinterpret_cast<uint16_t(*)[TM][D + 8]>(smem);
    float(&wm)[4][TM] = *reinterpret_cast<float(*)[4][TM]>(smem + MidLds<D>::kQueries);
    float(&wl)[4][TM] = *reinterpret_cast<float(*)[4][TM]>(smem + MidLds<D>::kQueries + 4 * TM * 4);
    float *lds = reinterpret_cast<float *>(smem + MidLds<D>::kFixed);
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31u, hl = lane >> 5;
    const uint32_t head = block % a.kv.kv_heads, unit = block / a.kv.kv_heads, part = unit % n_parts, slot = unit / n_parts;
    TileSpan t;
    if (!tile_span<D, TM, PREFIX>(a, slot, part, head, t)) return;
    const uint32_t rows = min(uint32_t(TM), t.row_end - t.row0);
    const uint32_t tile_lo = t.lo / KT, tile_hi = (t.hi + KT - 1) / KT, per = (tile_hi - tile_lo + n_parts - 1) / n_parts;
    const uint32_t first = min(tile_lo + part * per, tile_hi), end = min(first + per, tile_hi);

    const uint32_t row = t.row0 + min(col, rows - 1);
    uint32_t limit, least, amin, amost;  // the keys that this lane's row sees, and bounds over the rows
    if constexpr (PREFIX) {
        limit = amin = t.hi - 1;
        least = amost = 0;
    } else {
        const uint32_t top = t.before + (t.row0 + rows - 1) / a.group;
        limit = t.before + row / a.group;
        least = a.window && limit + 1 > a.window ? max(limit + 1 - a.window, a.prefix) : a.prefix;
        amin = t.before + t.row0 / a.group;
        amost = a.window && top + 1 > a.window ? max(top + 1 - a.window, a.prefix) : a.prefix;
    }

    const int32_t *table = a.kv.table + uint64_t(t.s) * a.kv.stride;
    const uint32_t smask = (1u << a.kv.page_shift) - 1;
    bool bad = false;
    // The pages of a tile's two halves of 16 keys (one page where UNI); outside [lo, hi) the nearest page inside.
    auto page_of = [&](uint32_t key) {
        const uint32_t e = min(max(key, t.lo), t.hi - 1) >> a.kv.page_shift;
        return uint32_t(((const __attribute__((address_space(4))) int32_t *)table)[__builtin_amdgcn_readfirstlane(e)]);
    };
    auto offset = [&](uint32_t p) {
        bad |= p >= a.kv.pages;
        return kv_offset<D, E4M3>(a.kv, p < a.kv.pages ? p : 0u, head);
    };
    const uint32_t krow = E4M3 ? 16 * ((col / 4) % 2) + 4 * (col / 8) + col % 4 : 16 * (col / 16) + 8 * ((col / 4) % 2) + 4 * ((col / 8) % 2) + col % 4;
    u32x4 kf[KL], vf[NV][DT];
    auto load_k = [&](uint32_t tile) {
        const uint64_t oa = offset(page_of(tile * KT));
        if constexpr (UNI) {
            const uint8_t *p = a.kv.k + oa + ((tile * KT) & smask) * 16;  // scalar
            const uint32_t off = ((hl << a.kv.page_shift) + krow) * 16;
#pragma unroll
            for (int j = 0; j < KL; ++j) kf[j] = *reinterpret_cast<const u32x4 *>(p + (uint64_t(2 * j) << a.kv.page_shift) * 16 + off);
        } else {
            const uint64_t ob = offset(page_of(tile * KT + 16));
            const uint8_t *p = a.kv.k + (krow < 16 ? oa : ob) + ((tile * KT + krow) & smask) * 16 + (uint64_t(hl) << a.kv.page_shift) * 16;
#pragma unroll
            for (int j = 0; j < KL; ++j) kf[j] = *reinterpret_cast<const u32x4 *>(p + (uint64_t(2 * j) << a.kv.page_shift) * 16);
        }
    };
    auto load_v = [&](uint32_t tile) {
        const uint64_t oa = offset(page_of(tile * KT));
        if constexpr (UNI) {
            const uint8_t *p = a.kv.v + oa + ((tile * KT) & smask) * (D * 16 / C);  // scalar
            const uint32_t off = (hl * D + col) * 16;
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int d = 0; d < DT; ++d) vf[n][d] = *reinterpret_cast<const u32x4 *>(p + off + (n * 2 * D + d * 32) * 16);
        } else {
            const uint64_t ob = offset(page_of(tile * KT + 16));
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const uint32_t k = E4M3 ? 16 * hl : 16 * n + 8 * hl;  // the chunk's first key in the tile
                const uint8_t *p = a.kv.v + (k < 16 ? oa : ob) + (uint64_t(((tile * KT + k) & smask) / C) * D + col) * 16;
#pragma unroll
                for (int d = 0; d < DT; ++d) vf[n][d] = *reinterpret_cast<const u32x4 *>(p + d * 512);
            }
        }
    };

    uint32_t tile = first + wave;
    u32x4 qv[TM * D / 8 / 256];
#pragma unroll
    for (uint32_t i = 0; i < TM * D / 8; i += 256) {
        const uint32_t it = min(i + tid, rows * (D / 8) - 1), r = t.row0 + it / (D / 8), d = it % (D / 8) * 8;
        qv[i / 256] = *reinterpret_cast<const u32x4 *>(a.q + (uint64_t(t.token0 + r / a.group) * a.q_heads + head * a.group + r % a.group) * D + d);
    }
    if (tile < end) load_k(tile);
#pragma unroll
    for (uint32_t i = 0; i < TM * D / 8; i += 256) {
        const uint32_t it = i + tid, r = it / (D / 8), d = it % (D / 8) * 8;
        if (r < rows) *reinterpret_cast<u32x4 *>(&qs[r][d]) = qv[i / 256];
    }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the LDS writes; K stays in flight
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    uint32_t qat = min(col, rows - 1) * (D + 8);

    float16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = float16_t{};
    const float far_m = far_max(a.c1);
    float m = -__builtin_inff(), l = 0.f;
    for (; tile < end; tile += 4) {
        load_v(tile);
        asm volatile("" : "+v"(qat));  // keeps the queries' loads in the loop, out of registers
        const uint16_t *qrow = &qs[0][0] + qat;
        float16_t sc = float16_t{};
#pragma unroll
        for (int j = 0; j < KL; ++j)
#pragma unroll
            for (int u = 0; u < U; ++u)
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                    chunk_half<E4M3>(kf[j], u), __builtin_bit_cast(half8_t, *reinterpret_cast<const u32x4 *>(qrow + (2 * j + hl) * C + 8 * u)), sc, 0, 0, 0);
        if (tile + 4 < end) load_k(tile + 4);
        const uint32_t t0 = tile * KT;
        const bool edge = t0 < amost || t0 + KT > amin + 1;
        auto key_of = [&](int v) { return E4M3 ? t0 + 16 * hl + uint32_t(v) : t0 + 16 * uint32_t(v / 8) + 8 * hl + uint32_t(v % 8); };
        if (edge) {
            keep_branch(sc);
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const uint32_t key = key_of(v);
                if (key > limit || key < least) sc[v] = -__builtin_inff();
            }
        }
        float top = sc[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) top = __builtin_fmaxf(top, sc[v]);
        top = max_halves(top);
        const float mn = __builtin_fmaxf(m, top);
        bool far = false;
        if (__ballot((mn - m) * a.c1 > kLag<HILO> || __builtin_fabsf(m) > far_m)) {
            const float f = mn == m ? 1.f : exp2f_fast((m - mn) * a.c1);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
            m = mn;
            if (__ballot(__builtin_fabsf(m) > far_m)) {
                const float zero = m == -__builtin_inff() ? 0.f : m;
                keep_branch(sc);
                sc -= zero;
                far = true;
            }
        }
        const float mc = far ? -kBias<HILO> : __builtin_fmaf(m, a.c1, -kBias<HILO>);
        half8_t ph[2], pl[2];
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const float p = exp2f_fast(__builtin_fmaf(sc[v], a.c1, -mc));
            if constexpr (HILO) l += p;
            const _Float16 h = _Float16(p);
            ph[v / 8][v % 8] = h;
            if constexpr (HILO) pl[v / 8][v % 8] = _Float16(p - float(h));
        }
        if constexpr (!HILO) l = add_halves(ph, l);
        if (edge) {  // V outside [lo, hi) may hold anything: 0 * NaN would reach the sums
#pragma unroll
            for (int n = 0; n < NV; ++n) {
#pragma unroll
                for (int d = 0; d < DT; ++d) keep_branch(vf[n][d]);
                u32x4 mask;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t mk = 0;
#pragma unroll
                    for (int e = 0; e < C / 4; ++e) {
                        const uint32_t key = key_of(n * 8 + w * (C / 4) + e);
                        if (key >= t.lo && key < t.hi) mk |= (E4M3 ? 0xffu : 0xffffu) << (e * (E4M3 ? 8 : 16));
                    }
                    mask[w] = mk;
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) vf[n][d] &= mask;
            }
        }
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const half8_t v = chunk_half<E4M3>(vf[n][d], u);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[n * U + u], o[d], 0, 0, 0);
                    if constexpr (HILO) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[n * U + u], o[d], 0, 0, 0);
                }
    }
    l += __shfl_xor(l, 32);
    if (__ballot(bad)) l = __builtin_nanf("");

    const uint32_t pitch = D + 4;
    if (hl == 0) {
        wm[wave][col] = m;
        wl[wave][col] = l;
    }
    if (col < rows) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int b = 0; b < 4; ++b)
                *reinterpret_cast<float4_t *>(&lds[(wave * TM + col) * pitch + d * 32 + 8 * b + 4 * hl]) =
                    float4_t{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
    }
    __syncthreads();
    const bool whole = !PREFIX && n_parts == 1 && a.pre_parts == 0;
    const uint64_t my_row = PREFIX ? a.pre_row + (uint64_t(part) * a.kv.kv_heads + head) * a.pre_rows + t.row0
                                   : (uint64_t(slot) * n_parts * a.kv.kv_heads + head + uint64_t(part) * a.kv.kv_heads) * TM;
    for (uint32_t it = tid; it < rows * (D / 4); it += 256) {
        const uint32_t r = it / (D / 4), d = it % (D / 4) * 4, gr = t.row0 + r;
        const float M = __builtin_fmaxf(__builtin_fmaxf(wm[0][r], wm[1][r]), __builtin_fmaxf(wm[2][r], wm[3][r]));
        float L = 0.f;
        float4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = M == -__builtin_inff() ? 1.f : exp2f_fast(__builtin_fmaf(wm[w][r] - M, a.c1, -kBias<HILO>));
            const float4_t x = *reinterpret_cast<const float4_t *>(&lds[(w * TM + r) * pitch + d]);
            L = __builtin_fmaf(f, wl[w][r], L);
            acc.x = __builtin_fmaf(f, x[0], acc.x);
            acc.y = __builtin_fmaf(f, x[1], acc.y);
            acc.z = __builtin_fmaf(f, x[2], acc.z);
            acc.w = __builtin_fmaf(f, x[3], acc.w);
        }
        if (whole) {
            const float f = a.v_scale / L;
            write_out<D>(a, t.token0 + gr / a.group, head * a.group + gr % a.group, d, float4{acc.x * f, acc.y * f, acc.z * f, acc.w * f});
        } else {
            *reinterpret_cast<float4 *>(a.rows + (my_row + r) * D + d) = acc;
            if (d == 0) *reinterpret_cast<float2 *>(a.stats + 2 * (my_row + r)) = float2{M, L};
        }
    }
}
template <int D, bool E4M3, bool UNI, bool HILO, bool PREFIX>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attn_mid_kernel(AttnArgs a) {
    attn_mid<D, E4M3, UNI, HILO, PREFIX>(a, blockIdx.x, PREFIX ? a.pre_parts : a.parts);
}

// ---- many rows: tiles of 32 rows a wave -----------------------------------------------------------------
//
// v_mfma_f32_32x32x16_f16.  A workgroup's waves take 32 rows each and share the key tiles (32 keys of K and
// V), which stream through two LDS buffers by direct loads; the cache's layout is the fragments'
// order, so every fragment is 512 contiguous bytes of LDS to each half of the wave.  Row m of the K
// operand, m = 8 b + 4 h + r, is key 16 (b / 2) + 8 h + 4 (b % 2) + r (fp16) or 16 h + 4 b + r (e4m3): the
// 16 scores of a lane are then the keys of the V chunks that its half h of the wave reads.
// PREFIX: the rows are those of the whole batch and the keys the shared prefix, which every row sees;
// the results stay parts.  HILO: P as a sum of two fp16, for fp32 outputs.
// Bound by the matrix pipe and what two waves a SIMD hide of the rest: 2,048 tokens at 32,768 keys, 16 heads on 8 of
// 256 dims, 1,010 us with the join's 14 (1,050 TFLOP/s; pipe busy 57%, L2 hits 96%).  With 128 dims e4m3, 12 prompts
// and a window of 1,500, by the vector ALU (10 instructions a matrix one): 205 us, 740 TFLOP/s.
constexpr int kTileWaves = 4, kTileBuffers = 2;
constexpr uint32_t kTileRows = 32 * kTileWaves, kMidRows = 32;

template <int D, bool E4M3, bool HILO, bool PREFIX>
__device__ __forceinline__ void attn_tile(const AttnArgs &a, uint32_t block, uint32_t n_parts) {
    constexpr int C = E4M3 ? 16 : 8, U = C / 8, KT = 32, NW = kTileWaves, NS = kTileBuffers, TM = kTileRows;
    constexpr int KS = D / 16;          // k steps of the first product
    constexpr int DT = D / 32;          // 32-dim tiles of the second
    constexpr int BYTES = KT * D * 16 / C;  // of a K or V tile
    uint8_t(&kt)[NS][BYTES] = *reinterpret_cast<uint8_t(*)[NS][BYTES]>(smem);
    uint8_t(&vt)[NS][BYTES] = *reinterpret_cast<uint8_t(*)[NS][BYTES]>(smem + NS * BYTES);
    const uint32_t kt_at = uint32_t(uintptr_t((__attribute__((address_space(3))) uint8_t *)smem)), vt_at = kt_at + NS * BYTES;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31u, hl = lane >> 5;
    const uint32_t head = block % a.kv.kv_heads, unit = block / a.kv.kv_heads, part = unit % n_parts, slot = unit / n_parts;

    TileSpan t;
    if (!tile_span<D, TM, PREFIX>(a, slot, part, head, t)) return;
    const uint32_t s = t.s, row0 = t.row0, row_end = t.row_end, token0 = t.token0, lo = t.lo, hi = t.hi;
    const uint32_t tile_lo = lo / KT, tile_hi = (hi + KT - 1) / KT, per = (tile_hi - tile_lo + n_parts - 1) / n_parts;
    const uint32_t first = min(tile_lo + part * per, tile_hi), end = min(first + per, tile_hi);

    const uint32_t wrow = row0 + wave * 32;
    const bool active = wrow < row_end;
    const uint32_t row = min(wrow + col, row_end - 1);
    const uint32_t token = token0 + row / a.group, qhead = head * a.group + row % a.group;
    uint32_t limit, least, wmin, wmax;  // the keys that this lane's row sees, and bounds over the wave's rows
    if constexpr (PREFIX) {
        limit = wmin = wmax = hi - 1;
        least = 0;
    } else {
        const uint32_t before = t.before;
        limit = before + row / a.group;
        least = a.window && limit + 1 > a.window ? max(limit + 1 - a.window, a.prefix) : a.prefix;
        wmin = before + min(wrow, row_end - 1) / a.group;
        wmax = before + min(wrow + 31, row_end - 1) / a.group;
    }
    const uint32_t wleast = !PREFIX && a.window && wmin + 1 > a.window ? max(wmin + 1 - a.window, a.prefix) : a.prefix * (PREFIX ? 0 : 1);
    const uint32_t wmost = !PREFIX && a.window && wmax + 1 > a.window ? max(wmax + 1 - a.window, a.prefix) : a.prefix * (PREFIX ? 0 : 1);

    half8_t qf[KS];
    {
        const uint16_t *src = a.q + (uint64_t(token) * a.q_heads + qhead) * D;
#pragma unroll
        for (int j = 0; j < KS / U; ++j)
#pragma unroll
            for (int u = 0; u < U; ++u)
                qf[j * U + u] = __builtin_bit_cast(half8_t, *reinterpret_cast<const u32x4 *>(src + (2 * j + hl) * C + 8 * u));
    }
    float16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = float16_t{};
    const float far_m = far_max(a.c1);
    float m = -__builtin_inff(), l = 0.f;
    bool bad = false;

    const int32_t *table = a.kv.table + uint64_t(s) * a.kv.stride;
    const uint32_t smask = (1u << a.kv.page_shift) - 1;
    // A tile's two halves of 16 keys lie in one page each (pages hold 16 tokens or more).  Halves outside
    // [lo, hi) take the nearest page that is inside: their keys are masked.
    auto page_of = [&](uint32_t key) {
        const uint32_t e = min(max(key, lo), hi - 1) >> a.kv.page_shift;
        return uint32_t(((const __attribute__((address_space(4))) int32_t *)table)[__builtin_amdgcn_readfirstlane(e)]);
    };
    // Pages of whole tiles: a wave takes NB consecutive KiB of each of K and V, at fixed offsets from the tile's scalar
    // addresses.  K's rows of 32 tokens lie a page's row apart, 1 KiB or more, so the offsets less 1024 i stay positive.
    constexpr uint32_t NB = BYTES / 1024 >= NW ? BYTES / 1024 / NW : 1;
    const bool whole_tiles = a.kv.page_shift >= 5, loads = BYTES / 1024 >= NW || wave < BYTES / 1024;
    uint32_t koff0 = (((2 * wave * NB + hl) << a.kv.page_shift) + (lane & 31u)) * 16;
    const uint32_t voff0 = (wave * NB * 64 + lane) * 16, kstep = (32u << a.kv.page_shift) - 1024;
    auto fetch = [&](uint32_t tile, uint32_t pa, uint32_t pb, uint32_t buf) {
        if (whole_tiles) {
            bad |= pa >= a.kv.pages;
            const uint64_t at = kv_offset<D, E4M3>(a.kv, pa < a.kv.pages ? pa : 0u, head);
            const uint32_t slot0 = (tile * KT) & smask;
            if (loads) {
                asm volatile("" : "+v"(koff0));  // formed again for every tile, not kept
                uint32_t koff[NB], voff[NB];
#pragma unroll
                for (uint32_t i = 0; i < NB; ++i) {
                    koff[i] = koff0 + i * kstep;
                    voff[i] = voff0;
                }
                dma16_run<NB>(a.kv.k + at + slot0 * 16, koff, kt_at + buf * BYTES + wave * NB * 1024);
                dma16_run<NB>(a.kv.v + at + uint64_t(slot0 / C) * (D * 16), voff, vt_at + buf * BYTES + wave * NB * 1024);
            }
            return;
        }
        bad |= pa >= a.kv.pages || pb >= a.kv.pages;
        const uint64_t oa = kv_offset<D, E4M3>(a.kv, pa < a.kv.pages ? pa : 0u, head), ob = kv_offset<D, E4M3>(a.kv, pb < a.kv.pages ? pb : 0u, head);
        const uint32_t sa = (tile * KT) & smask, sb = (tile * KT + 16) & smask;
        const bool second = (lane & 31u) >= 16;
        const uint8_t *ks = a.kv.k + (second ? ob : oa) + ((second ? sb : sa) + (lane & 15u)) * 16;
#pragma unroll
        for (int i = 0; i < BYTES / 1024; i += NW) {
            const uint32_t w = i + wave;  // 1 KiB: chunks 2 w and 2 w + 1 of 32 tokens
            if (BYTES / 1024 % NW == 0 || w < BYTES / 1024)
                dma16(ks + (uint64_t(2 * w + hl) << a.kv.page_shift) * 16, kt_at + buf * BYTES + w * 1024);
        }
#pragma unroll
        for (int i = 0; i < BYTES / 1024; i += NW) {
            const uint32_t w = i + wave, idx = w * 64, grp = idx / D;  // 64 dims of one token chunk
            const bool b2 = grp * C >= 16;
            const uint32_t sl = b2 ? sb + grp * C - 16 : sa + grp * C;
            if (BYTES / 1024 % NW == 0 || w < BYTES / 1024)
                dma16(a.kv.v + (b2 ? ob : oa) + (uint64_t(sl / C) * D + idx % D + lane) * 16, vt_at + buf * BYTES + w * 1024);
        }
    };

    // The first tile is on its way before the loop; each step asks for the next one.  (A loop of one round: without it
    // the 256-dim e4m3 instance spills, 238 -> 265 us for 3 x 1,024 tokens of 9,000 keys on pages of 16.)
    auto fetch_tile = [&](uint32_t tile, uint32_t buf) { fetch(tile, page_of(tile * KT), page_of(tile * KT + 16), buf); };
#pragma unroll
    for (uint32_t i = 0; i < NS - 1; ++i)
        if (first + i < end) fetch_tile(first + i, i);
    uint32_t pa = page_of((first + 1) * KT), pb = page_of((first + 1) * KT + 16);
    const uint32_t krow = E4M3 ? 16 * ((col / 4) % 2) + 4 * (col / 8) + col % 4 : 16 * (col / 16) + 8 * ((col / 4) % 2) + 4 * ((col / 8) % 2) + col % 4;
    uint32_t buf = 0;
    for (uint32_t tile = first; tile < end; ++tile, buf ^= 1) {
        // This tile has landed for every wave, and every wave is done with the buffer that the next loads go to (its
        // reads of it have returned).
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0);
        __builtin_amdgcn_s_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        if (tile + 1 < end) {
            fetch(tile + 1, pa, pb, buf ^ 1);
            pa = page_of((tile + 2) * KT);
            pb = page_of((tile + 2) * KT + 16);
        }
        const uint32_t t0 = tile * KT;
        if (t0 < lo || t0 + KT > hi) {  // V outside [lo, hi) may hold anything, and 0 * NaN would reach the sums
#pragma unroll
            for (uint32_t i = tid; i < BYTES / 16; i += 64 * NW) {
                u32x4 *c = reinterpret_cast<u32x4 *>(&vt[buf][i * 16]);
                const uint32_t k0 = t0 + i / D * C;
                u32x4 x = *c;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t mk = 0;
#pragma unroll
                    for (int e = 0; e < C / 4; ++e) {
                        const uint32_t key = k0 + w * (C / 4) + e;
                        if (key >= lo && key < hi) mk |= (E4M3 ? 0xffu : 0xffffu) << (e * (E4M3 ? 8 : 16));
                    }
                    x[w] &= mk;
                }
                *c = x;
            }
            __syncthreads();
        }
        if (!active || t0 > wmax || t0 + KT <= wleast) continue;
        const uint8_t *kp = &kt[buf][(hl * KT + krow) * 16], *vp = &vt[buf][(hl * D + col) * 16];
        float16_t sc = float16_t{};
#pragma unroll
        for (int j = 0; j < KS / U; ++j) {
            const u32x4 c = *reinterpret_cast<const u32x4 *>(kp + j * (2 * KT * 16));
#pragma unroll
            for (int u = 0; u < U; ++u) sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(chunk_half<E4M3>(c, u), qf[j * U + u], sc, 0, 0, 0);
        }
        const bool edge = t0 < wmost || t0 + KT > wmin + 1;
        // scores v = 8 n + e of this lane: key t0 + 16 n + 8 hl + e (fp16), t0 + 16 hl + v (e4m3)
        auto key_of = [&](int v) { return E4M3 ? t0 + 16 * hl + uint32_t(v) : t0 + 16 * uint32_t(v / 8) + 8 * hl + uint32_t(v % 8); };
        if (edge) {
            keep_branch(sc);
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const uint32_t key = key_of(v);
                if (key > limit || key < least) sc[v] = -__builtin_inff();
            }
        }
        float top = sc[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) top = __builtin_fmaxf(top, sc[v]);
        top = max_halves(top);
        const float mn = __builtin_fmaxf(m, top);
        bool far = false;
        if (__ballot((mn - m) * a.c1 > kLag<HILO> || __builtin_fabsf(m) > far_m)) {
            const float f = mn == m ? 1.f : exp2f_fast((m - mn) * a.c1);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
            m = mn;
            if (__ballot(__builtin_fabsf(m) > far_m)) {
                const float zero = m == -__builtin_inff() ? 0.f : m;
                keep_branch(sc);
                sc -= zero;
                far = true;
            }
        }
        const float mc = far ? -kBias<HILO> : __builtin_fmaf(m, a.c1, -kBias<HILO>);
        half8_t ph[2], pl[2];
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const float p = exp2f_fast(__builtin_fmaf(sc[v], a.c1, -mc));
            if constexpr (HILO) l += p;
            const _Float16 h = _Float16(p);
            ph[v / 8][v % 8] = h;
            if constexpr (HILO) pl[v / 8][v % 8] = _Float16(p - float(h));
        }
        if constexpr (!HILO) l = add_halves(ph, l);
#pragma unroll
        for (int n = 0; n < 2 / U; ++n)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const u32x4 c = *reinterpret_cast<const u32x4 *>(vp + ((E4M3 ? 0 : 2 * n) * D + d * 32) * 16);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const half8_t v = chunk_half<E4M3>(c, u);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[n * U + u], o[d], 0, 0, 0);
                    if constexpr (HILO) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[n * U + u], o[d], 0, 0, 0);
                }
            }
    }
    l += __shfl_xor(l, 32);
    if (__ballot(bad)) l = __builtin_nanf("");
    const bool whole = !PREFIX && n_parts == 1 && a.pre_parts == 0;
    const bool mine = wrow + col < row_end;
    const uint64_t own_step = uint64_t(a.kv.kv_heads) * (PREFIX ? a.pre_rows : TM);
    const uint64_t own_row = PREFIX ? a.pre_row + uint64_t(head) * a.pre_rows + row0 : (uint64_t(slot) * n_parts * a.kv.kv_heads + head) * TM;
    if (!mine) return;
    const float f = whole ? a.v_scale / l : kUnbias<HILO>;
    const uint64_t at = own_row + part * own_step + (wrow - row0) + col;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const uint32_t dim = d * 32 + 8 * b + 4 * hl;
            const float4 v{o[d][4 * b] * f, o[d][4 * b + 1] * f, o[d][4 * b + 2] * f, o[d][4 * b + 3] * f};
            if (whole) write_out<D>(a, token, qhead, dim, v);
            else *reinterpret_cast<float4 *>(a.rows + at * D + dim) = v;
        }
    if (!whole && hl == 0) *reinterpret_cast<float2 *>(a.stats + 2 * at) = float2{m, l * kUnbias<HILO>};
}
template <int D, bool E4M3>
struct TileLds {
    static constexpr uint32_t kBytes = 2 * kTileBuffers * 32 * D * (E4M3 ? 1 : 2);
};
template <int D, bool E4M3, bool HILO, bool PREFIX>
__global__ __launch_bounds__(64 * kTileWaves, 2) void attn_tile_kernel(AttnArgs a) {
    attn_tile<D, E4M3, HILO, PREFIX>(a, blockIdx.x, PREFIX ? a.pre_parts : a.parts);
}

// ---- a shared prefix and few rows of each sequence: both kinds of work in one launch --------------------------
//
// The prefix's row tiles (all sequences' rows, MID: 32 of them a tile, otherwise 128) and the sequences' own keys read different
// memory and do not depend on each other: side by side they keep the memory busy through each other's starts
// and ends (64 sequences of up to 500 keys of their own on 32,768 tokens, 256 dims, 8 key heads: 70 and 46 us one after
// the other, 92 side by side: 4.6 TB/s).  Bound by the bytes of the prefix, read once.
template <int D, bool E4M3, bool UNI, bool HILO, bool MID>
__global__ __launch_bounds__(256, D == 256 && MID ? 1 : 2) void attn_shared_kernel(AttnArgs a, uint32_t pre_blocks) {
    if (blockIdx.x < pre_blocks) {
        if constexpr (MID) attn_mid<D, E4M3, UNI, HILO, true>(a, blockIdx.x, a.pre_parts);
        else attn_tile<D, E4M3, HILO, true>(a, blockIdx.x, a.pre_parts);
    } else {
        attn_rows<D, E4M3, UNI, false, false>(a, blockIdx.x - pre_blocks);
    }
}

// Joins that launch's parts (64 sequences of 16 heads, some 33 parts a row: 8.6 us): D / 4 threads a
// row, which the few-row workgroups' notes for its token lead to its parts.
template <int D>
__global__ __launch_bounds__(256) void attn_shared_join_kernel(AttnArgs a) {
    constexpr uint32_t PER = 256 / (D / 4);
    const uint32_t head = blockIdx.x % a.kv.kv_heads, row = blockIdx.x / a.kv.kv_heads * PER + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    const int32_t token = int32_t(row / a.group);
    if (token >= int32_t(a.kv.tokens) || token < a.kv.q_start[0] || token >= a.kv.q_start[a.kv.seqs]) return;
    const uint4 note = a.tokens[token];  // first part, parts, first row of the sequence
    const uint32_t r = row - note.z;
    // (the bounds hold for every sequence of the batch; rows between sequences, of a contradicting q_start, have no note)
    if (note.y == 0 || note.y > a.row_slots || note.x > a.row_slots - note.y || r >= a.row_cap) return;
    const uint64_t own_row = (uint64_t(note.x) * a.kv.kv_heads + head) * a.row_cap;
    const Parts ps{note.y, note.y + a.pre_parts, own_row, uint64_t(a.kv.kv_heads) * a.row_cap, a.pre_row + uint64_t(head) * a.pre_rows + note.z,
                   uint64_t(a.kv.kv_heads) * a.pre_rows};
    join_row<D>(a, ps, r, d, uint32_t(token), head * a.group + row % a.group);
}

// Joins the tile kernel's parts: a workgroup takes kJoinRows rows of a row tile, a thread four dims of a row at a
// time, in part order.  A launch of its own, so that all of the chip reads the parts (128 rows of 256
// dims are 128 KiB a part; 2,048 tokens of 16 heads of 256 dims in two parts: 14 us, 4.8 TB/s).
constexpr uint32_t kJoinRows = 16;
template <int D, int TM>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    const uint32_t head = blockIdx.x % a.kv.kv_heads, unit = blockIdx.x / a.kv.kv_heads, slot = unit / (TM / kJoinRows);
    auto first_tile = [&](uint32_t i) {
        return uint32_t(uint64_t(min(uint32_t(max(a.kv.q_start[i], 0)), a.kv.tokens)) * a.group / TM) + i;
    };
    const uint32_t s = find_seq(a.kv.seqs, slot, first_tile);
    const KvSeq q = kv_seq(a.kv, s, a.prefix);
    const uint32_t row_end = q.n * a.group, at = slot - first_tile(s), tiles = (row_end + TM - 1) / TM;
    if (at >= tiles || !q.ok || (a.skip_small && row_end <= kRowsMax)) return;
    const uint32_t row0 = (tiles - 1 - at) * TM, r0 = unit % (TM / kJoinRows) * kJoinRows;
    const Parts ps{a.parts, a.parts + a.pre_parts, (uint64_t(slot) * a.parts * a.kv.kv_heads + head) * TM, uint64_t(a.kv.kv_heads) * TM,
                   a.pre_row + uint64_t(head) * a.pre_rows + uint64_t(q.q0) * a.group + row0, uint64_t(a.kv.kv_heads) * a.pre_rows};
    for (uint32_t it = threadIdx.x; it < kJoinRows * (D / 4); it += 256) {
        const uint32_t r = r0 + it / (D / 4), d = it % (D / 4) * 4, row = row0 + r;
        if (row >= row_end) return;
        join_row<D>(a, ps, r, d, q.q0 + row / a.group, head * a.group + row % a.group);
    }
}

// Estimated time (us) of row tiles of `rows` rows: `busy` of them (key heads counted), with `tiles` key tiles at most
// and `mean` on the average, in p key parts.  kTile and kMid: a key tile's time with 1, 2, ... workgroups on each CU, up
// to as many as fit (one sequence of 8 key heads, 2,048 and 8,192 keys before 1,024 to 16,384 rows; fp16 outputs of
// an fp16 cache: e4m3 caches and fp32 outputs go by the same figures, though the 128-dim instances of fp32 outputs
// have registers for two workgroups a CU, not three).  The longest start first, so the time is the longest workgroup's,
// or all of them through the slots of the chip with half of one at the end.  The other constants are fitted to 450
// calls of 17 to 5,800 tokens a sequence and up to 40,000 keys; on 300 others, of all types and outputs, the choice took
// 1.03 times the fastest of all choices on the average, at most 1.09 times in nine of ten and 1.17 in 97 of 100 (most of
// the others: batches far shorter than their bounds say).
struct TileWork {
    uint32_t head_dim, busy, tiles;
    double mean;
    double kv_bytes;  // keys and values that the row tiles read together
};
double tile_time(uint32_t rows, const TileWork &w, uint32_t p, bool join, uint32_t n_cus) {
    static const double kTile[3][4] = {{0.60, 0.67, 0.95, 1.28}, {0.75, 1.02, 1.55, 0}, {1.40, 1.96, 0, 0}};
    static const double kMid[3][4] = {{0.148, 0.203, 0, 0}, {0.21, 0.33, 0, 0}, {0.35, 0, 0, 0}};
    const int d = w.head_dim == 64 ? 0 : w.head_dim == 128 ? 1 : 2;
    const bool mid = rows == kMidRows;
    const double *step = mid ? kMid[d] : kTile[d];
    const uint64_t cus = n_cus, most = mid ? (d == 2 ? 1 : 2) : 4 - d, wgs = uint64_t(w.busy) * p;
    const uint64_t each = std::min(most, (wgs + cus - 1) / cus);
    const double start = mid ? 8.0 : 5.0, mean = w.mean / p;
    double t = step[each - 1] * double((w.tiles + p - 1) / p) + start;
    if (wgs > cus * most) t = std::max(t, (step[most - 1] * (mean + 0.5) + start) * double(wgs) / double(cus * most) + 0.5 * step[0] * mean);
    // every row tile reads all its keys, from L2 or beyond it: 14.5 TB/s together
    t = std::max(t, w.kv_bytes / 14.5e6);
    return t + (mid ? 1.0 : 11.0) + (join ? 4.0 + 0.14 * p + double(wgs) * rows * w.head_dim * 8.0 / 5.4e6 : 0.0);
}
// The estimated fastest number of key parts up to `most`, of some that grow by a third and those that just fill the
// chip one to four times (trying all took 70 us of host time at 256 of them).
double tile_parts(uint32_t rows, const TileWork &w, uint32_t most, bool prefix, uint32_t cus, uint32_t *parts) {
    static const uint32_t kSome[] = {1, 2, 3, 4, 6, 8, 11, 16, 22, 32, 44, 64, 88, 128, 176, 256};
    most = std::min(most, std::max(1u, w.tiles / 2));
    double least = 1e30;
    auto attempt = [&](uint32_t p) {
        if (p < 1 || p > most) return;
        const double t = tile_time(rows, w, p, prefix || p > 1, cus);
        if (t < least) {
            least = t;
            *parts = p;
        }
    };
    for (uint32_t p : kSome) attempt(p);
    for (uint32_t k = 1; k <= 4; ++k) attempt(k * cus / w.busy);
    return least;
}

AttnPlan plan_attn(const AttnShape &s, const Tuning &tune) {
    AttnPlan p;
    const uint32_t cus = uint32_t(device_cus()), group = s.q_heads / s.kv_heads, kt = s.type == KV_E4M3 ? 64 : 32;
    const bool small = s.max_q * group <= kRowsMax;
    const uint32_t keys = s.window ? std::min(s.max_kv, s.window + s.max_q) : s.max_kv - s.prefix;
    const uint64_t rows = uint64_t(s.tokens) * group;
    if (small || s.seqs > 1) {
        p.row_cap = std::min(kRowsMax, std::min(s.max_q, kRowsMax) * group);
        // Two workgroups a CU, all parts in as few rounds as the sequences allow: each sequence's last part is half
        // full on the average, so parts of total / target tiles are target + seqs / 2 in number.
        const uint32_t round = std::max(1u, 2 * cus / s.kv_heads), rounds = (s.seqs + round - 1) / round;
        p.target = std::min(kPartsMax / 2, std::max(1u, rounds * round - s.seqs / 2));
        // A part is four tiles or more, one for each wave.  Calls in us with 1 / 2 / 4 / 8 / 32: one token at 2,206 keys 13.4 /
        // 13.5 / 11.3 / 12.6 / 26, at 700 keys 10.4 / 9.4 / 10.2 / 12.8 / 19, three in a window of 1,024 (e4m3) 14.7 / 11.6 / 11.6 /
        // 13.6 / 16.5, 8 sequences up to 1,500 keys (e4m3) 10.8 / 10.9 / 10.6 / 11.0 / 12.7.  (32: the short ones without a join.)
        p.min_tiles = 4;
        const uint64_t most = uint64_t(s.seqs) * ((keys / kt + 2 + p.min_tiles - 1) / p.min_tiles);
        p.row_slots = uint32_t(std::min<uint64_t>(most, uint64_t(p.target) + s.seqs));
        p.own_rows = uint64_t(p.row_slots) * s.kv_heads * p.row_cap;
        p.counters = uint64_t(s.seqs) * s.kv_heads;
    }
    const double token_bytes = 2.0 * s.kv_heads * s.head_dim * (s.type == KV_E4M3 ? 1 : 2);
    if (!small) {
        // Row tiles that hold rows: the full ones, or one for each sequence that is not the few-row kernel's
        auto work = [&](uint32_t tm) {
            const uint64_t full = (rows + tm - 1) / tm, seqs = std::min<uint64_t>(s.seqs, rows / (kRowsMax + 1));
            const uint32_t per_head = uint32_t(std::max<uint64_t>(std::max(full, seqs), 1));
            const uint32_t seen = s.window ? std::min(s.max_kv, s.window + (tm + group - 1) / group) : s.max_kv - s.prefix;
            const double mean = std::max(1.0, s.window ? double(seen) : double(seen) - 0.5 * s.max_q);  // causal
            return TileWork{s.head_dim, per_head * s.kv_heads, (seen + 31) / 32, mean / 32, token_bytes * mean * per_head};
        };
        uint32_t pt = 1, pm = 1;
        const double tt = tile_parts(kTileRows, work(kTileRows), 32, s.prefix != 0, cus, &pt);
        const double tm = tile_parts(kMidRows, work(kMidRows), 32, s.prefix != 0, cus, &pm);
        const bool mid = tune.attn_mid < 0 ? tm < tt : tune.attn_mid != 0;
        p.tile_rows = mid ? kMidRows : kTileRows;
        p.parts = tune.attn_parts > 0 ? uint32_t(tune.attn_parts) : mid ? pm : pt;
        p.tile_slots = uint32_t(rows / p.tile_rows) + s.seqs;
        p.parts = std::max(1u, std::min(p.parts, (1u << 23) / (p.tile_slots * s.kv_heads)));  // a launch's workgroups, however tuned
        if (p.parts > 1 || s.prefix) p.own_rows = std::max(p.own_rows, uint64_t(p.tile_slots) * p.parts * s.kv_heads * p.tile_rows);
    }
    p.all_rows = p.own_rows;
    if (s.prefix) {
        auto work = [&](uint32_t tm) {
            const uint32_t per_head = uint32_t((rows + tm - 1) / tm);
            return TileWork{s.head_dim, per_head * s.kv_heads, (s.prefix + 31) / 32, s.prefix / 32.0, token_bytes * s.prefix * per_head};
        };
        uint32_t pt = 1, pm = 1;
        const double tt = tile_parts(kTileRows, work(kTileRows), kPartsMax / 2, true, cus, &pt);
        const double tm = tile_parts(kMidRows, work(kMidRows), kPartsMax / 2, true, cus, &pm);
        const bool mid = tune.attn_mid < 0 ? tm < tt : tune.attn_mid != 0;
        p.pre_tile_rows = mid ? kMidRows : kTileRows;
        p.pre_parts = tune.attn_parts > 0 ? std::min(uint32_t(tune.attn_parts), kPartsMax / 2) : mid ? pm : pt;
        p.pre_tiles = uint32_t((rows + p.pre_tile_rows - 1) / p.pre_tile_rows);
        p.pre_parts = std::max(1u, std::min(p.pre_parts, (1u << 23) / (p.pre_tiles * s.kv_heads)));
        p.pre_rows = p.pre_tiles * p.pre_tile_rows;
        p.all_rows += uint64_t(p.pre_parts) * s.kv_heads * p.pre_rows;
    }
    return p;
}

// The row tiles of `rows` rows: 128 with the keys shared in LDS, or 32.
template <int D, bool E4M3, bool PREFIX>
hipError_t launch_tiles(uint32_t rows, uint32_t wgs, const AttnArgs &a, hipStream_t stream) {
    const dim3 g(wgs), b(256);
    const bool uni = a.kv.page_shift >= 5;
    if (rows == kTileRows) {
        constexpr uint32_t lds = TileLds<D, E4M3>::kBytes;
        if (a.half_out) attn_tile_kernel<D, E4M3, false, PREFIX><<<g, b, lds, stream>>>(a);
        else attn_tile_kernel<D, E4M3, true, PREFIX><<<g, b, lds, stream>>>(a);
    } else {
        constexpr uint32_t lds = MidLds<D>::kBytes;
        if (uni && a.half_out) attn_mid_kernel<D, E4M3, true, false, PREFIX><<<g, b, lds, stream>>>(a);
        else if (uni) attn_mid_kernel<D, E4M3, true, true, PREFIX><<<g, b, lds, stream>>>(a);
        else if (a.half_out) attn_mid_kernel<D, E4M3, false, false, PREFIX><<<g, b, lds, stream>>>(a);
        else attn_mid_kernel<D, E4M3, false, true, PREFIX><<<g, b, lds, stream>>>(a);
    }
    return hipGetLastError();
}

// The prefix and few rows of each sequence in one launch.  UNI by the larger key tile (64 e4m3 keys of the few-row part).
template <int D, bool E4M3, bool UNI, bool HILO>
hipError_t launch_shared(const AttnPlan &p, const AttnArgs &a, hipStream_t stream) {
    const uint32_t pre = p.pre_tiles * p.pre_parts * a.kv.kv_heads, rows = RowsLds<D>::bytes(p.row_cap);
    const dim3 g(pre + p.row_slots * a.kv.kv_heads), b(256);
    if (p.pre_tile_rows == kTileRows)
        attn_shared_kernel<D, E4M3, UNI, HILO, false><<<g, b, std::max(rows, TileLds<D, E4M3>::kBytes), stream>>>(a, pre);
    else
        attn_shared_kernel<D, E4M3, UNI, HILO, true><<<g, b, std::max(rows, MidLds<D>::kBytes), stream>>>(a, pre);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    const uint32_t per = 256 / (D / 4);
    attn_shared_join_kernel<D><<<dim3((a.kv.tokens * a.group + per - 1) / per * a.kv.kv_heads), b, 0, stream>>>(a);
    return hipGetLastError();
}

template <int D, bool E4M3>
hipError_t launch(const AttnPlan &p, const AttnArgs &a, hipStream_t stream) {
    const bool uni = (1u << a.kv.page_shift) >= (E4M3 ? 64u : 32u);
    if (p.pre_parts && !p.tile_slots) {
        if (uni && a.half_out) return launch_shared<D, E4M3, true, false>(p, a, stream);
        if (uni) return launch_shared<D, E4M3, true, true>(p, a, stream);
        return a.half_out ? launch_shared<D, E4M3, false, false>(p, a, stream) : launch_shared<D, E4M3, false, true>(p, a, stream);
    }
    if (p.pre_parts)
        if (const hipError_t e = launch_tiles<D, E4M3, true>(p.pre_tile_rows, p.pre_tiles * p.pre_parts * a.kv.kv_heads, a, stream); e != hipSuccess) return e;
    if (p.row_slots) {
        const dim3 g(p.row_slots * a.kv.kv_heads);
        const uint32_t lds = RowsLds<D>::bytes(p.row_cap);
        if (uni && a.kv.seqs == 1) attn_rows_kernel<D, E4M3, true, true><<<g, dim3(256), lds, stream>>>(a);
        else if (uni) attn_rows_kernel<D, E4M3, true, false><<<g, dim3(256), lds, stream>>>(a);
        else attn_rows_kernel<D, E4M3, false, false><<<g, dim3(256), lds, stream>>>(a);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    if (p.tile_slots) {
        if (const hipError_t e = launch_tiles<D, E4M3, false>(p.tile_rows, p.tile_slots * p.parts * a.kv.kv_heads, a, stream); e != hipSuccess) return e;
        if (p.parts > 1 || p.pre_parts) {
            const dim3 g(p.tile_slots * (p.tile_rows / kJoinRows) * a.kv.kv_heads);
            if (p.tile_rows == kTileRows) attn_join_kernel<D, kTileRows><<<g, dim3(256), 0, stream>>>(a);
            else attn_join_kernel<D, kMidRows><<<g, dim3(256), 0, stream>>>(a);
            return hipGetLastError();
        }
    }
    return hipSuccess;
}

}  // namespace

AttnPlan plan_attention(const AttnShape &s, const Tuning &t) {
    AttnPlan p = plan_attn(s, t);
    // the rows, their statistics, and 16 bytes a token of notes for the separate join
    p.partial_floats = size_t(p.all_rows) * (s.head_dim + 2) + (s.prefix ? 4 * size_t(s.tokens) + 4 : 0);
    return p;
}

hipError_t launch_attention(const AttnShape &s, const AttnPlan &p, const KvArgs &kv, const uint16_t *q, float scale, float k_scale, float v_scale,
                            void *out, bool half_out, const Workspace &ws, hipStream_t stream) {
    AttnArgs a{};
    a.kv = kv;
    a.q = q;
    a.out = out;
    a.rows = ws.partial;
    a.stats = ws.partial + size_t(p.all_rows) * s.head_dim;
    a.counters = ws.counters;
    a.tokens = reinterpret_cast<uint4 *>(ws.partial + (size_t(p.all_rows) * (s.head_dim + 2) + 3) / 4 * 4);
    a.row_slots = p.row_slots;
    a.q_heads = s.q_heads;
    a.group = s.q_heads / s.kv_heads;
    a.window = s.window;
    a.prefix = s.prefix;
    a.c1 = scale * k_scale * kLog2e;
    a.v_scale = v_scale;
    a.half_out = half_out ? 1 : 0;
    a.target = p.target;
    a.min_tiles = p.min_tiles;
    a.row_cap = p.row_cap;
    a.parts = p.parts;
    a.skip_small = p.row_slots ? 1 : 0;
    a.pre_row = p.own_rows;
    a.pre_parts = p.pre_parts;
    a.pre_rows = p.pre_rows;
    const bool e = s.type == KV_E4M3;
    switch (s.head_dim) {
        case 64: return e ? launch<64, true>(p, a, stream) : launch<64, false>(p, a, stream);
        case 128: return e ? launch<128, true>(p, a, stream) : launch<128, false>(p, a, stream);
        case 256: return e ? launch<256, true>(p, a, stream) : launch<256, false>(p, a, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace ns
