// Attention over packed sequences of different lengths, causal or not, with grouped heads, for gfx950.
//
// Sequence s holds the query rows [cu_q[s], cu_q[s + 1]) of q and the key rows [cu_k[s], cu_k[s + 1]) of k and v, or the
// first k_lens[s] of these; query head h reads key head h / (heads / kv_heads). Query i of lq sees the keys j < lk and,
// causal, j <= i + lk - lq:
//   o_i = sum_j 2^(u_ij - m_i) v_j / sum_j 2^(u_ij - m_i),  u_ij = scale log2(e) q_i . k_j,
// for any m_i near the row's largest u; 0 where no key is left. The offsets are read on the device only (a captured graph
// may be replayed with others) and clamped to the buffers' rows, so no offset reaches outside them; nothing on the host
// depends on a length, the bounds max_q and max_k only choose among ways that are all correct.
//
// Rows: a key head's queries are taken as lq x group rows (row r = query r / group, head r % group of the group), so that
// K and V are read once for the whole group and a few queries with many heads still fill a tile.
//
// attn_packed_tile (prompts): a workgroup of 4 waves owns 128 rows, a wave 32; tiles of 64 keys go straight from memory
// into LDS (two buffers, 16-byte chunks permuted by row against bank conflicts), one barrier a tile. Scores are taken
// transposed, S^T = K Q^T on the 32x32x16 matrix instructions, so a lane holds 32 scores of one row; the probabilities
// become the B operand of O^T = V^T P^T from the registers they are in, and V^T is read out of the row-major V tile by
// the transposing LDS reads in the key order that the scores have. m goes by the first tile's maximum and is raised only for
// a tile with far larger scores. Tiles past a wave's last visible key are skipped, only tiles that some row sees in part are
// masked. Bound by MFMAs and the softmax's vector work, of which little overlaps: one bf16 prompt of 16384,
// 32 heads on 8 of 128, 1.9 ms (1.1 PFLOP/s, matrix units busy 60% of the cycles), 8 fp16 prompts of up to 4096, 24 heads of
// 64, 193 us (0.7; half the products for each exponential). Waves that take the next tile's scores among this tile's
// exponentials were slower at both (2.1 ms, 221 us).
//
// attn_packed_few (serving: sequences of up to kFewRows rows): bound by reading K and V once. A workgroup takes one chunk
// of a sequence's keys for all its rows; each of its waves walks its own 32-key tiles in LDS of its own, no barrier between
// them, and the waves' (m, l, O) are merged through LDS. The chunks of all sequences are one list: chunk c of a sequence that
// starts at key row b is entry b / chunk + s + c, so long and short sequences spread evenly; or, where that gives fewer
// entries (lengths alike; caches mostly empty: 4 sequences of up to 4000 keys in 65536 rows each 21 us, with the list
// 45), s per + c with per chunks for the longest. Parts of a sequence cut into several chunks go to the workspace in fp32 and
// attn_packed_combine merges them in order.
//
// Probabilities are rounded to the inputs' type for the matrix product, and the sum l adds the rounded values, so the
// weights still sum to 1. Each is off by up to u = 2^-9 (bf16) or 2^-12 (fp16) of itself, so an output by u (A + |o|) at most,
// A = sum p_j |v_j|; over values of mean zero that is about what the output's own rounding is (48 sequences in bf16: 2.3e-3
// of the result in all, 1.7e-3 with fp32 weights). Two bf16 parts a weight would take half as many matrix products again.
// bf16: m lies 2^24 above the row's maximum, so that sums of values near the type's largest stay finite. fp16: 2^8 below it,
// as small weights would vanish otherwise (a key 17.5 above 4096 others: a third of their weight).
#include "q8_dma.h"

#include <algorithm>
#include <type_traits>

namespace idolq {
namespace {

constexpr int kTileRows = 128;  // rows of an attn_packed_tile workgroup
constexpr int kTileKeys = 64;
constexpr int kShortKeys = 1024;  // key ranges up to here are not cut by attn_packed_few
constexpr int kTilePart = 256;  // least keys of a part
constexpr int kFewRows = 64;    // sequences of up to so many rows go to attn_packed_few where both kernels run
constexpr int kFewKeys = 32;    // keys of a wave's tile there
constexpr int kFewWaves = 4;
constexpr int64_t kListBytes = (int64_t)64 << 20;

struct PackedParams {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    const int32_t* cu_q;
    const int32_t* cu_k;
    const int32_t* k_lens;  // null: all of a sequence's key rows
    int64_t ldq, ldk, ldv, ldo;
    int total_q, total_k, seqs, heads, kv_heads, group;  // group: query heads per key head
    int causal;
    float scale_log2;  // scale * log2(e)
    int slots;         // attn_packed_tile: row tiles over all sequences, at most
    int ordered;       // they are taken in ordered_tile's order
    int few_rows;      // sequences of more rows are attn_packed_tile's, the others attn_packed_few's
    int chunk;         // attn_packed_few: keys of a chunk
    int per;           // and entries of a sequence (its last chunk takes the rest); 0: as many as its rows' chunks
    int part_rows;     // rows a sequence may have to be cut into parts
    int sparse;        // the parts' entries go by their keys, not by the list (see first_part)
    float* parts;      // O [entry][HD] of the parts' rows, then (m, l) [entry]
    int64_t part_count;
    int tile_chunk, tile_parts;  // attn_packed_tile: keys of a part, at most so many parts (1: none is cut)
    int64_t tile_entry;          // its first entry
};

// The rows [first, first + count) of sequence s, inside [0, total) whatever the offsets hold.
struct Rows {
    int first, count;
};
__device__ __forceinline__ int clamped(const int32_t* cu, int s, int total) { return min(max(cu[s], 0), total); }
__device__ __forceinline__ Rows rows_of(const int32_t* cu, int s, int total) {
    const int first = clamped(cu, s, total);
    return {first, max(clamped(cu, s + 1, total) - first, 0)};
}

// The keys of sequence s.
__device__ __forceinline__ Rows keys_of(const PackedParams& p, int s) {
    Rows r = rows_of(p.cu_k, s, p.total_k);
    if (p.k_lens) r.count = min(r.count, max(p.k_lens[s], 0));
    return r;
}

// Pieces of `size` in n (none in less than 1).
__device__ __forceinline__ int pieces(int n, int size) { return n > 0 ? (n - 1) / size + 1 : 0; }

// Entry `slot` of the list in which sequence s has the entries from first(s) on (first does not decrease): the last
// sequence with first(s) <= slot (0 if there is none), looked for by the whole wave, 64 sequences a step.
template <typename F>
__device__ __forceinline__ int find_sequence(int seqs, int64_t slot, F&& first) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = seqs;
    while (n > 1) {
        const int stride = pieces(n, 64);
        const bool before = (int64_t)lane * stride < n && first(lo + min(lane * stride, n - 1)) <= slot;
        const int found = (int)__popcll(__builtin_amdgcn_ballot_w64(before));  // none: the slot is before sequence 0's first
        const int at = max(found - 1, 0) * stride;
        lo += at, n = min(stride, n - at);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p);
}
// offset: a constant, which goes into the instruction
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at, int offset = 0) {
    const auto* base = reinterpret_cast<__attribute__((address_space(3))) const char*>((uintptr_t)at);
    return *reinterpret_cast<__attribute__((address_space(3))) const V*>(base + offset);
}
__device__ __forceinline__ s16x4 lds_read_transposed(uint32_t at, int offset) {
    auto* base = reinterpret_cast<__attribute__((address_space(3))) char*>((uintptr_t)at);
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(base + offset));
}

template <typename T>
struct Prob;
template <>
struct Prob<__bf16> {
    static constexpr float kBias = 24.0f;   // m lies this far above the maximum (fp32 sums of large values stay finite)
    static constexpr float kRise = 8.0f;    // a row whose largest score would move m further up than this does so
    static constexpr float kMost = 0x1p-9f;  // for a lane's sum of a tile that reaches this
    // Below this m, rounded in fp32, lies so near its place that keys with the largest score do not reach kMost: half a step
    // is 8 at most, 32 weights 2^(-24 + 8 + 5). Further out m might not move while o and l are scaled, tile by tile.
    static constexpr float kFar = 0x1p28f;
    static __device__ __forceinline__ float sum(bf16x2 a, float c) {
        return __builtin_amdgcn_fdot2_f32_bf16(a, bf16x2{(__bf16)1.0f, (__bf16)1.0f}, c, false);
    }
};
template <>
struct Prob<_Float16> {
    // The largest weight is 2^8 or more, so that those down to 2^-22 of it are normal numbers; smaller ones are multiples of
    // 2^-24, off by at most 2^-25: 2^-33 of the row's sum each. Scores of standard deviation 3 raise m more often than a
    // largest weight of 1 did (8 prompts of up to 4096, 24 heads of 64: 195 us then, 203 now; of 1: 206 both).
    static constexpr float kBias = -8.0f;
    static constexpr float kRise = 0.0f;
    static constexpr float kMost = 65504.0f;  // the largest fp16: no weight below it has become infinite
    static constexpr float kFar = 0x1p24f;  // half a step 1/2, 32 weights 2^(8 + 1/2 + 5)
    static __device__ __forceinline__ float sum(f16x2 a, float c) {
        return __builtin_amdgcn_fdot2(a, f16x2{(_Float16)1.0f, (_Float16)1.0f}, c, false);
    }
};

// 16-byte chunk `chunk` of row `row` lies at this place of the row in LDS. K is read 16 bytes of 16 rows at a time, V 64
// bytes of four rows (the transposing read): either way the lanes served together cover the 64 banks.
template <int HD>
__device__ __forceinline__ int k_place(int row, int chunk) {
    return chunk ^ (HD == 64 ? (row >> 1) & 7 : row & 15);
}
template <int HD>
__device__ __forceinline__ int v_place(int row, int chunk) {
    return chunk ^ (HD == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3));
}

// One wave's rows: the online softmax state and the queries of 32 rows, lane l holding row l % 32 (l / 32: which half of
// the depths or keys).
template <typename T, int HD>
struct WaveRows {
    typedef typename PipeMfma<T>::vec Vec;
    typedef typename PipeMfma<T>::pair Pair;
    static constexpr int kD = HD / 32;
    Vec q[HD / 16];
    f32x16 o[kD];        // o[t][r]: column 32 t + 8 (r / 4) + 4 (lane / 32) + r % 4
    float m, l;          // reference point; this lane's part of the sum
    float scale;
    uint32_t k_lane;     // this lane's bytes of a K tile: row lane % 32, chunk lane / 32 (XORed with 32 c for depths 16 c)
    uint32_t v_lane;     // and of a V tile for the transposing reads (XORed with 64 t for columns 32 t)

    __device__ __forceinline__ void start(float scale_log2, int lane) {
#pragma unroll
        for (int t = 0; t < kD; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[t][r] = 0.0f;
        m = 0.0f, l = 0.0f, scale = scale_log2;
        const int row = lane & 31, half = lane >> 5;
        k_lane = row * (HD * 2) + k_place<HD>(row, half) * 16;
        // lanes 16 g .. + 15 read four keys x 16 columns: key lane % 16 / 4 of the four, columns 4 (lane % 4) .. + 3
        const int key = (lane & 15) >> 2, col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        v_lane = (4 * half + key) * (HD * 2) + v_place<HD>(key, col / 8) * 16 + (col % 8) * 2;
    }

    // Query row `row` (its first element; null: zeros).
    __device__ __forceinline__ void load_q(const uint16_t* row, int lane) {
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
            uint4 raw = make_uint4(0, 0, 0, 0);
            if (row) raw = *reinterpret_cast<const uint4*>(row + 16 * c + 8 * (lane >> 5));
            q[c] = __builtin_bit_cast(Vec, raw);
        }
    }

    // V^T operand: columns 32 t + lane % 32, keys 16 kc + 4 (lane / 32) + {0 .. 3, 8 .. 11} of the tile at LDS address v.
    __device__ __forceinline__ Vec v_operand(uint32_t v, int kc, int t) const {
        const uint32_t at = v + (v_lane ^ (64 * t));
        const s16x4 lo = lds_read_transposed(at, kc * 16 * (HD * 2)), hi = lds_read_transposed(at, (kc * 16 + 8) * (HD * 2));
        return __builtin_bit_cast(Vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }

    // Values of V that are no number in a tile that masks some rows' keys: 0 * inf would reach the rows that do not see the
    // key. Such tiles are looked over (a pass over the tile's bytes; rare in a long sequence); where one holds an infinity or
    // a NaN, those are added to the rows that see their key, one by one, and cleared in LDS, and the product follows as always.
    static constexpr uint32_t kExp = std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u;
    // whether the `bytes` at LDS address `at` hold one (exponent all ones)
    static __device__ __forceinline__ bool not_finite(uint32_t at, int bytes, int lane) {
        constexpr uint32_t kOne = kExp == 0x7f80u ? 0x00800080u : 0x04000400u;
        uint32_t seen = 0;
        for (int i = 0; i < bytes; i += 1024) {
            const u32x4 w = lds_read<u32x4>(at + i + 16 * lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) seen |= (w[e] & 0x7fff7fffu) + kOne;
        }
        return __builtin_amdgcn_ballot_w64((seen & 0x80008000u) != 0) != 0;
    }
    // this wave's rows: add what they see of `keys` keys
    __device__ __forceinline__ void add_not_finite(uint32_t v, int keys, int visible, int lane) {
        for (int key = 0; key < keys; ++key) {
#pragma unroll
            for (int t = 0; t < kD; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int col = t * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                    const uint16_t x = lds_read<uint16_t>(v + key * (HD * 2) + v_place<HD>(key, col / 8) * 16 + (col % 8) * 2);
                    if ((x & kExp) == kExp && key < visible) o[t][r] += (float)__builtin_bit_cast(T, x);
                }
        }
    }
    static __device__ __forceinline__ void clear_not_finite(uint32_t at, int bytes, int lane) {
        for (int i = 2 * lane; i < bytes; i += 128)
            if ((lds_read<uint16_t>(at + i) & kExp) == kExp)
                *reinterpret_cast<__attribute__((address_space(3))) uint16_t*>((uintptr_t)(at + i)) = 0;
    }

    // One tile of 32 NS keys at LDS addresses k, v. masked: the lane's row sees only the tile's keys below `visible` (may be
    // 0 or less). first: the rows' first tile, which sets m. Both are the same in every lane.
    template <int NS>
    __device__ __forceinline__ void tile(uint32_t k, uint32_t v, bool first, bool masked, int visible, int lane) {
        const int half = lane >> 5;
        f32x16 s[NS];
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
                const Vec a = lds_read<Vec>(k + (k_lane ^ (32 * c)), st * 32 * (HD * 2));
                s[st] = PipeMfma<T>::run(a, q[c], c == 0 ? f32x16{} : s[st]);
            }
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[st][r] = fmaf(s[st][r], scale, -m);
        if (masked) {
            int rel = visible - 4 * half;
            asm volatile("" : "+v"(rel));  // keeps this a branch: as selects it would cost every tile 100 instructions
#pragma unroll
            for (int st = 0; st < NS; ++st)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (st * 32 + 8 * (r >> 2) + (r & 3) >= rel) s[st][r] = -INFINITY;
        }
        auto maximum = [&]() __attribute__((always_inline)) {
            float mx = -INFINITY;
#pragma unroll
            for (int st = 0; st < NS; ++st)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[st][r]);
            return fmaxf(mx, __shfl_xor(mx, 32));
        };
        // Where a row's reference point goes from m: kBias above its largest score, which lies mx above m. Scores of kFar and
        // more are their own reference point.
        auto raise_to = [&](float mx) __attribute__((always_inline)) {
            return mx + (fabsf(m + mx) < Prob<T>::kFar ? Prob<T>::kBias : 0.0f);
        };
        auto lower = [&](float by) __attribute__((always_inline)) {
            m += by;
#pragma unroll
            for (int st = 0; st < NS; ++st)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[st][r] -= by;
        };
        if (first) {
            const float mx = maximum();
            // A row without keys keeps weights of 0. One whose scores here are all -inf starts far below the scores to come,
            // so that the first finite ones raise m (as rounded there: 2^-13 in the exponent, as much as an fp16 weight).
            lower(mx == -INFINITY ? -0x1p12f : raise_to(mx));
        }
        // the probabilities as MFMA operands (chunk kc: 16 keys) and this lane's sum of them as rounded
        Vec pf[2 * NS];
        float lt;
        auto probabilities = [&]() __attribute__((always_inline)) {
            float ls[NS] = {};
#pragma unroll
            for (int st = 0; st < NS; ++st)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const f32x2 e = {__builtin_amdgcn_exp2f(s[st][r]), __builtin_amdgcn_exp2f(s[st][r + 1])};
                    const Pair h = __builtin_convertvector(e, Pair);
                    pf[2 * st + (r >> 3)][r & 7] = h.x;
                    pf[2 * st + (r >> 3)][(r & 7) + 1] = h.y;
                    ls[st] = Prob<T>::sum(h, ls[st]);
                }
            lt = ls[0];
            if (NS > 1) lt += ls[NS - 1];
        };
        probabilities();
        // A lane whose probabilities sum to kMost or more (2^8 to 2^15 times the largest that there was), or to inf or NaN,
        // sends the wave through the rare path: rows whose largest score lies kRise beyond its place below m raise m, scale o
        // and l, and the tile's probabilities are taken again. Rows that stay have weights of up to 2^8 (bf16: 2^-16).
        if (__builtin_amdgcn_ballot_w64(!(lt < Prob<T>::kMost)) != 0) {
            const float to = raise_to(maximum()), delta = to > Prob<T>::kRise ? to : 0.0f, alpha = __builtin_amdgcn_exp2f(-delta);
            l *= alpha;
#pragma unroll
            for (int t = 0; t < kD; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[t][r] *= alpha;
            lower(delta);
            probabilities();
        }
        l += lt;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kc = 0; kc < 2 * NS; ++kc)
#pragma unroll
            for (int t = 0; t < kD; ++t) o[t] = PipeMfma<T>::run(v_operand(v, kc, t), pf[kc], o[t]);
        __builtin_amdgcn_s_setprio(0);
    }
};

// Loads ROWS rows of HD elements into LDS (16-byte chunks in their places), all of a wave's lanes together; a row past
// `last` takes row `last` instead. PLACE: whose places.
template <int HD, int ROWS, bool IS_V>
struct RowLoader {
    static constexpr int kPer = 512 / HD;            // rows of one 1 KB load
    static constexpr int kLoads = ROWS / kPer;
    uint32_t off[kLoads];
    __device__ __forceinline__ void start(int first, int lane, uint32_t ld_bytes) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) off[j] = offset(first, j, lane, ld_bytes, 0x7fffffff);
    }
    static __device__ __forceinline__ uint32_t offset(int first, int j, int lane, uint32_t ld_bytes, int last) {
        const int row = first + j * kPer + lane / (HD / 8), place = lane % (HD / 8);
        const int chunk = IS_V ? v_place<HD>(row, place) : k_place<HD>(row, place);
        return (uint32_t)min(row, last) * ld_bytes + chunk * 16;
    }
    __device__ __forceinline__ void load(const char* base, uint32_t lds) const {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) lds_dma16(base, off[j], lds + 1024 * j);
    }
    static __device__ __forceinline__ void load_short(const char* base, uint32_t lds, int first, int lane, uint32_t ld_bytes, int last) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) lds_dma16(base, offset(first, j, lane, ld_bytes, last), lds + 1024 * j);
    }
};

// The parts first, first + step, .. of a row merged by 16 lanes (sub: which), HD / 16 columns each: entry(i) is part i's
// unnormalized columns and its (m, l); parts without a sum (m = -inf) are left out, others keep what is no number in them
// whatever their weight. Bound by the latency of its loads, so those of eight parts go together and the maximum is a running
// one (a pass for the maximum first: 4 us more for the call on 48 sequences below).
template <int HD, typename F>
__device__ __forceinline__ void merge_parts(const PackedParams& p, int first, int step, int parts, int sub, F&& entry,
                                            float (&o)[HD / 16], float& m, float& l) {
    constexpr int N = HD / 16, kAtOnce = 8;  // parts whose loads are in flight together
    const float* const ml = p.parts + p.part_count * HD;
    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c) o[c] = 0.0f;
    for (int i = first; i < parts; i += kAtOnce * step) {
        float2 e[kAtOnce];
        float4 v[kAtOnce][N / 4];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int64_t at = entry(min(i + u * step, parts - 1));
            e[u] = *reinterpret_cast<const float2*>(ml + 2 * at);
#pragma unroll
            for (int c = 0; c < N / 4; ++c) v[u][c] = *reinterpret_cast<const float4*>(p.parts + at * HD + sub * N + 4 * c);
        }
        float to = m;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            if (i + u * step >= parts) e[u].x = -INFINITY;
            to = fmaxf(to, e[u].x);
        }
        const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to);
        m = to, l *= keep;
#pragma unroll
        for (int c = 0; c < N; ++c) o[c] *= keep;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const bool none = e[u].x == -INFINITY;  // (selects, no branch: the loads of all eight stay in front of it)
            const float wgt = none ? 0.0f : __builtin_amdgcn_exp2f(e[u].x - m);
            l = fmaf(wgt, none ? 0.0f : e[u].y, l);
            const float* const f = reinterpret_cast<const float*>(v[u]);
#pragma unroll
            for (int c = 0; c < N; ++c) o[c] = fmaf(wgt, none ? 0.0f : f[c], o[c]);
        }
    }
}
template <typename T, int HD>
__device__ __forceinline__ void store_row(const PackedParams& p, const float (&o)[HD / 16], float l, int sub, int64_t to) {
    constexpr int N = HD / 16;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint32_t w[N / 2];
#pragma unroll
    for (int c = 0; c < N; c += 2) {
        const f32x2 f = {o[c] * inv, o[c + 1] * inv};
        w[c / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, typename PipeMfma<T>::pair));
    }
    uint16_t* const out = static_cast<uint16_t*>(p.out) + to + sub * N;
    if constexpr (N == 8)
        *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
    else
        *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
}

// The row tile of slot `slot`: its sequence, first row, and the keys that its last row sees.
struct TileOf {
    Rows q, k;
    int64_t rows, row0;
    int keys;
};
__device__ __forceinline__ int last_key(const PackedParams& p, const Rows& q, const Rows& k, int64_t row) {
    return p.causal ? k.count - (q.count - (int)(row / p.group)) : k.count - 1;
}
// The tiles in the order of their index in their sequence, the last tiles (which see the most keys) first, so that the
// workgroups that take longest do not start last (8 prompts of up to 4096, 24 heads of 64: 204 us by sequence, 197 so; the
// search costs a call whose tiles are cut into parts more than it gains): rank r is tile t where N(t + 1) <= r < N(t), N(t) = sum_s max(0, n_s - t)
// over the sequences' tile counts n_s. Up to kOrdered sequences, four a lane; -1 behind the last tile.
constexpr int kOrdered = 256;
__device__ __forceinline__ int ordered_tile(const PackedParams& p, int rank, int& s) {
    const int lane = threadIdx.x & 63;
    int n[kOrdered / 64], most = 0;
#pragma unroll
    for (int c = 0; c < kOrdered / 64; ++c) {
        const int i = lane + 64 * c;
        n[c] = 0;
        if (64 * c < p.seqs && i < p.seqs) {
            const int64_t rows = (int64_t)rows_of(p.cu_q, i, p.total_q).count * p.group;
            n[c] = rows <= p.few_rows ? 0 : (int)((rows + kTileRows - 1) / kTileRows);
        }
        most = max(most, n[c]);
    }
    auto all = [&](int v, auto op) __attribute__((always_inline)) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) v = op(v, __shfl_xor(v, off));
        return __builtin_amdgcn_readfirstlane(v);
    };
    auto count = [&](int t) __attribute__((always_inline)) {
        int v = 0;
#pragma unroll
        for (int c = 0; c < kOrdered / 64; ++c) v += max(n[c] - t, 0);
        return all(v, [](int a, int b) { return a + b; });
    };
    int lo = 0, hi = all(most, [](int a, int b) { return max(a, b); });  // N(lo) > rank >= N(hi)
    if (count(0) <= rank) return -1;
    int above = 0;  // N(hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1, c = count(mid);
        if (c > rank)
            lo = mid;
        else
            hi = mid, above = c;
    }
    int k = rank - above;  // the k-th sequence of more than lo tiles
#pragma unroll
    for (int c = 0; c < kOrdered / 64; ++c) {
        const uint64_t mask = __builtin_amdgcn_ballot_w64(n[c] > lo);
        const int prefix = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        const uint64_t hit = __builtin_amdgcn_ballot_w64(n[c] > lo && prefix == k);
        if (hit) s = 64 * c + __builtin_ctzll(hit);
        k -= __popcll(mask);
    }
    return lo;
}
__device__ __forceinline__ TileOf tile_of(const PackedParams& p, int64_t slot) {
    int s = 0;
    int64_t tile;
    if (p.ordered) {
        tile = ordered_tile(p, (int)slot, s);
    } else {
        auto first_slot = [&](int i) { return (int64_t)clamped(p.cu_q, i, p.total_q) * p.group / kTileRows + i; };
        slot = p.slots - 1 - slot;
        s = find_sequence(p.seqs, slot, first_slot);
        tile = slot - first_slot(s);
    }
    TileOf t;
    t.q = rows_of(p.cu_q, s, p.total_q), t.k = keys_of(p, s);
    t.rows = (int64_t)t.q.count * p.group, t.row0 = tile * kTileRows;
    if (t.row0 < 0 || t.row0 >= t.rows || t.rows <= p.few_rows) t.row0 = -1;  // no tile, or not attn_packed_tile's
    t.keys = t.row0 < 0 ? 0 : max(last_key(p, t.q, t.k, min(t.row0 + kTileRows, t.rows) - 1) + 1, 0);
    return t;
}
__device__ __forceinline__ int tile_parts_of(const PackedParams& p, int keys) {
    return min(max(pieces(keys, p.tile_chunk), 1), p.tile_parts);
}

template <typename T, int HD>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void attn_packed_tile(PackedParams p) {
    constexpr int kBytes = kTileKeys * HD * 2;  // of a K or V tile
    __shared__ __attribute__((aligned(1024))) char lds[4 * kBytes];  // [buffer][K, V]
    __shared__ int vote[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // neighbouring workgroups take different key heads, so a head's tiles meet in one XCD's L2
    const int kvh = blockIdx.x % p.kv_heads;
    const int64_t slot = blockIdx.x / p.kv_heads;
    const TileOf at = tile_of(p, slot);
    const int part = blockIdx.y, parts = tile_parts_of(p, at.keys);
    if (at.row0 < 0 || part >= parts) return;
    const Rows rq = at.q, rk = at.k;
    const int64_t rows = at.rows;

    // this lane's row, and the last key it sees (-1: none)
    const int64_t wave_row = at.row0 + wave * 32, row = wave_row + (lane & 31);
    const bool live = row < rows;
    const int token = live ? (int)(row / p.group) : 0, head = kvh * p.group + (live ? (int)(row - (int64_t)token * p.group) : 0);
    const int last = live ? last_key(p, rq, rk, row) : -1;
    // rows past the sequence's hold zeros and are not stored, so they need no mask
    const int wave_min = wave_row < rows ? __builtin_amdgcn_readfirstlane(last_key(p, rq, rk, wave_row)) : -1;
    const int wave_max = wave_row < rows ? __builtin_amdgcn_readfirstlane(last_key(p, rq, rk, min(wave_row + 31, rows - 1))) : -1;
    const int all_min = last_key(p, rq, rk, at.row0);  // every row of the workgroup sees the keys up to here
    // this part's tiles
    const int begin = part * (p.tile_chunk / kTileKeys);
    const int end = pieces(part == parts - 1 ? at.keys : (part + 1) * p.tile_chunk, kTileKeys);

    WaveRows<T, HD> w;
    w.start(p.scale_log2, lane);
    w.load_q(live ? static_cast<const uint16_t*>(p.q) + (int64_t)(rq.first + token) * p.ldq + (int64_t)head * HD : nullptr, lane);

    const uint32_t lds0 = lds_address(lds);
    const uint32_t ldk = (uint32_t)(p.ldk * 2), ldv = (uint32_t)(p.ldv * 2);
    const char* const kbase = static_cast<const char*>(p.k) + ((int64_t)rk.first * p.ldk + (int64_t)kvh * HD) * 2;
    const char* const vbase = static_cast<const char*>(p.v) + ((int64_t)rk.first * p.ldv + (int64_t)kvh * HD) * 2;
    typedef RowLoader<HD, 16, false> LoadK;
    typedef RowLoader<HD, 16, true> LoadV;
    LoadK lk;
    LoadV lv;
    lk.start(16 * wave, lane, ldk);
    lv.start(16 * wave, lane, ldv);
    auto load = [&](int j) __attribute__((always_inline)) {
        const char* kb = uniform_ptr(kbase + (int64_t)j * kTileKeys * ldk);
        const char* vb = uniform_ptr(vbase + (int64_t)j * kTileKeys * ldv);
        const uint32_t at = lds0 + (j & 1) * 2 * kBytes + wave * (kBytes / 4);
        const int left = rk.count - 1 - j * kTileKeys;
        if (left >= kTileKeys - 1) {
            lk.load(kb, at);
            lv.load(vb, at + kBytes);
        } else {
            LoadK::load_short(kb, at, 16 * wave, lane, ldk, left);
            LoadV::load_short(vb, at + kBytes, 16 * wave, lane, ldv, left);
        }
    };
    if (begin < end) load(begin);
    for (int j = begin; j < end; ++j) {
        wait_vm<0>();       // this wave's part of tile j
        __syncthreads();    // everyone's part; tile j - 1 is read
        if (j + 1 < end) load(j + 1);
        const int j0 = j * kTileKeys;
        const uint32_t k = lds0 + (j & 1) * 2 * kBytes, v = k + kBytes;
        if (j0 + kTileKeys - 1 > all_min) {  // some row of the workgroup sees the tile in part: V must be finite
            const bool found = WaveRows<T, HD>::not_finite(v + wave * (kBytes / 4), kBytes / 4, lane);
            if (lane == 0) vote[wave] = found;
            __syncthreads();
            if (vote[0] | vote[1] | vote[2] | vote[3]) {
                w.add_not_finite(v, kTileKeys, last + 1 - j0, lane);
                __syncthreads();
                WaveRows<T, HD>::clear_not_finite(v + wave * (kBytes / 4), kBytes / 4, lane);
            }
            __syncthreads();  // cleared; the votes are read
        }
        if (j0 > wave_max) continue;
        w.template tile<2>(k, v, j == begin, j0 + kTileKeys - 1 > wave_min, last + 1 - j0, lane);
    }

    const float l = w.l + __shfl_xor(w.l, 32);
    if (parts > 1) {
        const int64_t to = p.tile_entry + ((slot * p.tile_parts + part) * p.kv_heads + kvh) * kTileRows + wave * 32 + (lane & 31);
        if (!live) return;
#pragma unroll
        for (int t = 0; t < HD / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<float4*>(p.parts + to * HD + t * 32 + 8 * (r >> 2) + 4 * (lane >> 5)) =
                    make_float4(w.o[t][r], w.o[t][r + 1], w.o[t][r + 2], w.o[t][r + 3]);
        if (lane < 32)
            *reinterpret_cast<float2*>(p.parts + p.part_count * HD + 2 * to) = make_float2(l > 0.0f || l != l ? w.m : -INFINITY, l);
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    // the wave's 32 rows through its own part of LDS (after the last reads of the tiles) and out in 16-byte pieces
    __syncthreads();
    constexpr int kPitch = HD + 8;
    uint16_t* const ob = reinterpret_cast<uint16_t*>(lds) + wave * 32 * kPitch;
#pragma unroll
    for (int t = 0; t < HD / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const f32x2 f = {w.o[t][r] * inv, w.o[t][r + 1] * inv};
            *reinterpret_cast<uint32_t*>(&ob[(lane & 31) * kPitch + t * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)]) =
                __builtin_bit_cast(uint32_t, __builtin_convertvector(f, typename PipeMfma<T>::pair));
        }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
        const int r = (lane + 64 * i) / (HD / 8), c = (lane + 64 * i) % (HD / 8);
        const int64_t to = wave_row + r;
        if (to < rows) {
            const int tk = (int)(to / p.group);
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + (int64_t)(rq.first + tk) * p.ldo +
                                      (int64_t)(kvh * p.group + (int)(to - (int64_t)tk * p.group)) * HD + 8 * c) =
                *reinterpret_cast<const uint4*>(&ob[r * kPitch + 8 * c]);
        }
    }
}

// Into how many parts attn_packed_few cuts a sequence, and the first one's entry.
__device__ __forceinline__ int parts_of(const PackedParams& p, int64_t rows, int lk) {
    const int parts = rows > p.part_rows ? 1 : max(pieces(lk, p.chunk), 1);
    return p.per ? min(parts, p.per) : parts;
}
__device__ __forceinline__ int64_t first_chunk(const PackedParams& p, int s, int first_key) {
    return p.per ? (int64_t)s * p.per : (int64_t)first_key / p.chunk + s;
}
// The first part's entry in the workspace, of a sequence that is cut: its first chunk's, or, where few of many sequences can
// be cut, the half chunk that its first key is in. (A cut sequence has more than one chunk of keys, x > 1 chunks, and
// takes ceil(x) <= floor(2 x) entries, so it ends before the next one's first.)
__device__ __forceinline__ int64_t first_part(const PackedParams& p, int s, int first_key) {
    return p.sparse ? 2 * (int64_t)first_key / p.chunk : first_chunk(p, s, first_key);
}

// NW waves: 4 for long key ranges, so that a CU holds two or three workgroups and one's loads, start and merge pass under the
// others' work (48 sequences of up to 8192 keys, 32 heads on 8 of 128: 113 us in this kernel, 4.9 TB/s; one workgroup a CU
// whose waves load a tile ahead of their work into a second buffer 13 us more); as many as LDS holds for short ones, which
// are then one or two tiles a wave and need no cutting, no workspace and no merge (500 keys, 16 heads of 64: 9.2 us, cut 2 us
// more).
template <typename T, int HD, int NW>
__global__ __launch_bounds__(64 * NW, NW > 4 ? NW / 4 : HD == 64 ? 3 : 2) void attn_packed_few(PackedParams p) {
    constexpr int kBytes = kFewKeys * HD * 2;  // of a wave's K or V tile
    constexpr int kPitch = HD + 4;
    constexpr int kMerge = NW * 32 * kPitch * 4, kTiles = NW * 2 * kBytes;
    __shared__ __attribute__((aligned(1024))) char lds[kMerge > kTiles ? kMerge : kTiles];  // [wave][K, V]; the merge
    __shared__ float red_m[NW][32], red_l[NW][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kvh = blockIdx.x % p.kv_heads;
    const int64_t slot = blockIdx.x / p.kv_heads;
    const int s = p.per ? (int)(slot / p.per)
                        : find_sequence(p.seqs, slot, [&](int i) { return first_chunk(p, i, clamped(p.cu_k, i, p.total_k)); });
    const Rows rq = rows_of(p.cu_q, s, p.total_q), rk = keys_of(p, s);
    const int64_t rows = (int64_t)rq.count * p.group;
    const int part = (int)(slot - first_chunk(p, s, rk.first)), parts = parts_of(p, rows, rk.count);
    // (keys before the first sequence leave entries before its first one)
    if (rows == 0 || rows > p.few_rows || part < 0 || part >= parts) return;
    const int key0 = part * p.chunk, key1 = part == parts - 1 ? rk.count : key0 + p.chunk;

    const uint32_t k = lds_address(lds) + wave * 2 * kBytes, v = k + kBytes;  // this wave's tile
    const uint32_t ldk = (uint32_t)(p.ldk * 2), ldv = (uint32_t)(p.ldv * 2);
    const char* const kbase = static_cast<const char*>(p.k) + ((int64_t)(rk.first + key0) * p.ldk + (int64_t)kvh * HD) * 2;
    const char* const vbase = static_cast<const char*>(p.v) + ((int64_t)(rk.first + key0) * p.ldv + (int64_t)kvh * HD) * 2;
    typedef RowLoader<HD, kFewKeys, false> LoadK;
    typedef RowLoader<HD, kFewKeys, true> LoadV;

    for (int64_t row0 = 0; row0 < rows; row0 += 32) {
        const int64_t row = row0 + (lane & 31);
        const bool live = row < rows;
        const int token = live ? (int)(row / p.group) : 0, head = kvh * p.group + (live ? (int)(row - (int64_t)token * p.group) : 0);
        const int last = live ? last_key(p, rq, rk, row) - key0 : -1;  // inside the chunk
        const int all = last_key(p, rq, rk, row0) - key0;  // every row sees the chunk's keys up to here
        const int end = min(last_key(p, rq, rk, min(row0 + 31, rows - 1)) + 1, key1) - key0;  // keys of the chunk that some row sees
        const int tiles = pieces(end, kFewKeys);

        WaveRows<T, HD> w;
        w.start(p.scale_log2, lane);
        w.load_q(live ? static_cast<const uint16_t*>(p.q) + (int64_t)(rq.first + token) * p.ldq + (int64_t)head * HD : nullptr, lane);
        auto load = [&](int j) __attribute__((always_inline)) {
            const char* kb = uniform_ptr(kbase + (int64_t)j * kFewKeys * ldk);
            const char* vb = uniform_ptr(vbase + (int64_t)j * kFewKeys * ldv);
            const int left = rk.count - 1 - key0 - j * kFewKeys;
            LoadK::load_short(kb, k, 0, lane, ldk, left);
            LoadV::load_short(vb, v, 0, lane, ldv, left);
        };
        if (wave < tiles) load(wave);
        for (int j = wave; j < tiles; j += NW) {
            wait_vm<0>();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            const int j0 = j * kFewKeys;
            const int visible = min(last + 1, key1 - key0) - j0;
            const bool masked = j0 + kFewKeys - 1 > all || j0 + kFewKeys > key1 - key0;
            if (masked && WaveRows<T, HD>::not_finite(v, kBytes, lane)) {
                w.add_not_finite(v, kFewKeys, visible, lane);
                WaveRows<T, HD>::clear_not_finite(v, kBytes, lane);
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            }
            w.template tile<1>(k, v, j == wave, masked, visible, lane);
            if (j + NW < tiles) {
                __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the tile is read
                load(j + NW);
            }
        }

        // merge the waves: every tile is read (its loads have landed), so the buffers take the partial rows
        __syncthreads();
        float* const red = reinterpret_cast<float*>(lds);
        const float l = w.l + __shfl_xor(w.l, 32);
        if (lane < 32) {
            red_m[wave][lane] = l > 0.0f || l != l ? w.m : -INFINITY;
            red_l[wave][lane] = l;
        }
#pragma unroll
        for (int t = 0; t < HD / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                f32x4 f = {w.o[t][r], w.o[t][r + 1], w.o[t][r + 2], w.o[t][r + 3]};
                *reinterpret_cast<f32x4*>(&red[(wave * 32 + (lane & 31)) * kPitch + t * 32 + 8 * (r >> 2) + 4 * (lane >> 5)]) = f;
            }
        __syncthreads();
        // a row to 2 NW threads, N of its columns each
        constexpr int N = HD / (2 * NW);
        const int r = threadIdx.x / (2 * NW), piece = threadIdx.x % (2 * NW);
        const int64_t at = row0 + r;
        if (at < rows) {
            float mx = -INFINITY, sum = 0.0f, f[N] = {};
#pragma unroll
            for (int i = 0; i < NW; ++i) mx = fmaxf(mx, red_m[i][r]);
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                if (red_m[i][r] == -INFINITY) continue;
                const float wgt = __builtin_amdgcn_exp2f(red_m[i][r] - mx);
                sum = fmaf(wgt, red_l[i][r], sum);
#pragma unroll
                for (int d = 0; d < N; ++d) f[d] = fmaf(wgt, red[(i * 32 + r) * kPitch + piece * N + d], f[d]);
            }
            if (parts == 1) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const int tk = (int)(at / p.group);
                uint16_t* out = static_cast<uint16_t*>(p.out) + (int64_t)(rq.first + tk) * p.ldo +
                                (int64_t)(kvh * p.group + (int)(at - (int64_t)tk * p.group)) * HD + piece * N;
#pragma unroll
                for (int d = 0; d < N; d += 2) {
                    const f32x2 g = {f[d] * inv, f[d + 1] * inv};
                    *reinterpret_cast<uint32_t*>(out + d) = __builtin_bit_cast(uint32_t, __builtin_convertvector(g, typename PipeMfma<T>::pair));
                }
            } else {
                const int64_t to = ((first_part(p, s, rk.first) + part) * p.kv_heads + kvh) * p.part_rows + at;
#pragma unroll
                for (int d = 0; d < N; d += 2)
                    *reinterpret_cast<float2*>(p.parts + to * HD + piece * N + d) = make_float2(f[d], f[d + 1]);
                if (piece == 0)
                    *reinterpret_cast<float2*>(p.parts + p.part_count * HD + 2 * to) = make_float2(mx, sum);
            }
        }
        __syncthreads();
    }
}

// Merges the parts of the sequences that attn_packed_few cut. G groups of 16 lanes take every G-th part of a row each (few
// rows of many parts: G = 16, a workgroup a row), and their sums are added in order through LDS. SPARSE: a workgroup takes 16
// rows of an entry and works where a sequence's parts begin there.
template <typename T, int HD, int G, bool SPARSE>
__global__ __launch_bounds__(256) void attn_packed_combine(PackedParams p) {
    static_assert(!SPARSE || G == 1);
    constexpr int N = HD / 16;
    __shared__ float red_o[G > 1 ? G : 1][HD], red_m[G], red_l[G];
    const int grp = threadIdx.x >> 4, sub = threadIdx.x & 15;
    const int64_t id = G > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 16 + grp;  // (sequence, key head, row)
    int r = (int)(id % p.part_rows), kvh = (int)(id / p.part_rows % p.kv_heads);
    int64_t sq = id / p.part_rows / p.kv_heads;
    if constexpr (SPARSE) {  // (entry, key head, rows / 16)
        const int blocks = pieces(p.part_rows, 16);
        r = (int)blockIdx.x % blocks * 16 + grp, kvh = (int)blockIdx.x / blocks % p.kv_heads;
        const int64_t entry = (int)blockIdx.x / blocks / p.kv_heads;
        sq = find_sequence(p.seqs, entry, [&](int i) { return first_part(p, i, clamped(p.cu_k, i, p.total_k)); });
        if (first_part(p, (int)sq, clamped(p.cu_k, (int)sq, p.total_k)) != entry) return;
    }
    if (sq >= p.seqs) return;
    const int s = (int)sq;
    const Rows rq = rows_of(p.cu_q, s, p.total_q), rk = keys_of(p, s);
    const int64_t rows = (int64_t)rq.count * p.group;
    const int parts = parts_of(p, rows, rk.count);
    if (r >= rows || rows > p.few_rows || parts == 1) return;
    const int64_t first = first_part(p, s, rk.first) * p.kv_heads + kvh;  // part i: entry first + i kv_heads
    auto entry = [&](int i) { return (first + (int64_t)i * p.kv_heads) * p.part_rows + r; };
    float o[N], m, l;
    merge_parts<HD>(p, G > 1 ? grp : 0, G, parts, sub, entry, o, m, l);
    if constexpr (G > 1) {
#pragma unroll
        for (int c = 0; c < N; ++c) red_o[grp][sub * N + c] = o[c];
        if (sub == 0) red_m[grp] = m, red_l[grp] = l;
        __syncthreads();
        if (grp > 0) return;
        m = -INFINITY, l = 0.0f;
        for (int g = 0; g < G; ++g) m = fmaxf(m, red_m[g]);
#pragma unroll
        for (int c = 0; c < N; ++c) o[c] = 0.0f;
        for (int g = 0; g < G; ++g) {
            if (red_m[g] == -INFINITY) continue;
            const float wgt = __builtin_amdgcn_exp2f(red_m[g] - m);
            l = fmaf(wgt, red_l[g], l);
#pragma unroll
            for (int c = 0; c < N; ++c) o[c] = fmaf(wgt, red_o[g][sub * N + c], o[c]);
        }
    }
    const int tk = r / p.group;
    store_row<T, HD>(p, o, l, sub, (int64_t)(rq.first + tk) * p.ldo + (int64_t)(kvh * p.group + r - tk * p.group) * HD);
}

// The same for the row tiles that attn_packed_tile cut.
template <typename T, int HD>
__global__ __launch_bounds__(256) void attn_packed_combine_tiles(PackedParams p) {
    const int kvh = blockIdx.x % p.kv_heads;
    const int64_t slot = blockIdx.x / p.kv_heads;
    const TileOf at = tile_of(p, slot);
    const int parts = tile_parts_of(p, at.keys), r = blockIdx.y * 16 + (threadIdx.x >> 4);
    const int64_t row = at.row0 + r;
    if (at.row0 < 0 || parts == 1 || row >= at.rows) return;
    const int tk = (int)(row / p.group);
    float o[HD / 16], m, l;
    merge_parts<HD>(p, 0, 1, parts, threadIdx.x & 15,
                    [&](int i) { return p.tile_entry + ((slot * p.tile_parts + i) * p.kv_heads + kvh) * kTileRows + r; }, o, m, l);
    store_row<T, HD>(p, o, l, threadIdx.x & 15,
                     (int64_t)(at.q.first + tk) * p.ldo + (int64_t)(kvh * p.group + (int)(row - (int64_t)tk * p.group)) * HD);
}

// Which kernels a call runs and how it cuts the keys, from the shapes and the length bounds.
struct PackedPlan {
    bool tile, few;
    int64_t slots;      // attn_packed_tile's row tiles
    int few_rows;
    bool wide;          // attn_packed_few's form for short key ranges
    bool many_parts;    // attn_packed_combine's form for few rows of many parts
    int64_t chunk;      // keys of a chunk
    int64_t part_rows;  // 0: no sequence is cut
    int64_t entries;    // chunks
    int64_t per;        // of a sequence, or 0
    int64_t part_entries;  // the workspace's entries for parts of chunks
    bool sparse;        // they go by half chunks of keys
    int64_t tile_chunk, tile_parts;  // attn_packed_tile's keys of a part and parts (1: none is cut)
    int64_t few_entries, tile_entries;  // rows of parts in the workspace
    size_t bytes;       // workspace

    int64_t sparse_grid(int64_t kv_heads) const { return part_entries * kv_heads * ((part_rows + 15) / 16); }
    // whether every launch stays below 2^31 threads
    bool fits(int64_t seqs, int64_t kv_heads) const {
        return std::max({slots * kv_heads, entries * kv_heads, sparse ? sparse_grid(kv_heads) : seqs * kv_heads * part_rows}) <=
               0x7fffffff / 256;
    }
};
PackedPlan packed_plan(int64_t seqs, int64_t total_q, int64_t total_k, int64_t max_q, int64_t max_k, int64_t heads,
                       int64_t kv_heads, int64_t head_dim, bool workspace) {
    PackedPlan w{};
    const int64_t group = heads / kv_heads;
    max_q = max_q > 0 ? std::min(max_q, total_q) : total_q;
    max_k = max_k > 0 ? std::min(max_k, total_k) : total_k;
    w.slots = total_q * group / kTileRows + seqs;
    // Calls of few rows per sequence go to the key chunks; prompts that are their own context (no more keys than queries over
    // all), and calls whose row tiles are cut along the keys anyway, to the row tiles; other batches run both, each sequence
    // by its own rows.
    if (max_q * group <= kFewRows) {
        w.few = true, w.few_rows = 0x7fffffff;
    } else if (total_k <= total_q) {
        w.tile = true, w.few_rows = 0;
    } else {
        w.tile = w.few = true, w.few_rows = kFewRows;
    }
    w.tile_chunk = 0x7fffffff / kTileKeys * kTileKeys, w.tile_parts = 1;
    if (w.tile && workspace) {
        // Row tiles that leave CUs idle are cut along the keys: into parts that fill the device about once, not shorter
        // than kTilePart keys.
        const int64_t room = 256 * (head_dim == 64 ? 3 : 2);
        const int64_t tiles = (total_q * group / kTileRows + (seqs + 1) / 2) * kv_heads, keys = std::min(max_k, total_k / seqs + 1);
        if (tiles < room) {
            int64_t chunk = std::max<int64_t>((tiles * keys / room + kTileKeys - 1) / kTileKeys * kTileKeys, kTilePart);
            w.tile_parts = std::max<int64_t>((max_k + chunk - 1) / chunk, 1);
            // One long sequence among many short ones needs parts of its own length only: the row tiles together get up to
            // eight parts for every place on the device (up to 270 MB of workspace for these), 64 each at most.
            const int64_t most = std::max<int64_t>(std::min<int64_t>(8 * room / (w.slots * kv_heads), 64), 1);
            if (w.tile_parts > most) {
                w.tile_parts = most;
                chunk = (max_k + most * kTileKeys - 1) / (most * kTileKeys) * kTileKeys;
            }
            if (w.tile_parts > 1) w.tile_chunk = chunk, w.few = false, w.few_rows = 0;
        }
    }
    w.tile_entries = w.tile_parts > 1 ? w.slots * w.tile_parts * kv_heads * kTileRows : 0;
    if (w.few) {
        // chunks: about four workgroups a CU over all keys (lengths differ; with k_lens, of all rows at most max_k a
        // sequence), whole rounds of the waves' tiles
        const int64_t unit = kFewWaves * kFewKeys;
        w.chunk = (std::min(total_k, seqs * max_k) * kv_heads / 1024 + unit) / unit * unit;
        w.wide = max_k <= kShortKeys && seqs * kv_heads < (1 << 21);  // a grid holds 2^32 threads
        if (!workspace || w.wide || max_k <= w.chunk) {
            w.chunk = std::max<int64_t>((total_k + unit) / unit * unit, unit);
        } else {
            w.part_rows = std::min<int64_t>(max_q * group, kFewRows);
            w.many_parts = max_k / w.chunk >= 8;
        }
        w.entries = total_k / w.chunk + seqs;
        const int64_t per = std::max<int64_t>((max_k + w.chunk - 1) / w.chunk, 1);
        if (per <= w.entries / seqs) w.per = per, w.entries = seqs * per;
        // Only sequences of more than one chunk have parts, but the list gives every sequence part_rows rows of the workspace
        // (20000 sequences, 32 heads on 8 of 128, no bounds: 5.4 GB). Where that passes kListBytes the entries go by half
        // chunks of keys, 2 total_k / chunk + 1, if they are fewer: 2048 / kv_heads + 1 at most, 70 MB with 64 rows of 128 values.
        const int64_t halves = 2 * total_k / w.chunk + 1;
        w.sparse = w.entries * kv_heads * w.part_rows * (head_dim + 2) * 4 > kListBytes && halves < w.entries;
        w.part_entries = w.sparse ? halves : w.entries;
    }
    w.few_entries = w.part_entries * kv_heads * w.part_rows;
    w.bytes = (size_t)(w.few_entries + w.tile_entries) * (size_t)(head_dim + 2) * 4;
    // (without parts there may be fewer chunks)
    if (workspace && !w.fits(seqs, kv_heads)) return packed_plan(seqs, total_q, total_k, max_q, max_k, heads, kv_heads, head_dim, false);
    return w;
}

template <typename T, int HD>
int run(PackedParams p, const PackedPlan& w, hipStream_t s) {
    if (w.tile) {
        hipLaunchKernelGGL((attn_packed_tile<T, HD>), dim3((unsigned)(w.slots * p.kv_heads), (unsigned)w.tile_parts), dim3(256), 0, s, p);
        if (int rc = check_launch("attn_packed_tile")) return rc;
        if (w.tile_parts > 1) {
            hipLaunchKernelGGL((attn_packed_combine_tiles<T, HD>), dim3((unsigned)(w.slots * p.kv_heads), kTileRows / 16), dim3(256), 0, s, p);
            if (int rc = check_launch("attn_packed_combine_tiles")) return rc;
        }
    }
    if (w.few) {
        const dim3 grid((unsigned)(w.entries * p.kv_heads));
        constexpr int kWide = HD == 64 ? 16 : 8;  // 128 KB of tiles
        if (w.wide)
            hipLaunchKernelGGL((attn_packed_few<T, HD, kWide>), grid, dim3(64 * kWide), 0, s, p);
        else
            hipLaunchKernelGGL((attn_packed_few<T, HD, kFewWaves>), grid, dim3(64 * kFewWaves), 0, s, p);
        if (int rc = check_launch("attn_packed_few")) return rc;
        if (w.part_rows) {
            const int64_t rows = (int64_t)p.seqs * p.kv_heads * w.part_rows;
            if (w.sparse)
                hipLaunchKernelGGL((attn_packed_combine<T, HD, 1, true>), dim3((unsigned)w.sparse_grid(p.kv_heads)), dim3(256), 0, s, p);
            else if (w.many_parts)
                hipLaunchKernelGGL((attn_packed_combine<T, HD, 16, false>), dim3((unsigned)rows), dim3(256), 0, s, p);
            else
                hipLaunchKernelGGL((attn_packed_combine<T, HD, 1, false>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, s, p);
            return check_launch("attn_packed_combine");
        }
    }
    return IDOLQ_OK;
}

}  // namespace
}  // namespace idolq

using namespace idolq;

extern "C" size_t idolq_attention_packed_workspace(int64_t seqs, int64_t total_q, int64_t total_k, int64_t max_q,
                                                   int64_t max_k, int64_t heads, int64_t kv_heads, int64_t head_dim) {
    if (seqs <= 0 || total_q <= 0 || total_k <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0)
        return 0;
    return packed_plan(seqs, total_q, total_k, max_q, max_k, heads, kv_heads, head_dim, true).bytes;
}

extern "C" int idolq_attention_packed(const void* q, const void* k, const void* v, int dtype, int64_t seqs,
                                      const int32_t* cu_q, const int32_t* cu_k, const int32_t* k_lens, int64_t total_q,
                                      int64_t total_k, int64_t max_q, int64_t max_k, int64_t heads, int64_t kv_heads,
                                      int64_t head_dim,
                                      int64_t ldq, int64_t ldk, int64_t ldv, float scale, int causal, void* out,
                                      int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
    if (dtype != IDOLQ_F16 && dtype != IDOLQ_BF16)
        return fail(IDOLQ_EINVAL, "packed attention takes bf16 or fp16 (fp32 sequences: idolq_attention)");
    if (head_dim != 64 && head_dim != 128) return fail(IDOLQ_EINVAL, "packed attention needs head_dim 64 or 128");
    if (seqs < 0 || total_q < 0 || total_k < 0 || max_q < 0 || max_k < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0)
        return fail(IDOLQ_EINVAL, "bad packed attention shape (kv_heads must divide heads)");
    if (seqs > 0xfffff || total_q > 0x7fffffff || total_k > 0x7fffffff || heads > 4096)
        return fail(IDOLQ_EINVAL, "packed attention: too many sequences, rows or heads");
    if (ldq < heads * head_dim || ldo < heads * head_dim || ldk < kv_heads * head_dim || ldv < kv_heads * head_dim)
        return fail(IDOLQ_EINVAL, "row stride smaller than heads * head_dim");
    // offsets inside a tile of 64 rows are 32-bit
    if (ldk > (1 << 24) || ldv > (1 << 24)) return fail(IDOLQ_EINVAL, "packed attention: key row stride above 2^24");
    if (!(scale - scale == 0.0f)) return fail(IDOLQ_EINVAL, "the softmax scale must be finite");
    if (seqs == 0 || total_q == 0) return IDOLQ_OK;
    if (!q || !out || !cu_q || !cu_k || (total_k > 0 && (!k || !v)))
        return fail(IDOLQ_EINVAL, "q, k, v, out and the offsets must be non-null");
    if (!vec8_ok(q, dtype, ldq) || !vec8_ok(k, dtype, ldk) || !vec8_ok(v, dtype, ldv) || !vec8_ok(out, dtype, ldo))
        return fail(IDOLQ_EINVAL, "packed attention needs 16-byte aligned rows");
    PackedPlan w = packed_plan(seqs, total_q, total_k, max_q, max_k, heads, kv_heads, head_dim, true);
    if (w.bytes && (!workspace || workspace_bytes < w.bytes || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
        w = packed_plan(seqs, total_q, total_k, max_q, max_k, heads, kv_heads, head_dim, false);
    if (!w.fits(seqs, kv_heads)) return fail(IDOLQ_EINVAL, "packed attention: too many sequences, rows or heads");
    const RowBlock to{out, total_q, ldo * 2, heads * head_dim * 2};
    if (rows_overlap(to, {q, total_q, ldq * 2, heads * head_dim * 2}) || rows_overlap(to, {k, total_k, ldk * 2, kv_heads * head_dim * 2}) ||
        rows_overlap(to, {v, total_k, ldv * 2, kv_heads * head_dim * 2}))
        return fail(IDOLQ_EINVAL, "packed attention: out must not overlap q, k or v");
    PackedParams p{};
    p.q = q, p.k = k, p.v = v, p.out = out, p.cu_q = cu_q, p.cu_k = cu_k, p.k_lens = k_lens;
    p.ldq = ldq, p.ldk = ldk, p.ldv = ldv, p.ldo = ldo;
    p.total_q = (int)total_q, p.total_k = (int)total_k, p.seqs = (int)seqs;
    p.heads = (int)heads, p.kv_heads = (int)kv_heads, p.group = (int)(heads / kv_heads);
    p.causal = causal != 0;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.ordered = seqs > 1 && seqs <= kOrdered && w.tile_parts == 1;
    p.slots = (int)w.slots, p.few_rows = w.few_rows, p.chunk = (int)std::min<int64_t>(w.chunk, 0x7fffffff);
    p.part_rows = (int)w.part_rows, p.per = (int)w.per, p.sparse = w.sparse;
    p.parts = static_cast<float*>(workspace);
    p.part_count = w.few_entries + w.tile_entries;
    p.tile_chunk = (int)w.tile_chunk, p.tile_parts = (int)w.tile_parts, p.tile_entry = w.few_entries;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == IDOLQ_BF16) return head_dim == 64 ? run<__bf16, 64>(p, w, s) : run<__bf16, 128>(p, w, s);
    return head_dim == 64 ? run<_Float16, 64>(p, w, s) : run<_Float16, 128>(p, w, s);
}
