// Matrix-vector products on 4-bit weights with group scales (up to 16 activation rows) for gfx950, on GGUF Q4_0 and Q4_K
// blocks as they are stored: y = act(x W^T + bias + residual).
//
// Groups of 32 codes q share a scale and an offset: Q4_0 w = d (q - 8); Q4_K (super-blocks of 8 groups)
// w = (d sc) q - dmin mn with 6-bit sc and mn. The weights are not rounded: a group contributes
//   scale * sum_j x_j q_j - minimum * sum_j x_j,   minimum = 8 d or dmin mn,
// the sums from the matrix cores in fp32, the scaling in fp32.
//
// The weight bytes bound it (0.5625 a weight, read once), with the vector instructions per weight next: at 8 TB/s a SIMD
// has 2.8 of them for each weight it reads. So codes become MFMA operands without arithmetic: a masked shift puts two
// nibbles of a dword into the mantissas of two 16-bit values 16 + q (bf16 0x4180 | q << 3, fp16 0x4c00 | q << 6), one
// instruction a weight, and the 16s leave with a second product of the same activations by a constant: -16 (Q4_0: -24, the
// 8 too), which also gives sum x.
//
// v_mfma_f32_16x16x32 multiplies 16 weight rows (B columns, lane l's column l % 16) by 16 A rows, 32 depths at a time,
// eight of them from each lane of a column (its place l / 16).
//
// Up to 4 activations (FEW): lane l loads the 16 code bytes of one place of its row, so the four lanes of a row load 64
// (Q4_0: 72) bytes in a run, and the 32 depths of an MFMA come from up to four groups; A row r is activation r % 4 of
// group r / 4 alone, zero at the other groups' depths. The 16 sums of a weight row are 4 groups x 4 activations, lane l's
// four those of group l / 16 -- whose scale (Q4_0: of the block it loaded) folds them: four FMAs for 32 weights.
//
// 5 to 16 activations: an MFMA takes one group's 32 depths and all 16 activations as A rows. Each lane needs eight codes of
// every group: 8 bytes of the 32 that two groups share (Q4_K), or of the 16 of a block, low nibbles in lanes 0 .. 31 and high
// ones in the others (Q4_0: the halves load two blocks each and swap registers).
//
// fp32 activations enter as three bf16 parts (all 24 bits). A workgroup owns RT row tiles of 16; its 8 waves take steps of
// 256 depths in turn, each reads its own codes and activations into registers, and nothing waits for another wave before
// the end, where their sums are added through LDS in a fixed order.
//
// Measured, weights out of HBM: one bf16 token Q4_K 4096 x 4096 5.7 us, 8192 x 4096 8.2; Q4_0 4096 x 4096 6.4, 16384 x 8192
// 27 (2.8 TB/s); 12 fp16 tokens Q4_0 4096 x 4096 11.9. With a workgroup's activations staged through LDS, a barrier for each
// piece: 7.5, 10.2, 7.9, 25 and 23 us. With a second step's loads ahead in each wave, so fewer waves: 7.3 for 6.4.
#include "common.h"

namespace idolq {
namespace {

constexpr int kMaxM = 16;
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kStep = 256;  // depths a wave multiplies at a time: one Q4_K super-block, eight Q4_0 blocks

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2a __attribute__((ext_vector_type(2), aligned(4)));

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct Q4Params {
    const void* x;
    const uint8_t* w;
    const void* bias;
    const void* res;
    void* y;
    int64_t ldx, row_bytes, ldr, ldy;
    int m, k, n;
    int bias_dt, res_dt, y_dt, act, flags;
};

template <int XT>
struct Operand {  // bf16 operands (fp32 activations as three parts)
    static constexpr uint32_t kBase = 0x41804180u, kMask = 0x00780078u;
    static constexpr int kShift = 3;  // of a nibble into the mantissa
    static constexpr uint32_t kMinus16 = 0xc180c180u, kMinus24 = 0xc1c0c1c0u;
    static __device__ __forceinline__ f32x4 run(uint4 a, uint4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Operand<IDOLQ_F16> {
    static constexpr uint32_t kBase = 0x4c004c00u, kMask = 0x03c003c0u;
    static constexpr int kShift = 6;
    static constexpr uint32_t kMinus16 = 0xcc00cc00u, kMinus24 = 0xce00ce00u;
    static __device__ __forceinline__ f32x4 run(uint4 a, uint4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// The low (HIGH: high) nibbles of eight bytes as operands 16 + q, in the order of bytes 0 2 1 3 4 6 5 7.
template <int XT, bool HIGH>
__device__ __forceinline__ uint4 codes_of(uint32_t w0, uint32_t w1) {
    constexpr int s0 = Operand<XT>::kShift - (HIGH ? 4 : 0), s1 = s0 - 8;  // left shifts of bytes 0, 2 and of bytes 1, 3
    auto put = [](uint32_t w, int s) __attribute__((always_inline)) {
        return ((s >= 0 ? w << (s & 31) : w >> (-s & 31)) & Operand<XT>::kMask) | Operand<XT>::kBase;
    };
    return make_uint4(put(w0, s0), put(w0, s1), put(w1, s0), put(w1, s1));
}

__device__ __forceinline__ uint32_t half_word(const char* at) { return *reinterpret_cast<const uint16_t*>(at); }

// The value of the lane 4 BANKS before, in turn inside 16 lanes.
template <int BANKS>
__device__ __forceinline__ uint32_t turned(uint32_t v) {
    if constexpr (BANKS == 0) return v;
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + 4 * BANKS, 0xf, 0xf, false);  // row_ror
}

// lo in all lanes: a's value of lane l % 32; hi: a's value of lane 32 + l % 32.
__device__ __forceinline__ void both_halves(uint32_t a, uint32_t& lo, uint32_t& hi) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    lo = r[0], hi = r[1];
}

// What lanes read that have no activations at an operand's depths.
__device__ const uint4 zero_activations[8] = {};

// XT: activation type; KIND: block format; FEW: up to 4 activations, else up to 16; VEC: activation rows can be read 16
// bytes at a time; RT: row tiles. Two workgroups a CU (4 waves a SIMD: 128 registers) but for what spills then: 13 fp32
// tokens 4099 x 1568, whose 257 workgroups would need two rounds, 11.6 us, with one 13.9.
template <int XT, int KIND, bool FEW, bool VEC, int RT>
__global__ __launch_bounds__(kThreads, XT == IDOLQ_F32 && !FEW && RT == 2 ? 2 : 4) void q4_gemv_kernel(Q4Params p) {
    constexpr bool kQ40 = KIND == IDOLQ_KIND_Q4_0;
    constexpr int kParts = XT == IDOLQ_F32 ? 3 : 1, kSize = XT == IDOLQ_F32 ? 4 : 2;
    constexpr int kRows = FEW ? 4 : 16;
    __shared__ float red[kWaves][16 * RT][kRows + 1];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * (16 * RT);
    const char* wrows[RT];  // rows past n read the last row and are not stored
#pragma unroll
    for (int j = 0; j < RT; ++j)
        wrows[j] = reinterpret_cast<const char*>(p.w) + min(row0 + 16 * j + c16, (int64_t)p.n - 1) * p.row_bytes;
    const int steps = (p.k + kStep - 1) / kStep;
    const int blocks = p.k / 32;  // groups of a row

    // This lane's A rows; rows past m read the last activation, their sums are not used. Not FEW: activation r = lane % 16,
    // depths 8 g4 .. of each group. FEW: A row r is activation r % 4 of group r / 4 of the half, with depths only where that
    // group's codes are in this lane's place g4: operand t's where r / 4 == bank(t) -- Q4_0: g4; Q4_K, whose bytes hold
    // group 2 (g4 / 2) in the low and 2 (g4 / 2) + 1 in the high nibbles: 2 (g4 / 2) for t < 2, one more for the others --
    // and zeros elsewhere. The lanes of place g4 load each of the four operands' depths once (bank b those that kTurn[t]
    // banks of rotation bring to bank(t)), 16 bytes a lane and half.
    constexpr int kTurn[4] = {0, 1, kQ40 ? 2 : 0, 3};
    const int bank = c16 >> 2;
    const uint32_t keep[2] = {bank == (kQ40 ? g4 : g4 & 2) ? ~0u : 0u, bank == (kQ40 ? g4 : g4 | 1) ? ~0u : 0u};
    // first element in the half of this lane's loads (FEW): Q4_0 operand (g4 - bank) % 4, Q4_K by the bank's distance
    const int far = (bank - (kQ40 ? g4 : g4 & 2)) & 3;  // Q4_0: operand -far; Q4_K: 0: low 0, 3: low 1, 1: high 0, 2: high 1
    const int mine = kQ40 ? 32 * g4 + 8 * (-far & 3) : 32 * ((g4 & 2) + (far == 1 || far == 2)) + 16 * (g4 & 1) + (far >= 2 ? 8 : 0);
    const char* const xrow = static_cast<const char*>(p.x) + min(FEW ? c16 & 3 : c16, p.m - 1) * p.ldx * kSize;
    const char* const zero = reinterpret_cast<const char*>(zero_activations);
    constexpr int kLoads = FEW ? 1 : 4;  // of activations, per half

    // Steps and blocks past the end read the last ones. Codes of half h = depths 128 h .. + 127 of a step -- FEW Q4_0: this
    // lane's block 4 h + g4; FEW Q4_K: bytes 64 h + 16 g4 .. of the super-block's codes; else Q4_0: bytes 8 (g4 % 2) .. of
    // blocks 4 h + 2 (g4 / 2) and the next; Q4_K: bytes 64 h + 8 g4 .. and those 32 on.
    struct Buf {
        u32x4 code[RT][2];
        u32x4 head[RT];           // Q4_K: the super-block's scales
        uint32_t scale[RT][2];    // Q4_0: FEW: see load_block; else both blocks'
        uint32_t tail[RT][2][2];  // Q4_0, not FEW: see load_eight
        u32x4 x[2 * kLoads][XT == IDOLQ_F32 ? 2 : 1];  // activations; not FEW: of the operands 4 h + t
    };
    // Blocks begin at even addresses, codes two bytes on; wide loads are taken dword-aligned and shifted in place later
    // (one token through 16384 x 8192 with 2-byte aligned 16-byte loads 34 us, with these 27).
    // A block at a multiple of 4: its first 16 bytes, and the last two in `rest`; else its codes, and the scale in `rest`.
    auto load_block = [&](const char* at, uint32_t& rest) __attribute__((always_inline)) {
        const bool even = (reinterpret_cast<uintptr_t>(at) & 2) == 0;
        rest = half_word(at + (even ? 16 : 0));
        return *reinterpret_cast<const u32x4a*>(at + (even ? 0 : 2));
    };
    auto block_codes = [&](const u32x4& c, uint32_t rest, bool even, uint32_t& scale) __attribute__((always_inline)) {
        scale = even ? c[0] & 0xffff : rest;
        const int by = even ? 2 : 0;
        return u32x4{__builtin_amdgcn_alignbyte(c[1], c[0], by), __builtin_amdgcn_alignbyte(c[2], c[1], by),
                     __builtin_amdgcn_alignbyte(c[3], c[2], by), __builtin_amdgcn_alignbyte(rest, c[3], by)};
    };
    // Eight bytes at an even address: from the dword below on, with the last two in `tail`.
    auto load_eight = [&](const char* at, uint32_t& tail) __attribute__((always_inline)) {
        tail = half_word(at + 6);
        return *reinterpret_cast<const u32x2a*>(at - (reinterpret_cast<uintptr_t>(at) & 2));
    };
    auto eight_codes = [&](uint32_t c0, uint32_t c1, uint32_t tail, const char* at) __attribute__((always_inline)) {
        const int by = (int)(reinterpret_cast<uintptr_t>(at) & 2);
        return u32x2{__builtin_amdgcn_alignbyte(c1, c0, by), __builtin_amdgcn_alignbyte(tail, c1, by)};
    };
    auto load_x = [&](const char* at, u32x4 (&x)[XT == IDOLQ_F32 ? 2 : 1]) __attribute__((always_inline)) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (XT == IDOLQ_F32 ? 2 : 1); ++i) x[i] = *reinterpret_cast<const u32x4*>(at + 16 * i);
        } else if constexpr (XT == IDOLQ_F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e / 4][e % 4] = *reinterpret_cast<const uint32_t*>(at + 4 * e);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[0][e] = half_word(at + 4 * e) | half_word(at + 4 * e + 2) << 16;
        }
    };
    auto load = [&](int s, Buf& b) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int t = 0; t < kLoads; ++t) {
                const int first = 128 * h + (FEW ? mine : 32 * t + 8 * g4);
                const bool live = !kQ40 || 8 * s + (first >> 5) < blocks;
                load_x(live ? xrow + ((int64_t)s * kStep + first) * kSize : zero, b.x[kLoads * h + t]);
            }
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                if constexpr (kQ40 && FEW) {
                    b.code[j][h] = load_block(wrows[j] + 18 * min(8 * s + 4 * h + g4, blocks - 1), b.scale[j][h]);
                } else if constexpr (kQ40) {
                    const int block = 8 * s + 4 * h + 2 * (g4 >> 1);
                    const char* a0 = wrows[j] + 18 * min(block, blocks - 1);
                    const char* a1 = wrows[j] + 18 * min(block + 1, blocks - 1);
                    b.scale[j][h] = half_word(a0) | half_word(a1) << 16;
                    const u32x2 c0 = load_eight(a0 + 2 + 8 * (g4 & 1), b.tail[j][h][0]), c1 = load_eight(a1 + 2 + 8 * (g4 & 1), b.tail[j][h][1]);
                    b.code[j][h] = u32x4{c0[0], c0[1], c1[0], c1[1]};
                } else if constexpr (FEW) {
                    b.code[j][h] = *reinterpret_cast<const u32x4*>(wrows[j] + 144 * s + 16 + 64 * h + 16 * g4);
                } else {
                    const u32x2 c0 = *reinterpret_cast<const u32x2*>(wrows[j] + 144 * s + 16 + 64 * h + 8 * g4);
                    const u32x2 c1 = *reinterpret_cast<const u32x2*>(wrows[j] + 144 * s + 48 + 64 * h + 8 * g4);
                    b.code[j][h] = u32x4{c0[0], c0[1], c1[0], c1[1]};
                }
            }
        }
        if constexpr (!kQ40) {
#pragma unroll
            for (int j = 0; j < RT; ++j) b.head[j] = *reinterpret_cast<const u32x4*>(wrows[j] + 144 * s);
        }
    };

    Buf buf;
    if (wave < steps) load(wave, buf);
    // What the epilogue adds to this thread's first output, on its way already.
    auto added = [&](int o) __attribute__((always_inline)) {
        const int a = o / (16 * RT);
        const int64_t col = row0 + o % (16 * RT);
        float2 f = make_float2(0.0f, 0.0f);
        if (a < p.m && col < p.n) {
            if (p.bias) f.x = load_as_float(p.bias, p.bias_dt, col);
            if (p.res) f.y = load_as_float(p.res, p.res_dt, a * p.ldr + col);
        }
        return f;
    };
    const float2 first_added = added(tid);

    // Eight activations as operands, in the codes' order (1 and 2, 5 and 6 change places).
    auto operands = [&](const u32x4 (&x)[XT == IDOLQ_F32 ? 2 : 1], uint4 (&op)[kParts]) __attribute__((always_inline)) {
        if constexpr (XT == IDOLQ_F32) {
            constexpr int order[8] = {0, 2, 1, 3, 4, 6, 5, 7};
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_bit_cast(float, (uint32_t)x[order[e] / 4][order[e] % 4]);
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const f32x2 f = {v[e], v[e + 1]};
                    o[e / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
                    v[e] -= __builtin_bit_cast(float, o[e / 2] << 16);
                    v[e + 1] -= __builtin_bit_cast(float, o[e / 2] & 0xffff0000u);
                }
                op[part] = make_uint4(o[0], o[1], o[2], o[3]);
            }
        } else {
            auto low = [](uint32_t a, uint32_t b) __attribute__((always_inline)) { return __builtin_amdgcn_perm(b, a, 0x05040100); };
            auto high = [](uint32_t a, uint32_t b) __attribute__((always_inline)) { return __builtin_amdgcn_perm(b, a, 0x07060302); };
            op[0] = make_uint4(low(x[0][0], x[0][1]), high(x[0][0], x[0][1]), low(x[0][2], x[0][3]), high(x[0][2], x[0][3]));
        }
    };

    // FEW: group g4 of the half, activation e in element e. Else activation 4 g4 + e.
    f32x4 acc[RT] = {};
    constexpr uint32_t kMinus = kQ40 ? Operand<XT>::kMinus24 : Operand<XT>::kMinus16;
    const uint4 minus = make_uint4(kMinus, kMinus, kMinus, kMinus);
    // scale and minimum (times the -16 of the sums) of group 4 h + g of a Q4_K super-block
    auto scales = [&](const u32x4& head, int h, int g, float& scale, float& minimum) __attribute__((always_inline)) {
        const uint32_t a = head[1] >> (8 * g), m = head[2] >> (8 * g), c = head[3] >> (8 * g);
        const uint32_t sc = h == 0 ? a & 63 : (c & 15) | ((a >> 2) & 48);
        const uint32_t mn = h == 0 ? m & 63 : ((c >> 4) & 15) | ((m >> 2) & 48);
        scale = half_bits_to_float((uint16_t)head[0]) * (float)sc;
        minimum = half_bits_to_float((uint16_t)(head[0] >> 16)) * (float)mn * 0.0625f;
    };
    // dot: x by the codes' operands, sum: x by the constant
    auto fold = [&](f32x4& acc, float scale, float minimum, const f32x4& dot, const f32x4& sum) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc[e] = fmaf(scale, dot[e] + sum[e], acc[e]);
            if (!kQ40) acc[e] = fmaf(minimum, sum[e], acc[e]);
        }
    };
    auto multiply = [&](int s, const Buf& buf) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint4 op[RT][4];
            float scale[RT][4], minimum[RT][4] = {};
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                u32x4 w = buf.code[j][h];
                if constexpr (FEW) {
                    if constexpr (kQ40) {
                        uint32_t d;
                        const int block = 8 * s + 4 * h + g4;
                        w = block_codes(w, buf.scale[j][h],
                                        (reinterpret_cast<uintptr_t>(wrows[j] + 18 * min(block, blocks - 1)) & 2) == 0, d);
                        scale[j][0] = block < blocks ? half_bits_to_float((uint16_t)d) : 0.0f;
                    } else {
                        scales(buf.head[j], h, g4, scale[j][0], minimum[j][0]);
                    }
                    op[j][0] = codes_of<XT, false>(w[0], w[1]), op[j][1] = codes_of<XT, false>(w[2], w[3]);
                    op[j][2] = codes_of<XT, true>(w[0], w[1]), op[j][3] = codes_of<XT, true>(w[2], w[3]);
                } else if constexpr (kQ40) {
                    const int block = 8 * s + 4 * h + 2 * (g4 >> 1);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const u32x2 e = eight_codes(w[2 * i], w[2 * i + 1], buf.tail[j][h][i],
                                                    wrows[j] + 18 * min(block + i, blocks - 1) + 2);
                        w[2 * i] = e[0], w[2 * i + 1] = e[1];
                    }
                    uint32_t c[2][4], d[2];  // of the two blocks of each lane half
#pragma unroll
                    for (int e = 0; e < 4; ++e) both_halves(w[e], c[0][e], c[1][e]);
                    both_halves(buf.scale[j][h], d[0], d[1]);
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const int shift = 4 * (g4 >> 1);
                        op[j][t] = codes_of<XT, false>(c[t >> 1][2 * (t & 1)] >> shift, c[t >> 1][2 * (t & 1) + 1] >> shift);
                        scale[j][t] = 8 * s + 4 * h + t < blocks ? half_bits_to_float((uint16_t)(d[t >> 1] >> (16 * (t & 1)))) : 0.0f;
                    }
                } else {
                    op[j][0] = codes_of<XT, false>(w[0], w[1]), op[j][1] = codes_of<XT, true>(w[0], w[1]);
                    op[j][2] = codes_of<XT, false>(w[2], w[3]), op[j][3] = codes_of<XT, true>(w[2], w[3]);
#pragma unroll
                    for (int t = 0; t < 4; ++t) scales(buf.head[j], h, t, scale[j][t], minimum[j][t]);
                }
            }
            f32x4 dot[RT] = {}, sum = {0.0f, 0.0f, 0.0f, 0.0f};
            uint4 a[kParts];
            if (FEW) operands(buf.x[h], a);
            static_for<4>([&](auto t_tag) __attribute__((always_inline)) {
                constexpr int t = decltype(t_tag)::value;
                if constexpr (!FEW) {
                    sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 0; j < RT; ++j) dot[j] = sum;
                    operands(buf.x[4 * h + t], a);
                }
#pragma unroll
                for (int part = 0; part < kParts; ++part) {
                    uint4 x = a[part];
                    if constexpr (FEW) {
                        const uint32_t mask = keep[t >> 1];
                        x = make_uint4(turned<kTurn[t]>(x.x) & mask, turned<kTurn[t]>(x.y) & mask, turned<kTurn[t]>(x.z) & mask,
                                       turned<kTurn[t]>(x.w) & mask);
                    }
#pragma unroll
                    for (int j = 0; j < RT; ++j) dot[j] = Operand<XT>::run(x, op[j][t], dot[j]);
                    sum = Operand<XT>::run(x, minus, sum);
                }
                if constexpr (!FEW)
#pragma unroll
                    for (int j = 0; j < RT; ++j) fold(acc[j], scale[j][t], minimum[j][t], dot[j], sum);
            });
            if constexpr (FEW)
#pragma unroll
                for (int j = 0; j < RT; ++j) fold(acc[j], scale[j][0], minimum[j][0], dot[j], sum);
        }
    };

    // The loop's loads are unconditional, so that its waits count them.
    int s = wave;
    for (; s + kWaves < steps; s += kWaves) {
        multiply(s, buf);
        load(s + kWaves, buf);
    }
    if (s < steps) multiply(s, buf);

    // FEW: a weight row's sums over the lanes' groups. Then over the waves in order.
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float v = acc[j][e];
            if constexpr (FEW) {
                v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
                if (g4 == 0) red[wave][16 * j + c16][e] = v;
            } else {
                red[wave][16 * j + c16][4 * g4 + e] = v;
            }
        }
    __syncthreads();
    const bool round_first = (p.flags & IDOLQ_FLAG_ROUND_BEFORE_BIAS) != 0;
    for (int o = tid; o < 16 * RT * p.m; o += kThreads) {
        const int a = o / (16 * RT), r = o % (16 * RT);
        const int64_t col = row0 + r;
        if (col >= p.n) continue;
        const float2 add = o == tid ? first_added : added(o);
        float v = red[0][r][a];
        for (int t = 1; t < kWaves; ++t) v += red[t][r][a];
        if (round_first) v = round_through(p.y_dt, v);
        if (p.bias) v += add.x;
        if (p.res) v += add.y;
        store_from_float(p.y, p.y_dt, a * p.ldy + col, apply_act(p.act, v));
    }
}

// Row tiles of a workgroup: two, which share the activations' loads and operands, where that leaves two workgroups a CU;
// else one, as the depth has to fill the card. 16384 x 8192 with two and one: Q4_K, one fp32 token 29 and 36 us, 16 bf16
// tokens 40 and 51, 4 fp16 tokens 25.9 and 27.3; Q4_0, 4 bf16 tokens 11008 x 4096 14.7 and 12.6, one token 4096 x 4096 8.2
// and 6.4.
int row_tiles_for(const Q4Params& p) { return p.n >= 1024 * 16 ? 2 : 1; }

template <int XT, int KIND, bool FEW, int RT>
int launch_tiles(const Q4Params& p, hipStream_t s) {
    const dim3 grid((unsigned)(((int64_t)p.n + 16 * RT - 1) / (16 * RT))), block(kThreads);
    if (vec8_ok(p.x, XT, p.m > 1 ? p.ldx : 8))
        hipLaunchKernelGGL((q4_gemv_kernel<XT, KIND, FEW, true, RT>), grid, block, 0, s, p);
    else
        hipLaunchKernelGGL((q4_gemv_kernel<XT, KIND, FEW, false, RT>), grid, block, 0, s, p);
    return check_launch("q4_gemv_kernel");
}
template <int XT, int KIND, bool FEW>
int launch(const Q4Params& p, hipStream_t s) {
    return row_tiles_for(p) == 2 ? launch_tiles<XT, KIND, FEW, 2>(p, s) : launch_tiles<XT, KIND, FEW, 1>(p, s);
}
template <int XT, int KIND>
int by_rows(const Q4Params& p, hipStream_t s) {
    return p.m <= 4 ? launch<XT, KIND, true>(p, s) : launch<XT, KIND, false>(p, s);
}
template <int KIND>
int by_type(const Q4Params& p, int x_dt, hipStream_t s) {
    return x_dt == IDOLQ_BF16  ? by_rows<IDOLQ_BF16, KIND>(p, s)
           : x_dt == IDOLQ_F16 ? by_rows<IDOLQ_F16, KIND>(p, s)
                               : by_rows<IDOLQ_F32, KIND>(p, s);
}

}  // namespace
}  // namespace idolq

using namespace idolq;

extern "C" int idolq_q4_gemv(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* w, int kind,
                             int64_t n_total, int64_t n_offset, int64_t n, const void* bias, int bias_dtype,
                             const void* residual, int residual_dtype, int64_t ldr, int act, int flags, void* y,
                             int y_dtype, int64_t ldy, void* stream) {
    if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype) || (bias && !dtype_ok(bias_dtype)) || (residual && !dtype_ok(residual_dtype)))
        return fail(IDOLQ_EINVAL, "unknown dtype code");
    if (kind != IDOLQ_KIND_Q4_0 && kind != IDOLQ_KIND_Q4_K)
        return fail(IDOLQ_EINVAL, "4-bit products take Q4_0 or Q4_K blocks");
    const int64_t values = kind == IDOLQ_KIND_Q4_0 ? 32 : 256, bytes = kind == IDOLQ_KIND_Q4_0 ? 18 : 144;
    if (m < 0 || m > kMaxM) return fail(IDOLQ_EINVAL, "4-bit products take up to 16 activation rows");
    if (k <= 0 || k % values != 0 || k > (1 << 24))
        return fail(IDOLQ_EINVAL, kind == IDOLQ_KIND_Q4_0 ? "k must be a multiple of 32, up to 2^24"
                                                          : "k must be a multiple of 256, up to 2^24");
    if (n_total < 0 || n < 0 || n_offset < 0 || n > n_total - n_offset)
        return fail(IDOLQ_EINVAL, "weight window outside the matrix");
    if (n > (1 << 27)) return fail(IDOLQ_EINVAL, "4-bit products take up to 2^27 weight rows");
    if (ldx < k || ldy < n || (residual && ldr < n)) return fail(IDOLQ_EINVAL, "row stride too small");
    if (act < IDOLQ_ACT_NONE || act > IDOLQ_ACT_SILU) return fail(IDOLQ_EINVAL, "unknown activation");
    if ((flags & ~IDOLQ_FLAG_ROUND_BEFORE_BIAS) != 0) return fail(IDOLQ_EINVAL, "unknown flag for 4-bit products");
    if (m == 0 || n == 0) return IDOLQ_OK;
    if (!x || !w || !y) return fail(IDOLQ_EINVAL, "x, w and y must be non-null");
    const int64_t row_bytes = k / values * bytes;
    Q4Params p{};
    p.x = x, p.w = w + n_offset * row_bytes, p.res = residual, p.y = y;
    p.ldx = ldx, p.row_bytes = row_bytes, p.ldr = ldr, p.ldy = ldy;
    p.m = (int)m, p.k = (int)k, p.n = (int)n;
    p.bias_dt = bias_dtype, p.res_dt = residual_dtype, p.y_dt = y_dtype, p.act = act, p.flags = flags;
    if (bias) p.bias = static_cast<const char*>(bias) + n_offset * (int64_t)dtype_size(bias_dtype);
    if (reinterpret_cast<uintptr_t>(p.w) % (kind == IDOLQ_KIND_Q4_0 ? 2 : 16) != 0)
        return fail(IDOLQ_EINVAL, "Q4_0 blocks must be 2-byte aligned, Q4_K blocks 16-byte aligned");
    // y is written while others still read x; a residual's element is read by the thread that writes y's in its place
    const int64_t xs = (int64_t)dtype_size(x_dtype), ys = (int64_t)dtype_size(y_dtype);
    const RowBlock to{y, m, ldy * ys, n * ys};
    if (rows_overlap(to, {x, m, ldx * xs, k * xs})) return fail(IDOLQ_EINVAL, "y must not overlap x");
    if (residual && !(residual == y && residual_dtype == y_dtype && (ldr == ldy || m == 1))) {
        const int64_t rs = (int64_t)dtype_size(residual_dtype);
        if (rows_overlap(to, {residual, m, ldr * rs, n * rs})) return fail(IDOLQ_EINVAL, "y must not overlap the residual, unless it is y");
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    return kind == IDOLQ_KIND_Q4_0 ? by_type<IDOLQ_KIND_Q4_0>(p, x_dtype, s) : by_type<IDOLQ_KIND_Q4_K>(p, x_dtype, s);
}
