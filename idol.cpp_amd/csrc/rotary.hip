// Rotary positions with several axes for gfx950.
//
// A head's first 2 P elements are P pairs; pair j of a row at positions pos[0 .. axes) is turned by the angle
// t = pos[axis(j)] freqs[j]: (a, b) -> (a cos t - b sin t, b cos t + a sin t), with sin negated for the inverse (which
// is the gradient too). The first sections[0] pairs go by axis 0, the next sections[1] by axis 1, and so on. A pair is
// elements (j, j + P), or (2 j, 2 j + 1) interleaved; elements from 2 P on are copied.
//
// t / 2 pi is formed and reduced to half a turn in fp64 (position and frequency are exact there; fp32 would leave 1e-3 of
// a radian at position 1e5), sine and cosine are then taken in fp32.
//
// The bytes bound it (every element read and written once), so a thread keeps the sines and cosines of one unit of a row
// (V neighbouring pairs, the widest access up to 16 bytes that all strides, addresses and sections allow) in registers
// and walks the heads with it, kBatch heads' loads in flight at a time.
#include "common.h"

#include <algorithm>

namespace idolq {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kThreads = 256;
constexpr int kBatch = 4;

struct RotaryParams {
    const void* x[2];
    void* y[2];
    int64_t ldx[2], ldy[2];
    int heads[2];
    const void* pos;
    int64_t ldp;
    const float* freqs;
    int64_t rows;
    int pos_kind, head_dim, pairs, inverse;
    int units, unit_copies;  // per head: units of V pairs, then units copied
    int lanes;               // threads that share a row's heads
    int past;                // more is written than the L2s hold: stores go past them
    int first[kMaxAxes];     // the first pair of each axis (`pairs` for an axis that has none)
};

template <int BYTES>
struct Raw;
template <>
struct Raw<16> { typedef uint4 type; };
template <>
struct Raw<8> { typedef uint2 type; };
template <>
struct Raw<4> { typedef uint32_t type; };

template <int DT>
__device__ __forceinline__ float widen(const char* p) {
    if (DT == IDOLQ_F32) return *reinterpret_cast<const float*>(p);
    const uint16_t b = *reinterpret_cast<const uint16_t*>(p);
    return DT == IDOLQ_BF16 ? bf16_bits_to_float(b) : half_bits_to_float(b);
}
template <int DT>
__device__ __forceinline__ void narrow(char* p, float v) {
    if (DT == IDOLQ_F32)
        *reinterpret_cast<float*>(p) = v;
    else
        *reinterpret_cast<uint16_t*>(p) = DT == IDOLQ_BF16 ? float_to_bf16_bits(v) : float_to_half_bits(v);
}

// One access: N elements of DT in one load or store, or (SINGLE) the first n of them one by one.
template <int DT, int N, bool SINGLE>
struct Piece {
    static constexpr int kSize = DT == IDOLQ_F32 ? 4 : 2;
    alignas(16) char v[N * kSize];
    __device__ __forceinline__ void load(const char* p, int n) {
        if constexpr (SINGLE) {
#pragma unroll
            for (int i = 0; i < N; ++i) set(i, i < n ? widen<DT>(p + i * kSize) : 0.0f);
        } else {
            typedef typename Raw<N * kSize>::type raw;
            *reinterpret_cast<raw*>(v) = *reinterpret_cast<const raw*>(p);
        }
    }
    __device__ __forceinline__ void store(char* p, int n, bool past) const {
        if constexpr (SINGLE) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < n) narrow<DT>(p + i * kSize, get(i));
        } else {
            typedef uint32_t raw __attribute__((ext_vector_type(N * kSize / 4)));
            if (past)
                __builtin_nontemporal_store(*reinterpret_cast<const raw*>(v), reinterpret_cast<raw*>(p));
            else
                *reinterpret_cast<raw*>(p) = *reinterpret_cast<const raw*>(v);
        }
    }
    __device__ __forceinline__ float get(int i) const { return widen<DT>(v + i * kSize); }
    __device__ __forceinline__ void set(int i, float f) { narrow<DT>(v + i * kSize, f); }
};

// V pairs per unit: two accesses of V elements (halves), or one of 2 V (INTER).
template <int DT, int V, bool INTER>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryParams p) {
    constexpr int kSize = DT == IDOLQ_F32 ? 4 : 2;
    constexpr int N = INTER ? 2 * V : V;
    const int units = p.units + p.unit_copies;  // at most kThreads: head_dim is
    const int t = threadIdx.x, unit = t % units, lane = (t / units) % p.lanes, sub = t / (units * p.lanes);
    const int rows_per = kThreads / (units * p.lanes);
    const int64_t row = (int64_t)blockIdx.x * rows_per + sub;
    if (sub >= rows_per || row >= p.rows) return;
    const int all = p.heads[0] + p.heads[1];
    const bool copy = unit >= p.units;
    const int j0 = unit * V;  // the unit's first pair
    float cs[V], sn[V];
    if (!copy) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int j = j0 + i;
            int axis = 0;
#pragma unroll
            for (int a = 1; a < kMaxAxes; ++a) axis += j >= p.first[a];
            const int64_t at = row * p.ldp + axis;
            const double pos = p.pos_kind == IDOLQ_POS_F32   ? (double)static_cast<const float*>(p.pos)[at]
                               : p.pos_kind == IDOLQ_POS_I32 ? (double)static_cast<const int32_t*>(p.pos)[at]
                                                             : (double)static_cast<const int64_t*>(p.pos)[at];
            const double turns = pos * (double)p.freqs[j] * 0.15915494309189535;
            sincospif(2.0f * (float)(turns - rint(turns)), &sn[i], &cs[i]);
            if (p.inverse) sn[i] = -sn[i];
        }
    }
    // bytes of the unit's first access inside a head; the second one of halves lies `pairs` elements on
    const int ia = (copy ? 2 * p.pairs + (unit - p.units) * N : INTER ? 2 * j0 : j0) * kSize, gap = p.pairs * kSize;
    const char* const xr[2] = {static_cast<const char*>(p.x[0]) + row * p.ldx[0] * kSize + ia,
                               static_cast<const char*>(p.x[1]) + row * p.ldx[1] * kSize + ia};
    char* const yr[2] = {static_cast<char*>(p.y[0]) + row * p.ldy[0] * kSize + ia,
                         static_cast<char*>(p.y[1]) + row * p.ldy[1] * kSize + ia};
    const int head_bytes = p.head_dim * kSize;
    const int n = copy ? min(N, p.head_dim - ia / kSize) : N;  // elements of the unit (the last copied one may be short)
    for (int h0 = lane; h0 < all; h0 += kBatch * p.lanes) {
        Piece<DT, N, V == 1> a[kBatch], b[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int h = h0 + e * p.lanes, which = h < p.heads[0] ? 0 : 1;
            if (h >= all) break;
            const char* x = xr[which] + (int64_t)(h - (which ? p.heads[0] : 0)) * head_bytes;
            a[e].load(x, n);
            if (!INTER && !copy) b[e].load(x + gap, n);
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int h = h0 + e * p.lanes, which = h < p.heads[0] ? 0 : 1;
            if (h >= all) break;
            char* y = yr[which] + (int64_t)(h - (which ? p.heads[0] : 0)) * head_bytes;
            if (!copy) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float u = INTER ? a[e].get(2 * i) : a[e].get(i), w = INTER ? a[e].get(2 * i + 1) : b[e].get(i);
                    const float c = u * cs[i] - w * sn[i], d = w * cs[i] + u * sn[i];
                    if (INTER) {
                        a[e].set(2 * i, c);
                        a[e].set(2 * i + 1, d);
                    } else {
                        a[e].set(i, c);
                        b[e].set(i, d);
                    }
                }
                if (!INTER) b[e].store(y + gap, n, p.past);
            }
            a[e].store(y, n, p.past);
        }
    }
}

template <int DT, int V, bool INTER>
int launch(RotaryParams p, hipStream_t s) {
    constexpr int N = INTER ? 2 * V : V;
    p.units = p.pairs / V;
    p.unit_copies = (p.head_dim - 2 * p.pairs + N - 1) / N;
    const int units = p.units + p.unit_copies, all = p.heads[0] + p.heads[1];
    // Threads sharing a row's heads: the more, the wider the memory runs and the more of the chip a few rows fill; the
    // fewer, the more heads a sine serves. 12 unless that leaves fewer than 2^18 threads (32760 rows, 24 + 24 heads of 64 in
    // bf16: 86 us with 12, 92 with 8, 96 with 24). Outputs larger than the L2s (32 MB) are stored past them (100 us else
    // with 8).
    const int64_t fill = ((int64_t)1 << 18) / (p.rows * units) + 1;
    p.lanes = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(all, kThreads / units), std::max<int64_t>(12, fill)));
    p.past = p.rows * all * p.head_dim * (DT == IDOLQ_F32 ? 4 : 2) > ((int64_t)32 << 20);
    const int rows_per = kThreads / (units * p.lanes);
    const int64_t grid = (p.rows + rows_per - 1) / rows_per;
    if (grid >= (1 << 24)) return fail(IDOLQ_EINVAL, "too many rotary rows");
    hipLaunchKernelGGL((rotary_kernel<DT, V, INTER>), dim3((unsigned)grid), dim3(kThreads), 0, s, p);
    return check_launch("rotary_kernel");
}

// The widest unit whose accesses are whole: `step` is what every address, stride and section is a multiple of.
template <int DT, bool INTER>
int dispatch(const RotaryParams& p, int64_t step, hipStream_t s) {
    constexpr int kMost = (DT == IDOLQ_F32 ? 4 : 8) / (INTER ? 2 : 1);  // 16 bytes an access
    const int64_t v = INTER ? step / 2 : step;
    if (v >= kMost) return launch<DT, kMost, INTER>(p, s);
    if constexpr (kMost > 4)
        if (v >= 4) return launch<DT, 4, INTER>(p, s);
    if (v >= 2) return launch<DT, 2, INTER>(p, s);
    return launch<DT, 1, INTER>(p, s);
}

}  // namespace
}  // namespace idolq

using namespace idolq;

extern "C" int idolq_rotary(const void* x, void* y, int dtype, int64_t rows, int64_t heads, int64_t ldx, int64_t ldy,
                            const void* x2, void* y2, int64_t heads2, int64_t ldx2, int64_t ldy2, int64_t head_dim,
                            const void* pos, int pos_kind, int64_t ldp, int64_t axes, const int64_t* sections,
                            const float* freqs, int flags, void* stream) {
    if (!dtype_ok(dtype)) return fail(IDOLQ_EINVAL, "unknown dtype code");
    if (pos_kind != IDOLQ_POS_I32 && pos_kind != IDOLQ_POS_I64 && pos_kind != IDOLQ_POS_F32)
        return fail(IDOLQ_EINVAL, "unknown position type");
    if ((flags & ~(IDOLQ_ROTARY_INTERLEAVED | IDOLQ_ROTARY_INVERSE)) != 0) return fail(IDOLQ_EINVAL, "unknown rotary flag");
    if (axes < 1 || axes > kMaxAxes || !sections) return fail(IDOLQ_EINVAL, "rotary positions need 1 to 4 axes");
    if (rows < 0 || heads <= 0 || heads2 < 0 || head_dim < 2 || head_dim > kThreads || heads > 65535 || heads2 > 65535)
        return fail(IDOLQ_EINVAL, "bad rotary shape (needs heads > 0 and 2 <= head_dim <= 256)");
    RotaryParams p{};
    int64_t pairs = 0;
    for (int64_t a = 0; a < axes; ++a) {
        if (sections[a] < 0 || sections[a] > head_dim) return fail(IDOLQ_EINVAL, "rotary sections must be pair counts");
        p.first[a] = (int)pairs;
        pairs += sections[a];
    }
    if (pairs < 1 || 2 * pairs > head_dim) return fail(IDOLQ_EINVAL, "rotary sections must hold 1 to head_dim / 2 pairs");
    for (int64_t a = axes; a < kMaxAxes; ++a) p.first[a] = (int)pairs;
    if (ldx < heads * head_dim || ldy < heads * head_dim || (heads2 && (ldx2 < heads2 * head_dim || ldy2 < heads2 * head_dim)))
        return fail(IDOLQ_EINVAL, "row stride smaller than heads * head_dim");
    if (ldp < axes) return fail(IDOLQ_EINVAL, "position rows shorter than the axes");
    if (rows == 0) return IDOLQ_OK;
    if (!x || !y || !pos || !freqs || (heads2 && (!x2 || !y2)))
        return fail(IDOLQ_EINVAL, "rotary buffers must be non-null");
    const int64_t bytes = (int64_t)dtype_size(dtype), second = heads2 ? rows : 0;
    const RowBlock in[2] = {{x, rows, ldx * bytes, heads * head_dim * bytes}, {x2, second, ldx2 * bytes, heads2 * head_dim * bytes}};
    const RowBlock to[2] = {{y, rows, ldy * bytes, heads * head_dim * bytes}, {y2, second, ldy2 * bytes, heads2 * head_dim * bytes}};
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2; ++j) {
            const bool in_place = i == j && to[i].p == in[j].p && (to[i].ld == in[j].ld || rows == 1);
            if (!in_place && rows_overlap(to[i], in[j]))
                return fail(IDOLQ_EINVAL, "rotary outputs must not overlap inputs, but for each its own in place");
        }
    if (rows_overlap(to[0], to[1])) return fail(IDOLQ_EINVAL, "rotary outputs must not overlap");
    p.x[0] = x, p.x[1] = x2, p.y[0] = y, p.y[1] = y2;
    p.ldx[0] = ldx, p.ldx[1] = ldx2, p.ldy[0] = ldy, p.ldy[1] = ldy2;
    p.heads[0] = (int)heads, p.heads[1] = (int)heads2;
    p.pos = pos, p.ldp = ldp, p.freqs = freqs, p.rows = rows;
    p.pos_kind = pos_kind, p.head_dim = (int)head_dim, p.pairs = (int)pairs;
    p.inverse = (flags & IDOLQ_ROTARY_INVERSE) != 0;
    const bool inter = (flags & IDOLQ_ROTARY_INTERLEAVED) != 0;
    // the largest power of two of elements (up to 8) that divides every stride, address, the pairs and what is copied
    int64_t bits = (inter ? 2 * pairs : pairs) | head_dim | (head_dim - 2 * pairs) | ldx | ldy | 8;
    bits |= (int64_t)(reinterpret_cast<uintptr_t>(x) / bytes) | (int64_t)(reinterpret_cast<uintptr_t>(y) / bytes);
    if (heads2)
        bits |= ldx2 | ldy2 | (int64_t)(reinterpret_cast<uintptr_t>(x2) / bytes) | (int64_t)(reinterpret_cast<uintptr_t>(y2) / bytes);
    const int64_t step = bits & -bits;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == IDOLQ_F32) return inter ? dispatch<IDOLQ_F32, true>(p, step, s) : dispatch<IDOLQ_F32, false>(p, step, s);
    if (dtype == IDOLQ_F16) return inter ? dispatch<IDOLQ_F16, true>(p, step, s) : dispatch<IDOLQ_F16, false>(p, step, s);
    return inter ? dispatch<IDOLQ_BF16, true>(p, step, s) : dispatch<IDOLQ_BF16, false>(p, step, s);
}
