// Normalisation of rows together with the residual's addition, forward and backward, and the 8-bit form of rows.
//
//   POST   y = s + g n(x)            PRE   h = s + g x,  y = n(h)
//   n(v) = (v - m) r w + b,   m = mean(v) (0 for RMS),  r = 1 / sqrt(mean((v - m)^2) + eps)
//
// Backward, with v^ = (v - m) r, dn the gradient that reaches n (POST: g dy, PRE: dy) and t = dn w:
//
//   dv = r (t - mean(t) - v^ mean(t v^))       (RMS: without mean(t))
//   dw = sum over rows of dn v^,   db = sum over rows of dn
//   POST: dx = dv                   PRE: ds = dh + dv, dx = g ds
//
// All of it is bound by memory: forward reads x and s and writes y, backward reads dy and x (h) and writes dx, and
// nothing in between leaves the registers.  A row belongs to LPR lanes with CPL 16-byte chunks of 8 elements each (chunk
// c of lane l starts at element 8 (c LPR + l), so that neighbouring lanes read neighbouring chunks); several short rows
// share a wavefront, a row of more than 2048 elements belongs to a workgroup.  The sums over a row stay in the lanes
// (DPP and permlane exchanges) for all but the workgroup rows.  The mean comes first and the squared deviations are
// summed around it (two passes over registers): E[v^2] - m^2 would lose the variance of rows with a large mean.
//
// A workgroup walks over rows with a stride of the grid and asks for its next row before it works on the present one.
// Its lanes keep their columns, so weight and bias are read once and the column sums dw, db stay in registers until the
// end; one partial row per workgroup then goes to the workspace and a second kernel adds those in a fixed order.
//
// Measured on MI355X, where a large copy moves 5.1 TB/s: 262144 x 96 bf16 forward 36 us (4.3 TB/s), backward 37 us
// (4.0 TB/s) and 5 us for the parameters' sums; 16384 x 1536 pre-norm with h in fp32 and 8-bit rows 49 us (5.7 TB/s);
// 8-bit form of 8192 x 4096 bf16 16 us (6.3 TB/s, part of x still in the caches).  One row: 3 us, the launch itself.
// 4099 x 385 fp16, pre-norm: forward 7 us; backward 14 us, one workgroup to a CU and four to five rounds of loads one after
// the other (1.1 TB/s), and 4 us for the parameters' sums.
#include <type_traits>

#include "fwa2_common.hpp"

namespace fwa2 {

struct NormArgs {
    const void *x, *s, *weight, *bias, *gate;
    int64_t xs, ss;                 // row strides, elements
    void *y, *h;                    // contiguous
    uint8_t* y8;
    float* y8_scale;
    float2* stats;
    const void *dy, *dh;
    int64_t dys, dhs;
    void *dx, *ds;
    float* part;                    // [workgroups][2][dim]
    int64_t rows;
    uint32_t rows_per_gate, gates;
    int dim;
    float eps;
    int layer, pre, param_f32, gate_f32, want_params;
};

template <class T> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8 V; };
template <> struct Vec8<_Float16> { typedef f16x8 V; };
template <> struct Vec8<float> { typedef float V __attribute__((ext_vector_type(8))); };

// 8 elements from column c0 on, zeros beyond the row's end.  VEC: rows start on 16-byte boundaries and dim is a multiple
// of 8.  Otherwise a whole chunk is still one access of whatever alignment the row has, and only the chunk that
// crosses the row's end goes element by element, from clamped places: eight loads under way at once, where a test per
// element would wait for each.
template <bool VEC, class T>
__device__ __forceinline__ typename Vec8<T>::V row_load8(const T* row, int c0, int dim) {
    typename Vec8<T>::V v;
    if (VEC) {
        if (c0 < dim) v = *reinterpret_cast<const typename Vec8<T>::V*>(row + c0);
        else v = (T)0.f;
    } else if (c0 + 8 <= dim) {
        __builtin_memcpy(&v, row + c0, sizeof(v));
    } else {
        T e[8];
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = row[min(c0 + j, dim - 1)];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = c0 + j < dim ? e[j] : (T)0.f;
    }
    return v;
}
template <bool VEC, class T>
__device__ __forceinline__ void row_store8(T* row, int c0, int dim, const float* x) {
    typename Vec8<T>::V v;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = (T)x[j];
    if (VEC) {
        if (c0 < dim) *reinterpret_cast<typename Vec8<T>::V*>(row + c0) = v;
    } else if (c0 + 8 <= dim) {
        __builtin_memcpy(row + c0, &v, sizeof(v));
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c0 + j < dim) row[c0 + j] = v[j];
    }
}
// weight, bias: element type decided at run time, read once per workgroup; zeros beyond the last column.  Loads from clamped
// places and selects, no branch per value: a branch would wait for each load before the next one is asked for.
template <bool VEC, class T>
__device__ __forceinline__ void param_read8(const T* p, int c0, int dim, float* x) {
    if (VEC) {
        const typename Vec8<T>::V v = *reinterpret_cast<const typename Vec8<T>::V*>(p + min(c0, dim - 8));
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = c0 < dim ? (float)v[j] : 0.f;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float v = (float)p[min(c0 + j, dim - 1)];
            x[j] = c0 + j < dim ? v : 0.f;
        }
    }
}
template <bool VEC, class XT>
__device__ __forceinline__ void param_load8(const void* p, bool f32, int c0, int dim, float* x) {
    if (f32) param_read8<VEC>(reinterpret_cast<const float*>(p), c0, dim, x);
    else param_read8<VEC>(reinterpret_cast<const XT*>(p), c0, dim, x);
}
// The gate of the rows a lane walks over: its index moves by whole samples and a remainder from row to row (a division per
// row would cost more than the row's statistics).
template <class XT>
struct GateWalk {
    uint32_t at, left, skip, more;      // sample, rows into it; what a step adds to both
    __device__ __forceinline__ void init(const NormArgs& a, int64_t row, int64_t step) {
        at = left = skip = more = 0;
        if (a.gate == nullptr) return;
        at = (uint32_t)row / a.rows_per_gate;
        left = (uint32_t)row - at * a.rows_per_gate;
        skip = (uint32_t)step / a.rows_per_gate;
        more = (uint32_t)step - skip * a.rows_per_gate;
    }
    // (rows beyond the last: the last sample's gate)
    __device__ __forceinline__ float get(const NormArgs& a) const {
        if (a.gate == nullptr) return 1.f;
        const uint32_t i = at < a.gates ? at : a.gates - 1;
        return a.gate_f32 ? reinterpret_cast<const float*>(a.gate)[i] : (float)reinterpret_cast<const XT*>(a.gate)[i];
    }
    __device__ __forceinline__ void next(const NormArgs& a) {
        at += skip;
        left += more;
        if (left >= a.rows_per_gate) {
            left -= a.rows_per_gate;
            at++;
        }
    }
};

// ---- sums and maxima over the LPR lanes of a row -----------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) { return __builtin_amdgcn_update_dpp(0u, x, CTRL, 0xF, 0xF, true); }
struct AddF {
    static __device__ __forceinline__ uint32_t of(uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }
};
struct MaxU {       // of non-negative floats by their bits: a NaN wins over everything
    static __device__ __forceinline__ uint32_t of(uint32_t a, uint32_t b) { return a > b ? a : b; }
};
// Every lane of the group gets the result.  Within 16 lanes: quad swaps, then mirrors of 8 and of 16 lanes (after the
// quads agree, a mirrored lane holds the other half's value); above that the permlane swaps.
template <class OP, int LANES>
__device__ __forceinline__ uint32_t lanes_reduce(uint32_t x) {
    if (LANES >= 2) x = OP::of(x, dpp<0xB1>(x));
    if (LANES >= 4) x = OP::of(x, dpp<0x4E>(x));
    if (LANES >= 8) x = OP::of(x, dpp<0x141>(x));
    if (LANES >= 16) x = OP::of(x, dpp<0x140>(x));
    if (LANES >= 32) { const u32x2 r = __builtin_amdgcn_permlane16_swap(x, x, false, false); x = OP::of(r[0], r[1]); }
    if (LANES >= 64) { const u32x2 r = __builtin_amdgcn_permlane32_swap(x, x, false, false); x = OP::of(r[0], r[1]); }
    return x;
}
// Rows of a whole workgroup: one value per wavefront through LDS.  `slot` alternates between calls: when a wavefront
// passes the barrier of a call, every wavefront has read the values of the call before it, whose half may be reused.
template <class OP, int LPR>
__device__ __forceinline__ uint32_t row_reduce(uint32_t x, uint32_t* red, int& slot) {
    x = lanes_reduce<OP, (LPR < 64 ? LPR : 64)>(x);
    if (LPR <= 64) return x;
    constexpr int W = LPR <= 64 ? 1 : LPR / 64;
    uint32_t* mine = red + slot * 16;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) mine[threadIdx.x >> 6] = x;
    __syncthreads();
    x = mine[0];
#pragma unroll
    for (int i = 1; i < W; i++) x = OP::of(x, mine[i]);
    return x;
}
template <int LPR>
__device__ __forceinline__ float row_sum(float x, uint32_t* red, int& slot) {
    return __uint_as_float(row_reduce<AddF, LPR>(__float_as_uint(x), red, slot));
}

// Scale of a row from its largest magnitude (bits).  NaN and infinity pass through (a comparison with NaN is false).
struct RowScale {
    float scale, inv;
};
__device__ __forceinline__ RowScale scale_of(uint32_t amax_bits) {
    float amax = __uint_as_float(amax_bits);
    if (amax < 0x1p-100f) amax = 0x1p-100f;
    RowScale s;
    s.scale = amax * (1.f / 448.f);
    s.inv = 1.f / s.scale;
    return s;
}
// v / scale with the rounding of a division: rows of 16-bit values have quotients that fall exactly between two 8-bit
// values, and a plain product with the reciprocal would send those to either side.  One reciprocal per row and, per
// value, the quotient's estimate corrected by its remainder.
__device__ __forceinline__ float quotient(float v, const RowScale& s) {
    const float q = v * s.inv;
    return __builtin_fmaf(__builtin_fmaf(-q, s.scale, v), s.inv, q);
}
__device__ __forceinline__ u32x2 pack_e4m3(const float* v, const RowScale& s) {
    u32x2 r;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(v[4 * i], s), quotient(v[4 * i + 1], s), 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(v[4 * i + 2], s), quotient(v[4 * i + 3], s), w, true);
        r[i] = (uint32_t)w;
    }
    return r;
}
template <bool VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* row, int c0, int dim, const float* v, const RowScale& s) {
    const u32x2 q = pack_e4m3(v, s);
    if (VEC) {
        if (c0 < dim) *reinterpret_cast<u32x2*>(row + c0) = q;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c0 + j < dim) row[c0 + j] = (uint8_t)(q[j >> 2] >> (8 * (j & 3)));
    }
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

constexpr int norm_block(int lpr) { return lpr > 256 ? lpr : 256; }

// ---- forward ------------------------------------------------------------------------------------------------
template <class XT, class ST, int LPR, int CPL, bool VEC>
__global__ void __launch_bounds__(norm_block(LPR)) norm_fwd_kernel(const NormArgs a) {
    typedef typename Vec8<XT>::V XV;
    typedef typename Vec8<ST>::V SV;
    constexpr int RPB = norm_block(LPR) / LPR;      // rows a workgroup works on at a time
    __shared__ uint32_t red[32];
    int slot = 0;
    const int l = threadIdx.x % LPR;
    const int dim = a.dim;
    const float inv_dim = 1.f / (float)dim;
    const bool layer = a.layer, pre = a.pre;

    float w[CPL][8], b[CPL][8];
#pragma unroll
    for (int c = 0; c < CPL; c++) {
        const int c0 = 8 * (c * LPR + l);
        param_load8<VEC, XT>(a.weight, a.param_f32, c0, dim, w[c]);
#pragma unroll
        for (int j = 0; j < 8; j++) b[c][j] = 0.f;
        if (a.bias) param_load8<VEC, XT>(a.bias, a.param_f32, c0, dim, b[c]);
    }

    XV xr[CPL];
    SV sr[CPL];
    auto fetch = [&](int64_t row) __attribute__((always_inline)) {
        const XT* xp = reinterpret_cast<const XT*>(a.x) + row * a.xs;
        const ST* sp = reinterpret_cast<const ST*>(a.s) + row * a.ss;
#pragma unroll
        for (int c = 0; c < CPL; c++) xr[c] = row_load8<VEC>(xp, 8 * (c * LPR + l), dim);
        if (a.s != nullptr) {
#pragma unroll
            for (int c = 0; c < CPL; c++) sr[c] = row_load8<VEC>(sp, 8 * (c * LPR + l), dim);
        } else {
#pragma unroll
            for (int c = 0; c < CPL; c++) sr[c] = (ST)0.f;
        }
    };

    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
    // rows beyond the last are worked on as copies of the last one and not stored: every lane of a workgroup
    // makes the same number of rounds, which the exchanges and barriers inside need
    const int64_t last = a.rows - 1;
    fetch(row < last ? row : last);
    GateWalk<XT> gate;
    gate.init(a, row, step);
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.rows; base += step, row += step) {
        const bool ok = row <= last;
        const int64_t rr = ok ? row : last;
        const float g = gate.get(a);
        gate.next(a);
        float v[CPL][8], s[CPL][8];
#pragma unroll
        for (int c = 0; c < CPL; c++) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[c][j] = (float)xr[c][j];
                s[c][j] = (float)sr[c][j];
            }
        }
        if (base + step < a.rows) fetch(row + step < last ? row + step : last);

        if (pre) {
#pragma unroll
            for (int c = 0; c < CPL; c++) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[c][j] = s[c][j] + g * v[c][j];
                if (ok) row_store8<VEC>(reinterpret_cast<ST*>(a.h) + rr * dim, 8 * (c * LPR + l), dim, v[c]);
            }
        }
        float m = 0.f;
        if (layer) {
            float t = 0.f;
#pragma unroll
            for (int c = 0; c < CPL; c++)
#pragma unroll
                for (int j = 0; j < 8; j++) t += v[c][j];
            m = row_sum<LPR>(t, red, slot) * inv_dim;
        }
        float q = 0.f;
#pragma unroll
        for (int c = 0; c < CPL; c++) {
            const int c0 = 8 * (c * LPR + l);
            float qc = 0.f;     // columns beyond the row's end hold 0 - m: left out, whole chunks at a time where rows have those
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float d = VEC || c0 + j < dim ? v[c][j] - m : 0.f;
                v[c][j] = d;
                qc += d * d;
            }
            q += !VEC || c0 < dim ? qc : 0.f;
        }
        // one v_rsq_f32 (1 ulp) instead of a square root and a division (some 30 instructions); its argument is at least eps
        const float r = __builtin_amdgcn_rsqf(row_sum<LPR>(q, red, slot) * inv_dim + a.eps);
        if (a.stats != nullptr && ok && l == 0) a.stats[rr] = make_float2(m, r);

#pragma unroll
        for (int c = 0; c < CPL; c++) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[c][j] = __builtin_fmaf(v[c][j] * r, w[c][j], b[c][j]);
                if (!pre) v[c][j] = __builtin_fmaf(g, v[c][j], s[c][j]);
            }
        }
        if (a.y != nullptr && ok) {
#pragma unroll
            for (int c = 0; c < CPL; c++) {
                const int c0 = 8 * (c * LPR + l);
                if (pre) row_store8<VEC>(reinterpret_cast<XT*>(a.y) + rr * dim, c0, dim, v[c]);
                else row_store8<VEC>(reinterpret_cast<ST*>(a.y) + rr * dim, c0, dim, v[c]);
            }
        }
        if (a.y8 != nullptr) {
            uint32_t amax = 0;
#pragma unroll
            for (int c = 0; c < CPL; c++)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    amax = MaxU::of(amax, (VEC ? 8 * (c * LPR + l) < dim : 8 * (c * LPR + l) + j < dim) ? abs_bits(v[c][j]) : 0);
            const RowScale sc = scale_of(row_reduce<MaxU, LPR>(amax, red, slot));
            if (ok) {
                if (l == 0) a.y8_scale[rr] = sc.scale;
#pragma unroll
                for (int c = 0; c < CPL; c++) store_e4m3<VEC>(a.y8 + rr * dim, 8 * (c * LPR + l), dim, v[c], sc);
            }
        }
    }
}

// ---- backward -----------------------------------------------------------------------------------------------
// The rows' source v: x (POST); the saved h where the stream is fp32 (PRE); s + g x once more where it is not: h was rounded
// to 16 bits when it left the forward call, and v^ taken from it would carry that rounding into every sum over the rows
// (dweight 1.4 times as far from the exact one as its own rounding puts it) for one read less of nine.
template <class XT, class ST, bool PRE, int LPR, int CPL, bool VEC>
__global__ void __launch_bounds__(norm_block(LPR)) norm_bwd_kernel(const NormArgs a) {
    constexpr bool TWO = PRE && !std::is_same<ST, float>::value;    // v = s + g x
    typedef typename std::conditional<PRE, ST, XT>::type VT;       // of v (of s)
    typedef typename std::conditional<PRE, XT, ST>::type YT;       // of dy
    constexpr int RPB = norm_block(LPR) / LPR;
    __shared__ uint32_t red[32];
    __shared__ float cols[LPR <= 64 ? 2 * 8 * LPR * CPL : 1];
    int slot = 0;
    const int l = threadIdx.x % LPR;
    const int dim = a.dim;
    const float inv_dim = 1.f / (float)dim;
    const bool layer = a.layer;

    float w[CPL][8], dw[CPL][8], db[CPL][8];
#pragma unroll
    for (int c = 0; c < CPL; c++) {
        param_load8<VEC, XT>(a.weight, a.param_f32, 8 * (c * LPR + l), dim, w[c]);
#pragma unroll
        for (int j = 0; j < 8; j++) dw[c][j] = db[c][j] = 0.f;
    }

    typename Vec8<VT>::V vr[CPL];
    typename Vec8<XT>::V xr[TWO ? CPL : 1];
    typename Vec8<YT>::V yr[CPL];
    typename Vec8<ST>::V hr[PRE ? CPL : 1];
    float2 st;
    auto fetch = [&](int64_t row) __attribute__((always_inline)) {
        const VT* vp = TWO   ? reinterpret_cast<const VT*>(a.s) + row * a.ss
                       : PRE ? reinterpret_cast<const VT*>(a.h) + row * dim
                             : reinterpret_cast<const VT*>(a.x) + row * a.xs;
        const YT* yp = reinterpret_cast<const YT*>(a.dy) + row * a.dys;
        st = a.stats[row];
#pragma unroll
        for (int c = 0; c < CPL; c++) vr[c] = row_load8<VEC>(vp, 8 * (c * LPR + l), dim);
        if (TWO) {
            const XT* xp = reinterpret_cast<const XT*>(a.x) + row * a.xs;
#pragma unroll
            for (int c = 0; c < CPL; c++) xr[TWO ? c : 0] = row_load8<VEC>(xp, 8 * (c * LPR + l), dim);
        }
        if (!PRE || a.dy != nullptr) {
#pragma unroll
            for (int c = 0; c < CPL; c++) yr[c] = row_load8<VEC>(yp, 8 * (c * LPR + l), dim);
        } else {
#pragma unroll
            for (int c = 0; c < CPL; c++) yr[c] = (YT)0.f;
        }
        if (PRE) {
            const ST* hp = reinterpret_cast<const ST*>(a.dh) + row * a.dhs;
#pragma unroll
            for (int c = 0; c < CPL; c++) {
                if (a.dh != nullptr) hr[PRE ? c : 0] = row_load8<VEC>(hp, 8 * (c * LPR + l), dim);
                else hr[PRE ? c : 0] = (ST)0.f;
            }
        }
    };

    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
    const int64_t last = a.rows - 1;
    fetch(row < last ? row : last);
    GateWalk<XT> gate;
    gate.init(a, row, step);
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.rows; base += step, row += step) {
        const bool ok = row <= last;
        const int64_t rr = ok ? row : last;
        const float g = gate.get(a);
        gate.next(a);
        if (base + RPB > a.rows && !ok) {       // a row beyond the last: adds zeros to the column sums
            st = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < CPL; c++) {
                vr[c] = (VT)0.f;
                yr[c] = (YT)0.f;
                if (TWO) xr[TWO ? c : 0] = (XT)0.f;
            }
        }
        const float m = st.x, r = st.y;
        float v[CPL][8], t[CPL][8], up[PRE ? CPL : 1][8];
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int c = 0; c < CPL; c++) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float src = (float)vr[c][j];
                if (TWO) src += g * (float)xr[TWO ? c : 0][j];
                const float vh = (src - m) * r;
                const float dn = PRE ? (float)yr[c][j] : g * (float)yr[c][j];
                dw[c][j] += dn * vh;
                db[c][j] += dn;
                v[c][j] = vh;
                t[c][j] = dn * w[c][j];
                c1 += t[c][j];
                c2 += t[c][j] * vh;
                if (PRE) up[PRE ? c : 0][j] = (float)hr[PRE ? c : 0][j];
            }
        }
        if (base + step < a.rows) fetch(row + step < last ? row + step : last);
        if (a.dx == nullptr && a.ds == nullptr) continue;

        c1 = layer ? row_sum<LPR>(c1, red, slot) * inv_dim : 0.f;
        c2 = row_sum<LPR>(c2, red, slot) * inv_dim;
#pragma unroll
        for (int c = 0; c < CPL; c++) {
            const int c0 = 8 * (c * LPR + l);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                t[c][j] = r * (t[c][j] - c1 - v[c][j] * c2);
                if (PRE) t[c][j] += up[PRE ? c : 0][j];
            }
            if (!ok) continue;
            if (PRE) {
                if (a.ds != nullptr) row_store8<VEC>(reinterpret_cast<ST*>(a.ds) + rr * dim, c0, dim, t[c]);
                if (a.dx != nullptr) {
#pragma unroll
                    for (int j = 0; j < 8; j++) t[c][j] *= g;
                    row_store8<VEC>(reinterpret_cast<XT*>(a.dx) + rr * dim, c0, dim, t[c]);
                }
            } else {
                row_store8<VEC>(reinterpret_cast<XT*>(a.dx) + rr * dim, c0, dim, t[c]);
            }
        }
    }
    if (!a.want_params) return;

    // Column sums of the workgroup: over the rows that share a wavefront by lane exchange, over the wavefronts one
    // after the other through LDS (a fixed order), then one partial row per workgroup.
    float* part = a.part + (int64_t)blockIdx.x * 2 * dim;
    if (LPR <= 64) {
#pragma unroll
        for (int c = 0; c < CPL; c++)
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int off = LPR; off < 64; off <<= 1) {
                    dw[c][j] += __shfl_xor(dw[c][j], off);
                    db[c][j] += __shfl_xor(db[c][j], off);
                }
        constexpr int N = 8 * LPR * CPL;
        const int wave = threadIdx.x >> 6;
        for (int i = 0; i < 4; i++) {
            if (wave == i && (threadIdx.x & 63) < LPR) {
#pragma unroll
                for (int c = 0; c < CPL; c++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        // element j of chunk (c, l) sits in plane j: neighbouring lanes use neighbouring banks
                        const int at = j * LPR * CPL + c * LPR + l;
                        cols[at] = i ? cols[at] + dw[c][j] : dw[c][j];
                        cols[N + at] = i ? cols[N + at] + db[c][j] : db[c][j];
                    }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < dim; i += norm_block(LPR)) {
            const int at = (i & 7) * LPR * CPL + (i >> 3);
            part[i] = cols[at];
            part[dim + i] = cols[N + at];
        }
    } else {
#pragma unroll
        for (int c = 0; c < CPL; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int col = 8 * (c * LPR + l) + j;
                if (col < dim) {
                    part[col] = dw[c][j];
                    part[dim + col] = db[c][j];
                }
            }
    }
}

// ---- 8-bit form of rows -------------------------------------------------------------------------------------
template <class XT, int LPR, int CPL, bool VEC>
__global__ void __launch_bounds__(norm_block(LPR)) quantize_rows_kernel(const XT* x, int64_t rows, int dim, int64_t xs,
                                                                        uint8_t* q, float* scale) {
    constexpr int RPB = norm_block(LPR) / LPR;
    __shared__ uint32_t red[32];
    int slot = 0;
    const int l = threadIdx.x % LPR;
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < rows; base += (int64_t)gridDim.x * RPB) {
        const int64_t row = base + threadIdx.x / LPR;
        const bool ok = row < rows;
        const int64_t rr = ok ? row : rows - 1;
        float v[CPL][8];
        uint32_t amax = 0;
#pragma unroll
        for (int c = 0; c < CPL; c++) {
            const typename Vec8<XT>::V r = row_load8<VEC>(x + rr * xs, 8 * (c * LPR + l), dim);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[c][j] = (float)r[j];
                amax = MaxU::of(amax, abs_bits(v[c][j]));
            }
        }
        const RowScale sc = scale_of(row_reduce<MaxU, LPR>(amax, red, slot));
        if (!ok) continue;
        if (l == 0) scale[rr] = sc.scale;
#pragma unroll
        for (int c = 0; c < CPL; c++) store_e4m3<VEC>(q + rr * dim, 8 * (c * LPR + l), dim, v[c], sc);
    }
}

// ---- launch ---------------------------------------------------------------------------------------------------
// How a row of `dim` elements is spread over lanes: the fewest lanes that hold it with one chunk each up to 512 elements,
// a wavefront with up to 4 chunks per lane up to 2048 (registers: a chunk costs backward 40 of them), then workgroups.
#define FWA2_NORM_SHAPES(F)      \
    if (dim <= 64) F(8, 1)       \
    else if (dim <= 128) F(16, 1) \
    else if (dim <= 256) F(32, 1) \
    else if (dim <= 512) F(64, 1) \
    else if (dim <= 1024) F(64, 2) \
    else if (dim <= 1536) F(64, 3) \
    else if (dim <= 2048) F(64, 4) \
    else if (dim <= 4096) F(256, 2) \
    else if (dim <= 8192) F(256, 4) \
    else F(512, 4)

template <class XT, class ST>
static void forward_typed(const NormArgs& a, bool vec, int cus, hipStream_t st) {
    const int dim = a.dim;
#define FWA2_GO(LPR, CPL) {                                                                                        \
        constexpr int rpb = norm_block(LPR) / LPR;                                                                  \
        const int64_t tiles = (a.rows + rpb - 1) / rpb;                                                             \
        const int64_t most = (int64_t)cus * (2048 / norm_block(LPR));                                               \
        const dim3 grid((unsigned)(tiles < most ? tiles : most)), block(norm_block(LPR));                           \
        if (vec) hipLaunchKernelGGL((norm_fwd_kernel<XT, ST, LPR, CPL, true>), grid, block, 0, st, a);             \
        else hipLaunchKernelGGL((norm_fwd_kernel<XT, ST, LPR, CPL, false>), grid, block, 0, st, a);                \
    }
    FWA2_NORM_SHAPES(FWA2_GO)
#undef FWA2_GO
}
template <class XT, class ST>
static void backward_typed(const NormArgs& a, bool vec, int blocks, hipStream_t st) {
    const int dim = a.dim;
#define FWA2_GO(LPR, CPL) {                                                                                        \
        const dim3 grid(blocks), block(norm_block(LPR));                                                            \
        if (a.pre) {                                                                                                \
            if (vec) hipLaunchKernelGGL((norm_bwd_kernel<XT, ST, true, LPR, CPL, true>), grid, block, 0, st, a);   \
            else hipLaunchKernelGGL((norm_bwd_kernel<XT, ST, true, LPR, CPL, false>), grid, block, 0, st, a);      \
        } else {                                                                                                    \
            if (vec) hipLaunchKernelGGL((norm_bwd_kernel<XT, ST, false, LPR, CPL, true>), grid, block, 0, st, a);  \
            else hipLaunchKernelGGL((norm_bwd_kernel<XT, ST, false, LPR, CPL, false>), grid, block, 0, st, a);     \
        }                                                                                                           \
    }
    FWA2_NORM_SHAPES(FWA2_GO)
#undef FWA2_GO
}
// A launch has fewer than 2^32 threads: beyond so many workgroups each takes several stretches of rows.
constexpr int64_t kQuantizeBlocks = 1 << 16;
template <class XT>
static void quantize_typed(const void* x, int64_t rows, int dim, int64_t xs, void* q, float* scale, bool vec, hipStream_t st) {
#define FWA2_GO(LPR, CPL) {                                                                                        \
        constexpr int rpb = norm_block(LPR) / LPR;                                                                  \
        const int64_t tiles = (rows + rpb - 1) / rpb;                                                               \
        const dim3 grid((unsigned)(tiles < kQuantizeBlocks ? tiles : kQuantizeBlocks)), block(norm_block(LPR));     \
        if (vec) hipLaunchKernelGGL((quantize_rows_kernel<XT, LPR, CPL, true>), grid, block, 0, st,                \
                                    reinterpret_cast<const XT*>(x), rows, dim, xs, reinterpret_cast<uint8_t*>(q), scale); \
        else hipLaunchKernelGGL((quantize_rows_kernel<XT, LPR, CPL, false>), grid, block, 0, st,                   \
                                reinterpret_cast<const XT*>(x), rows, dim, xs, reinterpret_cast<uint8_t*>(q), scale); \
    }
    FWA2_NORM_SHAPES(FWA2_GO)
#undef FWA2_GO
}

// One half of this file per compile (the build compiles it twice): the bf16 side with fp32 rows and the host code, and
// the fp16 side.
#if FWA2_HALF == 1
#define FWA2_NORM_T __bf16
#define FWA2_NORM_FN(name) name##_bf16
#else
#define FWA2_NORM_T _Float16
#define FWA2_NORM_FN(name) name##_f16
#endif
void FWA2_NORM_FN(norm_forward)(const NormArgs& a, bool s32, bool vec, int cus, hipStream_t st) {
    if (s32) forward_typed<FWA2_NORM_T, float>(a, vec, cus, st);
    else forward_typed<FWA2_NORM_T, FWA2_NORM_T>(a, vec, cus, st);
}
void FWA2_NORM_FN(norm_backward)(const NormArgs& a, bool s32, bool vec, int blocks, hipStream_t st) {
    if (s32) backward_typed<FWA2_NORM_T, float>(a, vec, blocks, st);
    else backward_typed<FWA2_NORM_T, FWA2_NORM_T>(a, vec, blocks, st);
}
void FWA2_NORM_FN(norm_quantize)(const void* x, int64_t rows, int dim, int64_t xs, void* q, float* scale, bool vec, hipStream_t st) {
    quantize_typed<FWA2_NORM_T>(x, rows, dim, xs, q, scale, vec, st);
}

#if FWA2_HALF == 1
void norm_forward_f16(const NormArgs& a, bool s32, bool vec, int cus, hipStream_t st);
void norm_backward_f16(const NormArgs& a, bool s32, bool vec, int blocks, hipStream_t st);
void norm_quantize_f16(const void* x, int64_t rows, int dim, int64_t xs, void* q, float* scale, bool vec, hipStream_t st);

// dweight, dbias = sums of the partial rows.  A workgroup owns 64 columns of one of the two; its 16 wavefronts take
// every 16th partial row (a fixed assignment) and their sums are added in order.
__global__ void __launch_bounds__(1024) norm_params_kernel(const float* part, int parts, int dim, void* dweight, void* dbias,
                                                           int dt) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + lane, which = blockIdx.y;
    void* out = which ? dbias : dweight;
    if (out == nullptr) return;
    float t = 0.f;
    if (col < dim) {
        const float* p = part + (int64_t)which * dim + col;
#pragma unroll 16
        for (int i = wave; i < parts; i += 16) t += p[(int64_t)i * 2 * dim];
    }
    s[wave][lane] = t;
    __syncthreads();
    if (wave == 0 && col < dim) {
        for (int i = 1; i < 16; i++) t += s[i][lane];
        if (dt == FWA2_F32) reinterpret_cast<float*>(out)[col] = t;
        else if (dt == FWA2_BF16) reinterpret_cast<__bf16*>(out)[col] = (__bf16)t;
        else reinterpret_cast<_Float16*>(out)[col] = (_Float16)t;
    }
}

static int norm_rows_per_block(int dim) { return dim <= 64 ? 32 : dim <= 128 ? 16 : dim <= 256 ? 8 : dim <= 2048 ? 4 : 1; }

// Workgroups of a backward call: enough to fill the chip, and few enough that the partial rows (8 bytes per column and
// workgroup) stay well below the 6 to 12 bytes per element that the rows themselves move.
int norm_bwd_blocks(int64_t rows, int dim, int cus) {
    const int rpb = norm_rows_per_block(dim);
    const int64_t tiles = (rows + rpb - 1) / rpb;
    int64_t most = 4 * (int64_t)cus;
    const int64_t fair = rows / 32 > cus ? rows / 32 : cus;
    if (most > fair) most = fair;
    return (int)(tiles < most ? tiles : most);
}

static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static NormArgs norm_args(const fwa2_norm* p) {
    NormArgs a = {};
    a.x = p->x; a.s = p->shortcut; a.weight = p->weight; a.bias = p->bias; a.gate = p->gate;
    a.xs = p->x_stride; a.ss = p->shortcut_stride;
    a.y = p->y; a.h = p->h;
    a.y8 = reinterpret_cast<uint8_t*>(p->y8);
    a.y8_scale = p->y8_scale;
    a.stats = reinterpret_cast<float2*>(p->stats);
    a.dy = p->dy; a.dh = p->dh; a.dys = p->dy_stride; a.dhs = p->dh_stride;
    a.dx = p->dx; a.ds = p->dshortcut;
    a.part = reinterpret_cast<float*>(p->workspace);
    a.rows = p->rows;
    a.rows_per_gate = (uint32_t)(p->gate ? p->rows_per_gate : 1);
    a.gates = (uint32_t)(p->gate ? p->rows / p->rows_per_gate : 1);
    a.dim = p->dim;
    a.eps = p->eps;
    a.layer = p->kind == FWA2_NORM_LAYER;
    a.pre = p->placement == FWA2_NORM_PRE;
    a.param_f32 = p->param_dtype == FWA2_F32;
    a.gate_f32 = p->gate_dtype == FWA2_F32;
    a.want_params = p->dweight != nullptr || p->dbias != nullptr;
    return a;
}

hipError_t launch_norm_forward(const fwa2_norm* p, int cus, hipStream_t st) {
    const NormArgs a = norm_args(p);
    // 16-byte accesses: whole chunks per row, every row on a 16-byte boundary (outputs are contiguous, 8-byte for y8)
    const bool vec = p->dim % 8 == 0 && al16(p->x) && p->x_stride % 8 == 0 &&
                     (!p->shortcut || (al16(p->shortcut) && p->shortcut_stride % 8 == 0)) && al16(p->y) && al16(p->h) && al16(p->y8) &&
                     al16(p->weight) && al16(p->bias);
    const bool s32 = p->stream_dtype == FWA2_F32;
    if (p->dtype == FWA2_BF16) norm_forward_bf16(a, s32, vec, cus, st);
    else if (p->dtype == FWA2_F16) norm_forward_f16(a, s32, vec, cus, st);
    else forward_typed<float, float>(a, vec, cus, st);
    return hipGetLastError();
}

hipError_t launch_norm_backward(const fwa2_norm* p, int cus, hipStream_t st) {
    const NormArgs a = norm_args(p);
    const bool pre = p->placement == FWA2_NORM_PRE;
    const bool two = pre && p->stream_dtype != FWA2_F32;
    const bool vec = p->dim % 8 == 0 && (!pre || two ? al16(p->x) && p->x_stride % 8 == 0 : al16(p->h)) &&
                     (!two || (al16(p->shortcut) && p->shortcut_stride % 8 == 0)) &&
                     (!p->dy || (al16(p->dy) && p->dy_stride % 8 == 0)) && (!pre || !p->dh || (al16(p->dh) && p->dh_stride % 8 == 0)) &&
                     al16(p->dx) && (!pre || al16(p->dshortcut)) && al16(p->weight);
    const bool s32 = p->stream_dtype == FWA2_F32;
    const int blocks = norm_bwd_blocks(p->rows, p->dim, cus);
    if (p->dtype == FWA2_BF16) norm_backward_bf16(a, s32, vec, blocks, st);
    else if (p->dtype == FWA2_F16) norm_backward_f16(a, s32, vec, blocks, st);
    else backward_typed<float, float>(a, vec, blocks, st);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.want_params) return e;
    const dim3 grid((p->dim + 63) / 64, 2);
    hipLaunchKernelGGL(norm_params_kernel, grid, dim3(1024), 0, st, a.part, blocks, p->dim, p->dweight, p->dbias, p->param_dtype);
    return hipGetLastError();
}

hipError_t launch_quantize_rows(const void* x, int dtype, int64_t rows, int dim, int64_t xs, void* q, float* scale, hipStream_t st) {
    const bool vec = dim % 8 == 0 && al16(x) && xs % 8 == 0 && al16(q);
    if (dtype == FWA2_BF16) norm_quantize_bf16(x, rows, dim, xs, q, scale, vec, st);
    else if (dtype == FWA2_F16) norm_quantize_f16(x, rows, dim, xs, q, scale, vec, st);
    else quantize_typed<float>(x, rows, dim, xs, q, scale, vec, st);
    return hipGetLastError();
}

size_t norm_workspace_bytes(const fwa2_norm* p, int cus) {
    if (p->dweight == nullptr && p->dbias == nullptr) return 0;
    return (size_t)norm_bwd_blocks(p->rows, p->dim, cus) * 2 * p->dim * sizeof(float);
}
#endif

}  // namespace fwa2
