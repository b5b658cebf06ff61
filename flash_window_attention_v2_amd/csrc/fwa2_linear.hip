// Matrix products with an epilogue: y = act(x W^T + b) + residual, its backward pass, and the same product over 8-bit rows.
//
// One tile kernel computes D[p][q] = sum_k P[p][k] Q[q][k] with P's index along the accumulator rows of the MFMA, so that
// a lane holds consecutive p of one q: q is the row of the output in memory, p its column.  The three products of a
// linear layer differ in which operands have the contraction index innermost in memory:
//
//   forward   y[m][n]  = sum_k x[m][k] W[n][k]      Q = x  (k innermost)   P = W   (k innermost)
//   dx        dx[m][k] = sum_n dz[m][n] W[n][k]     Q = dz (n innermost)   P = W^T (k = p innermost: "transposed")
//   dW        dW[n][k] = sum_m dz[m][n] x[m][k]     Q = dz^T (transposed)  P = x^T (transposed)
//
// Operand tiles go from memory to LDS without passing through registers (16 bytes per lane), as they lie in memory: rows of
// KB bytes of the contraction, or, transposed, KE contraction rows of the tile's columns, which ds_read_b64_tr_b16
// turns into MFMA operands.  The landing place of a lane is fixed (lane * 16), so the layout is chosen by which chunk a lane
// asks for: chunk c of row r sits at c ^ f(r), with f such that the 16 (32) lanes that an operand read serves at a time
// touch every bank once.
//
// dW contracts over the rows of the batch and has few output tiles: the rows are split over workgroups, whose fp32
// partial tiles are added in a fixed order by a second kernel.  dbias is the same contraction against ones and rides on the
// matrix pipe of the workgroups with the first column tile.
#include "fwa2_common.hpp"

// One half of this file per compile: 1 the bf16 products and the host code, 2 fp16, 3 the 8-bit products.
#ifndef FWA2_HALF
#define FWA2_HALF 1
#endif

namespace fwa2 {

struct LinArgs {
    const char *p, *q;            // operands
    int64_t p_stride, q_stride;   // bytes between their memory rows
    int64_t nq, nk;               // extents: q rows of the output, contraction
    int np;                       // columns of the output
    int tiles_p;
    int64_t tiles;                // output tiles
    int splits;                   // of the contraction
    int64_t k_per_split;          // a multiple of the stage
    void* out;                    // [nq, np] of the element type, contiguous
    float* part;                  // [splits, nq, np] fp32 instead, with splits > 1
    float* part_db;               // [splits, nq] fp32, with splits > 1
    void* db;                     // [nq] of the element type (dW product only), or null
    // epilogue
    const void* bias;
    const char* residual;
    int64_t residual_stride;      // bytes
    void* z;
    const float *q_scale, *p_scale;
    int act;
    int out_vec;                  // output rows (and residual, z, bias) take 16-byte accesses
    int out_bf16;                 // 8-bit products: element type of the output
};

// What the hardware reads where a tile reaches over the end of the contraction.
static __device__ __attribute__((aligned(16))) const uint32_t k_zeros[4] = {0, 0, 0, 0};

template <int DT> struct LinElem { static constexpr int bytes = 2; };
template <> struct LinElem<FWA2_E4M3> { static constexpr int bytes = 1; };

// ---- activations -------------------------------------------------------------------------------------------
__device__ __forceinline__ float act_of(float z, int act) {
    switch (act) {
        case FWA2_ACT_GELU: return z * (0.5f * (1.f + erff(z * 0.70710678118654752f)));
        case FWA2_ACT_GELU_TANH: {
            // z sigmoid(2u) = z / 2 (1 + tanh(u))
            const float u2 = z * (1.5957691216057308f + 0.07135481282553505f * z * z);
            return z / (1.f + __expf(-u2));
        }
        case FWA2_ACT_SILU: return z / (1.f + __expf(-z));
        case FWA2_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
        default: return z;
    }
}
// d act / dz.  Beyond |z| = 100 every slope is 0 or 1 to fp32, and z (kept in 16 bits, possibly overflowed to infinity) must
// not meet a zero factor; NaN stays NaN (the comparison is false).
__device__ __forceinline__ float slope_of(float z, int act) {
    if (fabsf(z) > 100.f) z = copysignf(100.f, z);
    switch (act) {
        case FWA2_ACT_GELU:
            return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.3989422804014327f * __expf(-0.5f * z * z);
        case FWA2_ACT_GELU_TANH: {
            const float z2 = z * z;
            const float s = 1.f / (1.f + __expf(-z * (1.5957691216057308f + 0.07135481282553505f * z2)));
            return s + z * s * (1.f - s) * (1.5957691216057308f + 0.21406443847660515f * z2);
        }
        case FWA2_ACT_SILU: {
            const float s = 1.f / (1.f + __expf(-z));
            return s * (1.f + z * (1.f - s));
        }
        case FWA2_ACT_RELU: return z > 0.f ? 1.f : (z != z ? z : 0.f);
        default: return 1.f;
    }
}

// ---- memory to LDS -----------------------------------------------------------------------------------------
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void tile_dma(const void* uniform_base, uint32_t byte_offset, uint32_t lds) {
    asm volatile("s_nop 3\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(byte_offset), "s"(uniform_base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void tile_dma(const void* src, uint32_t lds) {
    asm volatile("s_nop 3\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory"); }

// Chunk permutation of a memory row in LDS.  Plain rows of KB = 128 (64) bytes: two (four) rows share the 256 bytes that
// the banks span, and an operand read serves rows {0-3, 12-15} of one chunk with rows {4-11} of its neighbour.
template <int KB>
__device__ __forceinline__ int plain_swizzle(int row) {
    if (KB == 128) return (row >> 1) & 7;
    const int v = (row >> 2) & 3;
    return ((v & 1) << 1) ^ ((v >> 1) * 3);
}
// Transposed rows of R columns: a read serves 8 contraction rows {0-3, 8-11} with 32 bytes each.  In units of 32 bytes.
template <int R>
__device__ __forceinline__ int turned_swizzle(int k) {
    if (R >= 128) return (k & 3) | (((k >> 3) & 1) << 2);
    return ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
}

// One operand's tile: R rows (columns, transposed) by one stage of the contraction.
template <int DT, bool TURNED, int R, int KB, int NW, bool VEC>
struct Operand {
    static constexpr int EB = LinElem<DT>::bytes;
    static constexpr int KE = KB / EB;                      // contraction elements of a stage
    static constexpr int BYTES = R * KB;
    static constexpr int CPR = TURNED ? R * EB / 16 : KB / 16;  // 16-byte chunks of a row in LDS
    static constexpr int NI = BYTES / 1024 / NW;            // copies per wavefront and stage
    static_assert(NI * 1024 * NW == BYTES, "whole copies");
    static constexpr int CE = 16 / EB;                      // elements of a chunk

    const char* base;       // uniform: first row (column) of the tile, first contraction element of the split
    int64_t stride;
    int64_t step;           // bytes from stage to stage
    uint32_t off[VEC ? NI : 1];
    int rows;               // rows (columns) of the tile inside the matrix
    int wave, lane;

    __device__ __forceinline__ void init(const char* ptr, int64_t str, int64_t first, int64_t extent, int64_t k0, int w, int l) {
        stride = str;
        wave = w;
        lane = l;
        const int64_t left = extent - first;
        rows = left < R ? (int)left : R;
        if (TURNED) {
            base = ptr + k0 * str + first * EB;
            step = (int64_t)KE * str;
        } else {
            base = ptr + first * str + k0 * EB;
            step = KB;
        }
        base = reinterpret_cast<const char*>(uniform_pointer(base));
        if (VEC) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                int row, c;
                place(i, row, c);
                off[i] = offset(row, c);
            }
        }
    }
    // LDS row of this lane's part of copy i, and the memory chunk that belongs there
    __device__ __forceinline__ void place(int i, int& row, int& c) const {
        const int ci = (i * NW + wave) * 64 + lane;
        row = ci / CPR;
        c = ci % CPR;
        c ^= TURNED ? 2 * turned_swizzle<R>(row) : plain_swizzle<KB>(row);
    }
    // Rows (columns) beyond the matrix repeat the last ones: what they produce is not stored.
    __device__ __forceinline__ uint32_t offset(int row, int c) const {
        if (TURNED) return (uint32_t)row * (uint32_t)stride + (uint32_t)(c * CE < rows ? c * 16 : rows * EB - 16);
        return (uint32_t)(row < rows ? row : rows - 1) * (uint32_t)stride + (uint32_t)c * 16;
    }
    // Ask for stage kt, of which `left` contraction elements are inside the matrix.
    __device__ __forceinline__ void issue(int64_t kt, int left, char* lds) const {
        const char* at = base + kt * step;
        const uint32_t dst = lds_address(lds) + wave * 1024;
        if (left >= KE) {
#pragma unroll
            for (int i = 0; i < NI; i++) tile_dma(at, off[i], dst + i * NW * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                int row, c;
                place(i, row, c);
                const bool in = TURNED ? row < left : c * CE < left;
                const void* src = in ? (const void*)(at + offset(row, c)) : (const void*)k_zeros;
                tile_dma(src, dst + i * NW * 1024);
            }
        }
    }
    // The same through registers, for rows off 16-byte boundaries and extents that end inside a chunk.
    __device__ __forceinline__ void fetch(int64_t kt, int left, u32x4* r) const {
        const char* at = base + kt * step;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            int row, c;
            place(i, row, c);
            int n;              // elements of the chunk inside the matrix
            const char* src;
            if (TURNED) {
                n = row < left ? rows - c * CE : 0;
                src = at + (int64_t)row * stride + c * 16;
            } else {
                n = left - c * CE;
                src = at + (int64_t)(row < rows ? row : rows - 1) * stride + c * 16;
            }
            r[i] = u32x4{0, 0, 0, 0};
            if (n >= CE) {
                __builtin_memcpy(&r[i], src, 16);
            } else if (n > 0) {
                for (int j = 0; j < CE; j++) {
                    if (j >= n) break;
                    uint32_t e;
                    if (EB == 2) e = reinterpret_cast<const uint16_t*>(src)[j];
                    else e = reinterpret_cast<const uint8_t*>(src)[j];
                    const int bit = j * EB * 8;
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (x == bit / 32) r[i][x] |= e << (bit % 32);
                }
            }
        }
    }
    __device__ __forceinline__ void put(const u32x4* r, char* lds) const {
#pragma unroll
        for (int i = 0; i < NI; i++) *reinterpret_cast<u32x4*>(lds + ((i * NW + wave) * 64 + lane) * 16) = r[i];
    }
};

// MFMA operands of 16 rows out of a staged tile.
template <int DT> struct Frag {
    typedef typename Elem<DT>::V8 V;
    static constexpr int K = 32;
    static __device__ __forceinline__ V plain(const char* tile, int row, int swz, int g, int kk, int kb) {
        return *reinterpret_cast<const V*>(tile + row * kb + (((kk * 4 + g) ^ swz) * 16));
    }
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) { return Elem<DT>::mfma16(a, b, c); }
};
typedef int i32x8 __attribute__((ext_vector_type(8)));
template <> struct Frag<FWA2_E4M3> {
    typedef i32x8 V;
    static constexpr int K = 128;
    // A lane takes chunks g and g + 4 of its row: which contraction elements a lane holds does not matter as long as both
    // operands agree, and these two keep the banks apart.
    static __device__ __forceinline__ V plain(const char* tile, int row, int swz, int g, int kk, int kb) {
        const u32x4 a = *reinterpret_cast<const u32x4*>(tile + row * kb + ((g ^ swz) * 16));
        const u32x4 b = *reinterpret_cast<const u32x4*>(tile + row * kb + (((g + 4) ^ swz) * 16));
        V v;
#pragma unroll
        for (int i = 0; i < 4; i++) { v[i] = (int)a[i]; v[4 + i] = (int)b[i]; }
        return v;
    }
    // The 8-bit unit adds products in groups of 8 contraction elements aligned to the group's largest and drops what lies
    // below 2^-13 of that (measured, for this form as for the 32-element one); the groups are added in fp32.  Against the
    // 2^-4 half steps of the operands that is nothing, and the alternative, converting the tiles to 16 bits for the
    // exact products of the other unit, halves the matrix rate.
    // 0x7f: a block scale of 2^0 in every byte
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
    }
};
template <int DT, int R>
__device__ __forceinline__ typename Elem<DT>::V8 frag_turned(const char* tile, int t16, int l16, int g, int kk) {
    const int k = kk * 32 + 8 * g + (l16 >> 2);
    const int at = k * R * 2 + ((t16 ^ turned_swizzle<R>(k)) * 32) + (l16 & 3) * 8;
    typedef typename Elem<DT>::E E;
    const E* lo = reinterpret_cast<const E*>(tile + at);
    return lds_tr8<DT>(lo, lo + 4 * R);
}

// Which tile a workgroup computes.  Workgroups go to the 8 XCDs in turn, each with an L2 of its own: consecutive tiles are
// given to one XCD, column tiles first, so that the tiles that share a block of Q rows meet in one L2.
__device__ __forceinline__ int64_t tile_of_block(int64_t block, int64_t total) {
    const int64_t per = (total + 7) / 8;
    return (block & 7) * per + (block >> 3);
}

template <class OT>
__device__ __forceinline__ void epilogue8(const LinArgs& a, float* v, const float* bias, int64_t q, int p, int n) {
    typedef OT V8 __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] += bias[j];
    OT* z = reinterpret_cast<OT*>(a.z);
    OT* out = reinterpret_cast<OT*>(a.out);
    const int64_t at = q * a.np + p;
    if (a.out_vec) {        // np is a multiple of 8: the chunk is inside or outside as a whole
        if (z != nullptr) {
            V8 t;
#pragma unroll
            for (int j = 0; j < 8; j++) t[j] = (OT)v[j];
            *reinterpret_cast<V8*>(z + at) = t;
        }
        if (a.act != FWA2_ACT_NONE)
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = act_of(v[j], a.act);
        if (a.residual != nullptr) {
            const V8 r = *reinterpret_cast<const V8*>(reinterpret_cast<const OT*>(a.residual + q * a.residual_stride) + p);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] += (float)r[j];
        }
        V8 t;
#pragma unroll
        for (int j = 0; j < 8; j++) t[j] = (OT)v[j];
        *reinterpret_cast<V8*>(out + at) = t;
    } else {
        const OT* r = reinterpret_cast<const OT*>(a.residual + q * a.residual_stride);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (j >= n) continue;
            if (z != nullptr) z[at + j] = (OT)v[j];
            float y = act_of(v[j], a.act);
            if (a.residual != nullptr) y += (float)r[p + j];
            out[at + j] = (OT)y;
        }
    }
}
template <class OT>
__device__ __forceinline__ void bias8(const LinArgs& a, int p, float* b) {
#pragma unroll
    for (int j = 0; j < 8; j++) b[j] = a.bias != nullptr && p + j < a.np ? (float)reinterpret_cast<const OT*>(a.bias)[p + j] : 0.f;
}

// Two accumulator tiles of 16 output columns become 8 consecutive columns per lane: the lanes of rows 1 and 3 of the first
// change places with those of rows 0 and 2 of the second.  Column of the lane's first value within the 32:
__device__ __forceinline__ int pair_column(int g) { return ((g & 1) << 4) | ((g >> 1) << 3); }
__device__ __forceinline__ void pair_swap(f32x4 a, f32x4 b, float* v) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const u32x2 s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[r]), __float_as_uint(b[r]), false, false);
        v[r] = __uint_as_float(s[0]);
        v[4 + r] = __uint_as_float(s[1]);
    }
}

template <int DT, bool PT, bool QT, int BP, int BQ, int WP, int WQ, int KB, int STAGES, bool VEC>
__global__ void __launch_bounds__(64 * WP * WQ) linear_kernel(const LinArgs a) {
    constexpr int NW = WP * WQ;
    constexpr int TP = BP / WP, TQ = BQ / WQ;       // a wavefront's part of the tile
    constexpr int FP = TP / 16, FQ = TQ / 16;
    static_assert(TP % 32 == 0 && TQ % 16 == 0, "");
    typedef Operand<DT, PT, BP, KB, NW, VEC> OP;
    typedef Operand<DT, QT, BQ, KB, NW, VEC> OQ;
    constexpr int KE = OP::KE;
    constexpr int KSTEPS = KE / Frag<DT>::K;
    constexpr int STAGE = OP::BYTES + OQ::BYTES;
    constexpr bool DB = PT && QT;
    __shared__ __attribute__((aligned(1024))) char lds[STAGES * STAGE];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave % WP, wq = wave / WP;
    const int l16 = lane & 15, g = lane >> 4;

    const int64_t total = a.tiles * a.splits;
    const int64_t t = tile_of_block(blockIdx.x, total);
    if (t >= total) return;
    const int64_t tile = t / a.splits;
    const int split = (int)(t - tile * a.splits);
    const int64_t q0 = (tile / a.tiles_p) * BQ;
    const int p0 = (int)(tile % a.tiles_p) * BP;
    const int64_t k0 = split * a.k_per_split;
    const int64_t k1 = k0 + a.k_per_split < a.nk ? k0 + a.k_per_split : a.nk;
    const int64_t len = k1 - k0;
    const int64_t nkt = (len + KE - 1) / KE;
    auto left_of = [&](int64_t kt) { const int64_t l = len - kt * KE; return l < KE ? (int)l : KE; };

    OP P;
    OQ Q;
    P.init(a.p, a.p_stride, p0, a.np, k0, wave, lane);
    Q.init(a.q, a.q_stride, q0, a.nq, k0, wave, lane);

    f32x4 acc[FQ][FP];
#pragma unroll
    for (int i = 0; i < FQ; i++)
#pragma unroll
        for (int j = 0; j < FP; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 accb[DB ? FQ : 1];
#pragma unroll
    for (int i = 0; i < (DB ? FQ : 1); i++) accb[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const bool sum_rows = DB && a.db != nullptr && p0 == 0 && wp == 0;

    auto compute = [&](const char* buf, int left) __attribute__((always_inline)) {
        const char* tp = buf;
        const char* tq = buf + OP::BYTES;
        const int swz = plain_swizzle<KB>(l16);
#pragma unroll
        for (int kk = 0; kk < KSTEPS; kk++) {
            if (kk * Frag<DT>::K >= left) break;
            typename Frag<DT>::V fp[FP], fq[FQ];
#pragma unroll
            for (int j = 0; j < FP; j++) {
                if constexpr (PT) fp[j] = frag_turned<DT, BP>(tp, wp * FP + j, l16, g, kk);
                else fp[j] = Frag<DT>::plain(tp, wp * TP + 16 * j + l16, swz, g, kk, KB);
            }
#pragma unroll
            for (int i = 0; i < FQ; i++) {
                if constexpr (QT) fq[i] = frag_turned<DT, BQ>(tq, wq * FQ + i, l16, g, kk);
                else fq[i] = Frag<DT>::plain(tq, wq * TQ + 16 * i + l16, swz, g, kk, KB);
            }
#pragma unroll
            for (int i = 0; i < FQ; i++)
#pragma unroll
                for (int j = 0; j < FP; j++) acc[i][j] = Frag<DT>::mfma(fp[j], fq[i], acc[i][j]);
            if constexpr (DB) {
                if (sum_rows) {
                    typename Frag<DT>::V ones;
#pragma unroll
                    for (int j = 0; j < 8; j++) ones[j] = (typename Elem<DT>::E)1.f;
#pragma unroll
                    for (int i = 0; i < FQ; i++) accb[i] = Frag<DT>::mfma(ones, fq[i], accb[i]);
                }
            }
        }
    };

    if constexpr (VEC) {
        static_assert(STAGES >= 2, "");
#pragma unroll
        for (int s = 0; s < STAGES - 1; s++) {
            if (s < nkt) {
                P.issue(s, left_of(s), lds + s * STAGE);
                Q.issue(s, left_of(s), lds + s * STAGE + OP::BYTES);
            }
        }
        int cur = 0, nxt = STAGES - 1;
        for (int64_t kt = 0; kt < nkt; kt++) {
            // stage kt has landed when at most the copies of the later stages are still out
            if (kt + STAGES - 1 <= nkt) wait_vm<(STAGES - 2) * (OP::NI + OQ::NI)>();
            else wait_vm<0>();
            lds_barrier();      // ... for every wavefront, and all have read the stage that the next copies overwrite
            const int64_t kn = kt + STAGES - 1;
            if (kn < nkt) {
                P.issue(kn, left_of(kn), lds + nxt * STAGE);
                Q.issue(kn, left_of(kn), lds + nxt * STAGE + OP::BYTES);
            }
            compute(lds + cur * STAGE, left_of(kt));
            cur = cur + 1 == STAGES ? 0 : cur + 1;
            nxt = nxt + 1 == STAGES ? 0 : nxt + 1;
        }
    } else {
        u32x4 rp[OP::NI], rq[OQ::NI];
        P.fetch(0, left_of(0), rp);
        Q.fetch(0, left_of(0), rq);
        for (int64_t kt = 0; kt < nkt; kt++) {
            char* buf = lds + (kt & 1) * STAGE;
            P.put(rp, buf);
            Q.put(rq, buf + OP::BYTES);
            lds_barrier();      // this stage is whole; the other half was read before the previous barrier's successor
            if (kt + 1 < nkt) {
                P.fetch(kt + 1, left_of(kt + 1), rp);
                Q.fetch(kt + 1, left_of(kt + 1), rq);
            }
            compute(buf, left_of(kt));
        }
    }

    const int64_t qw = q0 + wq * TQ + l16;
    const int pw = p0 + wp * TP;
    if (a.splits > 1) {
        float* out = a.part + (int64_t)split * a.nq * a.np;
#pragma unroll
        for (int i = 0; i < FQ; i++) {
            const int64_t q = qw + 16 * i;
            if (q >= a.nq) continue;
#pragma unroll
            for (int j = 0; j < FP; j++) {
                const int p = pw + 16 * j + 4 * g;
                float* o = out + q * a.np + p;
                if (a.np % 4 == 0) {
                    if (p < a.np) *reinterpret_cast<f32x4*>(o) = acc[i][j];
                } else {
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (p + r < a.np) o[r] = acc[i][j][r];
                }
            }
            if (DB && sum_rows && g == 0) a.part_db[split * a.nq + q] = accb[DB ? i : 0][0];
        }
        return;
    }
    auto finish = [&](auto tag) __attribute__((always_inline)) {
        typedef decltype(tag) OT;
#pragma unroll
        for (int u = 0; u < FP / 2; u++) {
            const int p = pw + 32 * u + pair_column(g);
            float bias[8], ps[8];
            bias8<OT>(a, p, bias);
            if constexpr (DT == FWA2_E4M3) {
#pragma unroll
                for (int j = 0; j < 8; j++) ps[j] = p + j < a.np ? a.p_scale[p + j] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < FQ; i++) {
                const int64_t q = qw + 16 * i;
                float v[8];
                pair_swap(acc[i][2 * u], acc[i][2 * u + 1], v);     // exchanged by all lanes, stored by those inside
                if (q >= a.nq || p >= a.np) continue;
                if constexpr (DT == FWA2_E4M3) {
                    const float qs = a.q_scale[q];
#pragma unroll
                    for (int j = 0; j < 8; j++) v[j] *= qs * ps[j];
                }
                epilogue8<OT>(a, v, bias, q, p, a.np - p);
            }
        }
        if (DB && sum_rows && g == 0) {
#pragma unroll
            for (int i = 0; i < FQ; i++)
                if (qw + 16 * i < a.nq) reinterpret_cast<OT*>(a.db)[qw + 16 * i] = (OT)accb[DB ? i : 0][0];
        }
    };
    if constexpr (DT == FWA2_E4M3) {
        if (a.out_bf16) finish((__bf16)0.f);
        else finish((_Float16)0.f);
    } else {
        finish((typename Elem<DT == FWA2_E4M3 ? FWA2_F16 : DT>::E)0.f);
    }
}

#if FWA2_HALF != 3
// dW, db = sums of the partial tiles, rounded once.  A workgroup owns 256 values; its 16 wavefronts take every 16th partial
// (a fixed assignment) and their sums are added in order.
template <class E>
__global__ void __launch_bounds__(1024) linear_sum_kernel(const float* part, const float* part_db, int splits, int64_t cells,
                                                          int64_t nq, E* out, E* db) {
    __shared__ float s[16][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t blocks = (cells + 255) / 256;
    const bool rows = blockIdx.x >= blocks;         // the workgroups behind those of dW sum db
    const float* src = rows ? part_db : part;
    const int64_t n = rows ? nq : cells;
    const int64_t i0 = (rows ? blockIdx.x - blocks : (int64_t)blockIdx.x) * 256 + 4 * lane;
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    if (n % 4 == 0) {
        if (i0 < n) {
#pragma unroll 4
            for (int k = wave; k < splits; k += 16) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(src + (int64_t)k * n + i0);
#pragma unroll
                for (int j = 0; j < 4; j++) t[j] += v[j];
            }
        }
    } else {
        for (int k = wave; k < splits; k += 16)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i0 + j < n) t[j] += src[(int64_t)k * n + i0 + j];
    }
#pragma unroll
    for (int j = 0; j < 4; j++) s[wave][4 * lane + j] = t[j];
    __syncthreads();
    if (threadIdx.x < 256) {
        const int64_t i = i0 - 4 * lane + threadIdx.x;
        if (i < n) {
            float v = 0.f;
            for (int k = 0; k < 16; k++) v += s[k][threadIdx.x];
            (rows ? db : out)[i] = (E)v;
        }
    }
}

// dz = dy act'(z), contiguous.
template <class E>
__global__ void __launch_bounds__(256) act_backward_kernel(const E* dy, int64_t dy_stride, const E* z, E* dz, int64_t rows,
                                                           int n, int act, int vec) {
    typedef E V8 __attribute__((ext_vector_type(8)));
    const int chunks = (n + 7) / 8;
    const int64_t total = rows * chunks;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / chunks;
        const int c = (int)(i - row * chunks) * 8;
        const E* a = dy + row * dy_stride + c;
        const E* b = z + row * n + c;
        E* o = dz + row * n + c;
        if (vec) {
            const V8 g = *reinterpret_cast<const V8*>(a), v = *reinterpret_cast<const V8*>(b);
            V8 r;
#pragma unroll
            for (int j = 0; j < 8; j++) r[j] = (E)((float)g[j] * slope_of((float)v[j], act));
            *reinterpret_cast<V8*>(o) = r;
        } else {
            for (int j = 0; j < 8 && c + j < n; j++) o[j] = (E)((float)a[j] * slope_of((float)b[j], act));
        }
    }
}
#endif

// ---- launch ---------------------------------------------------------------------------------------------------
// Sizes of a product: q rows, p columns, contraction.
struct LinPlan {
    int bp, bq, ke;
    int splits;
    int64_t k_per_split, tiles;
    int tiles_p;
};

// Tiles of 128 x 128 when they fill the chip, of 64 x 64 otherwise.
static LinPlan plan_product(int64_t nq, int np, int64_t nk, bool split, int elem_bytes, int cus) {
    LinPlan pl;
    pl.ke = 128 / elem_bytes;
    auto count = [&](int b) { return ((nq + b - 1) / b) * ((np + b - 1) / b); };
    const bool big = count(128) >= cus || (split && nq > 64 && np > 64);
    pl.bp = pl.bq = big ? 128 : 64;
    pl.tiles_p = (np + pl.bp - 1) / pl.bp;
    pl.tiles = count(pl.bp);
    pl.splits = 1;
    const int64_t stages = (nk + pl.ke - 1) / pl.ke;
    if (split) {
        // two workgroups per CU, and at least 4 stages each
        int64_t s = (2 * (int64_t)cus + pl.tiles - 1) / pl.tiles;
        if (s > stages / 4) s = stages / 4;
        if (s > 1) pl.splits = (int)s;
    }
    const int64_t per = (stages + pl.splits - 1) / pl.splits;
    pl.k_per_split = per * pl.ke;
    pl.splits = (int)((stages + per - 1) / per);
    return pl;
}

template <int DT, bool PT, bool QT>
static void launch_product(LinArgs a, const LinPlan& pl, bool vec, hipStream_t st) {
    a.tiles = pl.tiles; a.tiles_p = pl.tiles_p; a.splits = pl.splits; a.k_per_split = pl.k_per_split;
    const int64_t total = pl.tiles * pl.splits;
    const dim3 grid((unsigned)(8 * ((total + 7) / 8))), block(256);
    if (pl.bp == 128) {
        if (vec) hipLaunchKernelGGL((linear_kernel<DT, PT, QT, 128, 128, 2, 2, 128, 2, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((linear_kernel<DT, PT, QT, 128, 128, 2, 2, 128, 2, false>), grid, block, 0, st, a);
    } else {
        if (vec) hipLaunchKernelGGL((linear_kernel<DT, PT, QT, 64, 64, 2, 2, 128, 3, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((linear_kernel<DT, PT, QT, 64, 64, 2, 2, 128, 2, false>), grid, block, 0, st, a);
    }
}

static inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// rows of `bytes`-sized elements on 16-byte boundaries, whole chunks
static inline bool rows16(const void* p, int64_t stride, int64_t len, int bytes) {
    return al16(p) && stride * bytes % 16 == 0 && len * bytes % 16 == 0;
}

static LinArgs forward_args(const fwa2_linear* p) {
    const int xb = p->x_dtype == FWA2_E4M3 ? 1 : 2;
    LinArgs a = {};
    a.q = reinterpret_cast<const char*>(p->x); a.q_stride = p->x_stride * xb;
    a.p = reinterpret_cast<const char*>(p->weight); a.p_stride = p->weight_stride * xb;
    a.nq = p->rows; a.np = p->out_features; a.nk = p->in_features;
    a.out = p->y; a.z = p->z; a.bias = p->bias; a.act = p->activation;
    a.residual = reinterpret_cast<const char*>(p->residual); a.residual_stride = p->residual_stride * 2;
    a.q_scale = p->x_scale; a.p_scale = p->weight_scale;
    a.out_bf16 = p->dtype == FWA2_BF16;
    a.out_vec = p->out_features % 8 == 0 && al16(p->y) && al16(p->z) && (!p->residual || rows16(p->residual, p->residual_stride, 8, 2));
    return a;
}

#if FWA2_HALF == 3
void linear_forward_e4m3(const fwa2_linear* p, int cus, hipStream_t st) {
    const bool vec = rows16(p->x, p->x_stride, p->in_features, 1) && rows16(p->weight, p->weight_stride, p->in_features, 1);
    launch_product<FWA2_E4M3, false, false>(forward_args(p), plan_product(p->rows, p->out_features, p->in_features, false, 1, cus), vec, st);
}
#else
#if FWA2_HALF == 1
#define FWA2_LIN_DT FWA2_BF16
#define FWA2_LIN_FN(name) name##_bf16
#else
#define FWA2_LIN_DT FWA2_F16
#define FWA2_LIN_FN(name) name##_f16
#endif
void FWA2_LIN_FN(linear_forward)(const fwa2_linear* p, int cus, hipStream_t st) {
    const bool vec = rows16(p->x, p->x_stride, p->in_features, 2) && rows16(p->weight, p->weight_stride, p->in_features, 2);
    launch_product<FWA2_LIN_DT, false, false>(forward_args(p), plan_product(p->rows, p->out_features, p->in_features, false, 2, cus), vec, st);
}
void FWA2_LIN_FN(linear_backward)(const fwa2_linear* p, int cus, hipStream_t st) {
    typedef Elem<FWA2_LIN_DT>::E E;
    const int64_t m = p->rows;
    const int n = p->out_features, k = p->in_features;
    const char* dz = reinterpret_cast<const char*>(p->dy);
    int64_t dz_stride = p->dy_stride;
    char* ws = reinterpret_cast<char*>(p->workspace);
    if (p->activation != FWA2_ACT_NONE) {
        const int64_t chunks = m * ((n + 7) / 8);
        const int64_t blocks = (chunks + 255) / 256, most = 16 * (int64_t)cus;
        const int vec = rows16(p->dy, p->dy_stride, n, 2) && al16(p->z);
        hipLaunchKernelGGL(act_backward_kernel<E>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st,
                           reinterpret_cast<const E*>(p->dy), p->dy_stride, reinterpret_cast<const E*>(p->z),
                           reinterpret_cast<E*>(ws), m, n, p->activation, vec);
        dz = ws;
        dz_stride = n;
        ws += ((size_t)m * n * 2 + 255) / 256 * 256;
    }
    const bool vec = rows16(dz, dz_stride, n, 2);
    if (p->dx != nullptr) {
        LinArgs a = {};
        a.q = dz; a.q_stride = dz_stride * 2;
        a.p = reinterpret_cast<const char*>(p->weight); a.p_stride = p->weight_stride * 2;
        a.nq = m; a.np = k; a.nk = n;
        a.out = p->dx;
        a.out_vec = k % 8 == 0 && al16(p->dx);
        launch_product<FWA2_LIN_DT, true, false>(a, plan_product(m, k, n, false, 2, cus),
                                                 vec && rows16(p->weight, p->weight_stride, k, 2), st);
    }
    if (p->dweight != nullptr) {
        LinArgs a = {};
        a.q = dz; a.q_stride = dz_stride * 2;
        a.p = reinterpret_cast<const char*>(p->x); a.p_stride = p->x_stride * 2;
        a.nq = n; a.np = k; a.nk = m;
        a.out = p->dweight; a.db = p->dbias;
        a.out_vec = k % 8 == 0 && al16(p->dweight);
        const LinPlan pl = plan_product(n, k, m, true, 2, cus);
        const int64_t cells = (int64_t)n * k;
        a.part = reinterpret_cast<float*>(ws);
        a.part_db = a.part + (int64_t)pl.splits * cells;
        launch_product<FWA2_LIN_DT, true, true>(a, pl, vec && rows16(p->x, p->x_stride, k, 2), st);
        if (pl.splits > 1) {
            const int64_t blocks = (cells + 255) / 256 + (p->dbias ? (n + 255) / 256 : 0);
            hipLaunchKernelGGL(linear_sum_kernel<E>, dim3((unsigned)blocks), dim3(1024), 0, st, a.part, a.part_db, pl.splits,
                               cells, (int64_t)n, reinterpret_cast<E*>(p->dweight), reinterpret_cast<E*>(p->dbias));
        }
    }
}
#endif

#if FWA2_HALF == 1
void linear_forward_f16(const fwa2_linear* p, int cus, hipStream_t st);
void linear_backward_f16(const fwa2_linear* p, int cus, hipStream_t st);
void linear_forward_e4m3(const fwa2_linear* p, int cus, hipStream_t st);

size_t linear_workspace_bytes(const fwa2_linear* p, bool backward, int cus) {
    if (!backward) return 0;
    size_t need = p->activation != FWA2_ACT_NONE ? ((size_t)p->rows * p->out_features * 2 + 255) / 256 * 256 : 0;
    if (p->dweight != nullptr) {
        const LinPlan pl = plan_product(p->out_features, p->in_features, p->rows, true, 2, cus);
        if (pl.splits > 1) need += (size_t)pl.splits * p->out_features * ((size_t)p->in_features + 1) * sizeof(float);
    }
    return need;
}

// Whether every launch of the call has a grid that fits.
bool linear_fits(const fwa2_linear* p) {
    const double m = p->rows / 64.0 + 1, n = p->out_features / 64.0 + 1, k = p->in_features / 64.0 + 1;
    return m * n < 8e6 && m * k < 8e6 && n * k < 8e6;
}

hipError_t launch_linear_forward(const fwa2_linear* p, int cus, hipStream_t st) {
    if (p->x_dtype == FWA2_E4M3) linear_forward_e4m3(p, cus, st);
    else if (p->dtype == FWA2_BF16) linear_forward_bf16(p, cus, st);
    else linear_forward_f16(p, cus, st);
    return hipGetLastError();
}
hipError_t launch_linear_backward(const fwa2_linear* p, int cus, hipStream_t st) {
    if (p->dtype == FWA2_BF16) linear_backward_bf16(p, cus, st);
    else linear_backward_f16(p, cus, st);
    return hipGetLastError();
}
#endif

}  // namespace fwa2
