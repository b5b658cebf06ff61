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
//
// What bounds it, measured on MI355X kernel by kernel under a profiler, two sets of inputs in turn.  Short contractions:
// memory.  262144 x 96 -> 384 with GELU 66 us for 252 MB (3.8 TB/s; a large copy reaches 5.1, and the stores queue behind a
// tile's loads); 65536 x 768 -> 192 with a residual 34 us (4.4 TB/s).  Long ones: the matrix pipe.  8192 x 4096 -> 4096 bf16
// 258 us = 1 066 TFLOP/s (back to back without the profiler 246; the library's plain product of that size 205), 8-bit 139 to
// 147 us, up to 1 980 TFLOP/s; the pipe is busy 59 % and 51 % of these.  Between the two every product of a training step sits
// near both limits: 16384 x 384 -> 1536, forward with z 40 us (2.8 TB/s), dx 29 us, dW 34 + 10 us.
#include <initializer_list>
#include <type_traits>

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
    uint32_t tiles, tiles_p;      // output tiles, and those of a row of tiles
    uint32_t splits;              // of the contraction
    uint64_t by_tiles, by_tiles_p;    // ceil(2^40 / divisor): workgroup indices stay below 2^23
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
    int stream_out;               // non-temporal stores (stream_results)
    int out_bf16;                 // 8-bit products: element type of the output
};

// What the hardware reads where a tile reaches over the end of the contraction.
static __device__ __attribute__((aligned(16))) const uint32_t k_zeros[4] = {0, 0, 0, 0};

template <int DT> struct LinElem { static constexpr int bytes = 2; };
template <> struct LinElem<FWA2_E4M3> { static constexpr int bytes = 1; };

// ---- activations -------------------------------------------------------------------------------------------
// Upper tail Q(u) = 1 - Phi(u) of the normal distribution for u >= 0.  log2 Q is so smooth that a polynomial of degree 7 (a
// minimax fit over [0, 6], weighted by (u + 0.35) Q(u), value at 0 fixed) gives Q to 8e-7 absolutely and 5e-5 relatively
// over the fit, and falls on beyond it (6e-16 at 8, 0 from 20 on, where u is cut so that infinity meets a zero).  Eight
// instructions and one exponential: the library's erff takes about 40, which in the epilogue of a product with few
// contraction elements (262144 x 96 -> 384) are 130 us of vector instructions next to 49 us of memory traffic; the whole
// kernel now takes 66.
__device__ __forceinline__ float normal_tail(float u) {
    float p = -1.1775869097618852e-06f;
    p = __builtin_fmaf(p, u, 4.9426900659454986e-05f);
    p = __builtin_fmaf(p, u, -0.0008448792505078018f);
    p = __builtin_fmaf(p, u, 0.008222263306379318f);
    p = __builtin_fmaf(p, u, -0.053498417139053345f);
    p = __builtin_fmaf(p, u, -0.4588005840778351f);
    p = __builtin_fmaf(p, u, -1.151161789894104f);
    p = __builtin_fmaf(p, u, -1.0f);
    return fast_exp2(p);
}
// z Phi(z) = max(z, 0) - u Q(u) with u = |z|, the maximum as (z + |z|) / 2 so that NaN and infinity pass through
__device__ __forceinline__ float gelu_of(float z) {
    const float u = fminf(fabsf(z), 20.f);
    return __builtin_fmaf(0.5f, z + fabsf(z), -u * normal_tail(u));
}
__device__ __forceinline__ float sigmoid_of(float x) { return fast_rcp(1.f + fast_exp2(-kLog2e * x)); }
constexpr float kTanhA = 1.5957691216057308f;       // 2 sqrt(2 / pi): z / 2 (1 + tanh(u)) = z sigmoid(2 u)
constexpr float kTanhB = 0.07135481282553505f;      // 0.044715 times that

__device__ __forceinline__ float act_of(float z, int act) {
    switch (act) {
        case FWA2_ACT_GELU: return gelu_of(z);
        case FWA2_ACT_GELU_TANH: return z * sigmoid_of(z * (kTanhA + kTanhB * z * z));
        case FWA2_ACT_SILU: return z * sigmoid_of(z);
        case FWA2_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
        default: return z;
    }
}
// 8 values; ACT < 0: the decision is taken here, once
template <int ACT>
__device__ __forceinline__ void act8(float* v, int act) {
    if (ACT >= 0) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = act_of(v[j], ACT);
    } else if (act == FWA2_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = act_of(v[j], FWA2_ACT_GELU);
    } else if (act == FWA2_ACT_GELU_TANH) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = act_of(v[j], FWA2_ACT_GELU_TANH);
    } else if (act == FWA2_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = act_of(v[j], FWA2_ACT_SILU);
    } else if (act == FWA2_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = act_of(v[j], FWA2_ACT_RELU);
    }
}
// d act / dz.  Beyond |z| = 100 every slope is 0 or 1 to fp32, and z (kept in 16 bits, possibly overflowed to infinity) must
// not meet a zero factor; NaN stays NaN (the comparison is false).
__device__ __forceinline__ float slope_of(float z, int act) {
    if (fabsf(z) > 100.f) z = copysignf(100.f, z);
    switch (act) {
        case FWA2_ACT_GELU: {       // Phi(z) + z phi(z)
            const float q = normal_tail(fminf(fabsf(z), 20.f));
            const float phi = fast_exp2(-0.72134752044448170f * z * z) * 0.3989422804014327f;
            return __builtin_fmaf(z, phi, z > 0.f ? 1.f - q : q);
        }
        case FWA2_ACT_GELU_TANH: {
            const float z2 = z * z;
            const float s = sigmoid_of(z * (kTanhA + kTanhB * z2));
            return s + z * s * (1.f - s) * (kTanhA + 3.f * kTanhB * z2);
        }
        case FWA2_ACT_SILU: {
            const float s = sigmoid_of(z);
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

// Chunk permutation of a memory row in LDS.  Plain rows of KB = 64 (128) bytes: four (two) rows share the 256 bytes that the
// banks span, and an operand read serves rows {0-3, 12-15, 20-27} (then the other 16) of one chunk at a time.
template <int KB>
__device__ __forceinline__ int plain_swizzle(int row) { return KB == 64 ? (row >> 2) & 3 : (row >> 1) & 7; }
// Transposed rows of R columns: a read serves 4 contraction rows with 64 bytes (4 chunks) each.  Rows of a multiple of 256
// bytes all start on the same bank; of an odd multiple of 128, every second one does.
template <int R>
__device__ __forceinline__ int turned_swizzle(int k) { return R % 128 == 0 ? 4 * (k & 3) : 4 * ((k >> 1) & 1); }

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

    // LDS rows of a copy; 0: copies end inside rows (192 transposed columns: 24 chunks a row)
    static constexpr int RPC = 64 % CPR == 0 ? 64 / CPR : 0;
    // the swizzles look at bits 0 .. 3 of a row, and the copies of a wavefront lie a multiple of that apart
    static_assert(RPC == 0 || NW * RPC % (TURNED ? 4 : 16) == 0, "");

    const char* base;       // uniform: first row (column) of the tile, first contraction element of the split
    int64_t stride;
    int64_t step;           // bytes from stage to stage
    uint32_t off[NI];       // of this lane's chunk of each copy
    int rows;               // rows (columns) of the tile inside the matrix
    int row0, chunk0;       // of this lane's part of copy 0 (place)
    int wave, lane;

    static __device__ __forceinline__ int swizzled(int row, int c) { return c ^ (TURNED ? turned_swizzle<R>(row) : plain_swizzle<KB>(row)); }
    // LDS row of this lane's part of copy i, and the memory chunk that belongs there
    __device__ __forceinline__ void place(int i, int& row, int& chunk) const {
        if (RPC > 0) {
            row = row0 + i * NW * RPC;
            chunk = chunk0;
        } else {
            const int ci = (i * NW + wave) * 64 + lane;
            row = ci / CPR;
            chunk = swizzled(row, ci - row * CPR);
        }
    }

    // Rows (columns) beyond the matrix repeat the last ones: what they produce is not stored.
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
        row0 = wave * RPC + lane / CPR;
        chunk0 = swizzled(row0, lane % CPR);
#pragma unroll
        for (int i = 0; i < NI; i++) {
            int r, chunk;
            place(i, r, chunk);
            if (TURNED) off[i] = (uint32_t)r * (uint32_t)stride + (uint32_t)(chunk * CE < rows ? chunk * 16 : rows * EB - 16);
            else off[i] = (uint32_t)(r < rows ? r : rows - 1) * (uint32_t)stride + (uint32_t)chunk * 16;
        }
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
                int row, chunk;
                place(i, row, chunk);
                const bool in = TURNED ? row < left : chunk * CE < left;
                const void* src = in ? (const void*)(at + off[i]) : (const void*)k_zeros;
                tile_dma(src, dst + i * NW * 1024);
            }
        }
    }
    // The same through registers, for rows off 16-byte boundaries and extents that end inside a chunk.
    __device__ __forceinline__ void fetch(int64_t kt, int left, u32x4* r) const {
        const char* at = base + kt * step;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            int at_row, chunk;
            place(i, at_row, chunk);
            int n;              // elements of the chunk inside the matrix
            const char* src;
            if (TURNED) {
                n = at_row < left ? rows - chunk * CE : 0;
                src = at + (int64_t)at_row * stride + chunk * 16;
            } else {
                n = left - chunk * CE;
                src = at + (int64_t)(at_row < rows ? at_row : rows - 1) * stride + chunk * 16;
            }
            r[i] = u32x4{0, 0, 0, 0};
            if (n >= CE) {
                __builtin_memcpy(&r[i], src, 16);
            } else if (n > 0) {
                // from clamped places: all loads under way at once, where a test per element would wait for each
                uint32_t e[CE];
#pragma unroll
                for (int j = 0; j < CE; j++) {
                    const int at_j = min(j, n - 1);
                    if (EB == 2) e[j] = reinterpret_cast<const uint16_t*>(src)[at_j];
                    else e[j] = reinterpret_cast<const uint8_t*>(src)[at_j];
                }
#pragma unroll
                for (int j = 0; j < CE; j++) {
                    const int bit = j * EB * 8;
                    r[i][bit / 32] |= (j < n ? e[j] : 0u) << (bit % 32);
                }
            }
        }
    }
    __device__ __forceinline__ void put(const u32x4* r, char* lds) const {
#pragma unroll
        for (int i = 0; i < NI; i++) *reinterpret_cast<u32x4*>(lds + ((i * NW + wave) * 64 + lane) * 16) = r[i];
    }
};

// MFMA operands of 32 rows out of a staged tile: lane (row = lane % 32, half = lane / 32).  Which contraction elements a lane
// holds does not matter as long as both operands agree.
template <int DT> struct Frag {             // v_mfma_f32_32x32x16
    typedef typename Elem<DT>::V8 V;
    static constexpr int BYTES = 32;        // of a row per product
    template <int KB>
    static __device__ __forceinline__ V plain(const char* tile, int row, int swz, int half, int s) {
        return *reinterpret_cast<const V*>(tile + row * KB + (((2 * s + half) ^ swz) * 16));
    }
    template <int R>
    static __device__ __forceinline__ V turned(const char* tile, int t32, int lane, int s) {
        const int i = lane & 15, g = lane >> 4;
        const int k = 16 * s + 8 * (g >> 1) + (i >> 2);
        const int chunk = (4 * t32 + 2 * (g & 1) + ((i & 3) >> 1)) ^ turned_swizzle<R>(k);
        typedef typename Elem<DT>::E E;
        const E* lo = reinterpret_cast<const E*>(tile + k * R * 2 + chunk * 16 + (i & 1) * 8);
        return lds_tr8<DT>(lo, lo + 4 * R);
    }
    static __device__ __forceinline__ f32x16 mfma(V a, V b, f32x16 c) { return Elem<DT>::mfma32(a, b, c); }
};
typedef int i32x8 __attribute__((ext_vector_type(8)));
template <> struct Frag<FWA2_E4M3> {        // v_mfma_f32_32x32x64
    typedef i32x8 V;
    static constexpr int BYTES = 64;
    template <int KB>
    static __device__ __forceinline__ V plain(const char* tile, int row, int swz, int half, int s) {
        const u32x4 a = *reinterpret_cast<const u32x4*>(tile + row * KB + (((4 * s + half) ^ swz) * 16));
        const u32x4 b = *reinterpret_cast<const u32x4*>(tile + row * KB + (((4 * s + 2 + half) ^ swz) * 16));
        V v;
#pragma unroll
        for (int i = 0; i < 4; i++) { v[i] = (int)a[i]; v[4 + i] = (int)b[i]; }
        return v;
    }
    template <int R>
    static __device__ __forceinline__ V turned(const char*, int, int, int) { return V{}; }
    // The 8-bit unit adds products in groups of 8 contraction elements aligned to the group's largest and drops what lies
    // below 2^-13 of that (measured, for the 16x16x128 form as for the 16x16x32 one); the groups are added in fp32.  Against
    // the 2^-4 half steps of the operands that is nothing, and the alternative, converting the tiles to 16 bits for
    // the exact products of the other unit, halves the matrix rate.
    // 0x7f: a block scale of 2^0 in every byte
    static __device__ __forceinline__ f32x16 mfma(V a, V b, f32x16 c) {
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
    }
};

// Which tile a workgroup computes.  Workgroups go to the 8 XCDs in turn, each with an L2 of its own: consecutive tiles are
// given to one XCD, column tiles first, so that the tiles that share a block of Q rows meet in one L2.
__device__ __forceinline__ uint32_t tile_of_block(uint32_t block, uint32_t total) {
    const uint32_t per = (total + 7) / 8;
    return (block & 7) * per + (block >> 3);
}
// n / d for n < 2^23, d < 2^17, from ceil(2^40 / d): the excess of the quotient is below n d / 2^40 / d < 1 / d
__device__ __forceinline__ uint32_t divide(uint32_t n, uint64_t by) { return (uint32_t)((n * by) >> 40); }

// The values as fp32 numbers of their own: what follows must not be folded into the arithmetic before it.  (The compiler
// turns a multiply-add and its conversion to fp16 into one instruction with one rounding in some forms of the epilogue and
// not in others; a call with and one without gradients would then differ in the last bit.)
__device__ __forceinline__ void settle8(float* v) {
#pragma unroll
    for (int j = 0; j < 8; j++) asm("" : "+v"(v[j]));
}

// N bias values from column p on.  Columns beyond the last repeat it (their results are not stored): no branch, and with
// whole groups (np a multiple of 8, bias aligned) one load.
template <class OT, int N>
__device__ __forceinline__ void load_bias(const LinArgs& a, int p, float* b) {
    typedef OT VN __attribute__((ext_vector_type(N)));
    const OT* src = reinterpret_cast<const OT*>(a.bias);
    if (a.out_vec) {
        const VN v = *reinterpret_cast<const VN*>(src + min(p, a.np - N));
#pragma unroll
        for (int j = 0; j < N; j++) b[j] = (float)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) b[j] = (float)src[min(p + j, a.np - 1)];
    }
}

// Where 16-byte chunk c of row q of a wavefront's 32 x TP block of results lies in LDS: rows of TP floats, chunks permuted so
// that neither the writes (one chunk of 16 rows at a time) nor the reads (whole rows) pile up on a bank.
template <int TP>
__device__ __forceinline__ int result_chunk(int q, int c) {
    const int x = TP == 32 ? (q >> 1) & 7 : TP % 64 == 0 ? q & 15 : q & 7;
    return q * (TP / 4) + (c ^ x);
}

// The results of a wavefront: acc (rows of 32, 4 consecutive columns of 32 different rows per lane) changes hands through
// `mine` (32 x TP floats of LDS that only this wavefront uses), so that TP / 8 neighbouring lanes hold whole stretches of a
// row, and residual, z and result move in full cache lines: stored as they are, 32 rows would get 32 bytes each.
template <int TP>
struct Results {
    static constexpr int LPR = TP / 8;             // lanes of a row
    static constexpr int RPI = 64 / LPR;           // rows per instruction (TP = 96: 5, and four lanes idle)
    static constexpr int NR = (32 + RPI - 1) / RPI;
    char* mine;
    int l32, half, rl, cl;

    __device__ __forceinline__ void init(char* m, int lane) {
        mine = m;
        l32 = lane & 31;
        half = lane >> 5;
        rl = lane / LPR;
        cl = lane - rl * LPR;
    }
    template <int FP>
    __device__ __forceinline__ void put(const f32x16 (&acc)[FP]) const {
#pragma unroll
        for (int j = 0; j < FP; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const f32x4 v = {acc[j][4 * r], acc[j][4 * r + 1], acc[j][4 * r + 2], acc[j][4 * r + 3]};
                *reinterpret_cast<f32x4*>(mine + 16 * result_chunk<TP>(l32, 8 * j + 2 * r + half)) = v;
            }
        asm volatile("" ::: "memory");      // a wavefront's LDS accesses stay in order
    }
    __device__ __forceinline__ void get(int row, float* v) const {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(mine + 16 * result_chunk<TP>(row, 2 * cl));
        const f32x4 hi = *reinterpret_cast<const f32x4*>(mine + 16 * result_chunk<TP>(row, 2 * cl + 1));
#pragma unroll
        for (int e = 0; e < 4; e++) { v[e] = lo[e]; v[4 + e] = hi[e]; }
    }
};

// bias, and before it the scales of an 8-bit product
template <int DT, class OT>
struct Columns {
    float bias[8], ps[8];
    __device__ __forceinline__ void init(const LinArgs& a, int p) {
#pragma unroll
        for (int e = 0; e < 8; e++) bias[e] = 0.f;
        if (a.bias != nullptr) load_bias<OT, 8>(a, p, bias);
        if constexpr (DT == FWA2_E4M3) {
#pragma unroll
            for (int e = 0; e < 8; e++) ps[e] = a.p_scale[min(p + e, a.np - 1)];
        }
    }
    __device__ __forceinline__ void apply(const LinArgs& a, float* v, int64_t q) const {
        if constexpr (DT == FWA2_E4M3) {
            const float qs = a.q_scale[q];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = v[e] * (qs * ps[e]) + bias[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += bias[e];
        }
    }
};

// Epilogue of a wavefront's TQ x TP block with its first row at qw, first column at pw; output rows take 16-byte accesses (np
// is a multiple of 8: a lane's 8 columns are inside or outside together).
// Buffer accesses: rows beyond the last lie outside the buffer's size, lanes outside the columns are sent there, and the
// hardware drops such stores and returns zeros for such loads; no branches, and all rows in one stretch of code.  A
// wavefront's rows span less than 2^31 bytes (row strides are below 2^22 elements).
template <int DT, class OT, int TP, int TQ, int ACT, int FQ, int FP>
__device__ __forceinline__ void store_results(const LinArgs& a, const Results<TP>& r, f32x16 (&acc)[FQ][FP], int64_t qw, int pw) {
    typedef OT V8 __attribute__((ext_vector_type(8)));
    constexpr int RPI = Results<TP>::RPI, NR = Results<TP>::NR;
    const int p = pw + 8 * r.cl;
    const bool inside = r.rl < RPI && p < a.np;
    Columns<DT, OT> columns;
    columns.init(a, p);
    const int rows = a.nq - qw < TQ ? (int)(a.nq - qw) : TQ;
    const bool any = rows > 0;
    auto buffer = [&](const void* base, int64_t row_bytes) __attribute__((always_inline)) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(uniform_pointer(reinterpret_cast<const char*>(base) + qw * row_bytes)), 0,
                                                 any ? (int)(rows * row_bytes) : 0, 0x00027000);
    };
    const auto out_rows = buffer(a.out, (int64_t)a.np * 2);
    const uint32_t out_step = (uint32_t)a.np * 2, res_step = (uint32_t)a.residual_stride;
    const uint32_t out_at = inside ? (uint32_t)r.rl * out_step + (uint32_t)p * 2 : 0x80000000u;
    const uint32_t from = inside ? (uint32_t)r.rl * res_step + (uint32_t)p * 2 : 0x80000000u;
    auto body = [&](auto has_residual, auto has_z, auto stream) __attribute__((always_inline)) {
        constexpr int policy = decltype(stream)::value ? kStreamPolicy : 0;
        const auto res_rows = buffer(a.residual, has_residual ? a.residual_stride : 0);
        const auto z_rows = buffer(a.z, has_z ? (int64_t)a.np * 2 : 0);
#pragma unroll
        for (int i = 0; i < FQ; i++) {
            u32x4 res[NR];
            if (has_residual) {
#pragma unroll
                for (int k = 0; k < NR; k++)
                    res[k] = __builtin_amdgcn_raw_buffer_load_b128(res_rows, from + (32 * i + k * RPI) * res_step, 0, 0);
            }
            r.put(acc[i]);
#pragma unroll
            for (int k = 0; k < NR; k++) {
                const uint32_t skip = 32 % RPI != 0 && k * RPI + r.rl >= 32 ? 0x80000000u : 0u;
                float v[8];
                r.get(32 % RPI == 0 ? k * RPI + r.rl : min(k * RPI + r.rl, 31), v);
                columns.apply(a, v, any ? qw + min(32 * i + k * RPI + r.rl, rows - 1) : 0);
                settle8(v);
                V8 t;
                if (has_z) {
#pragma unroll
                    for (int j = 0; j < 8; j++) t[j] = (OT)v[j];
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, t), z_rows, (out_at | skip) + (32 * i + k * RPI) * out_step, 0, policy);
                }
                act8<ACT>(v, a.act);
                settle8(v);
                if (has_residual) {
                    const V8 x = __builtin_bit_cast(V8, res[k]);
#pragma unroll
                    for (int j = 0; j < 8; j++) v[j] += (float)x[j];
                }
                settle8(v);
#pragma unroll
                for (int j = 0; j < 8; j++) t[j] = (OT)v[j];
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, t), out_rows, (out_at | skip) + (32 * i + k * RPI) * out_step, 0, policy);
            }
            asm volatile("" ::: "memory");
        }
    };
    const std::true_type yes;
    const std::false_type no;
    auto with_policy = [&](auto stream) __attribute__((always_inline)) {
        if (a.residual != nullptr) {
            if (ACT != FWA2_ACT_NONE && a.z != nullptr) body(yes, yes, stream);
            else body(yes, no, stream);
        } else {
            if (ACT != FWA2_ACT_NONE && a.z != nullptr) body(no, yes, stream);
            else body(no, no, stream);
        }
    };
    if (a.stream_out) with_policy(yes);
    else with_policy(no);
}

// ACT: the activation, or -1 where it is decided at run time.  WAVES: wavefronts per SIMD the registers are limited for.
template <int DT, bool PT, bool QT, int BP, int BQ, int WP, int WQ, int KB, int STAGES, bool VEC, int ACT, int WAVES>
__global__ void __launch_bounds__(64 * WP * WQ, WAVES) linear_kernel(const LinArgs a) {
    constexpr int NW = WP * WQ;
    constexpr int TP = BP / WP, TQ = BQ / WQ;       // a wavefront's part of the tile
    constexpr int FP = TP / 32, FQ = TQ / 32;
    static_assert(TP % 32 == 0 && TQ % 32 == 0 && STAGES >= 2, "");
    typedef Operand<DT, PT, BP, KB, NW, VEC> OP;
    typedef Operand<DT, QT, BQ, KB, NW, VEC> OQ;
    typedef Frag<DT> F;
    typedef typename F::V FV;
    constexpr int KE = OP::KE;
    constexpr int STEPS = KB / F::BYTES;         // products of a stage and 32 x 32 tile
    constexpr int STAGE = OP::BYTES + OQ::BYTES;
    constexpr int COPIES = OP::NI + OQ::NI;         // outstanding memory operations of a stage, per wavefront
    constexpr bool DB = PT && QT;
    typedef typename Elem<DT == FWA2_E4M3 ? FWA2_F16 : DT>::E E16;
    constexpr int RESULTS = NW * 32 * TP * 4;       // the results pass through the same memory afterwards
    __shared__ __attribute__((aligned(1024))) char lds[STAGES * STAGE > RESULTS ? STAGES * STAGE : RESULTS];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave % WP, wq = wave / WP;
    const int l32 = lane & 31, half = lane >> 5;

    const uint32_t total = a.tiles * a.splits;
    const uint32_t t = tile_of_block(blockIdx.x, total);
    if (t >= total) return;
    // split by split: the tiles that read the same stretch of the contraction run side by side
    const uint32_t split = a.splits > 1 ? divide(t, a.by_tiles) : 0;
    const uint32_t tile = t - split * a.tiles;
    const uint32_t tile_q = divide(tile, a.by_tiles_p);
    const int64_t q0 = (int64_t)tile_q * BQ;
    const int p0 = (int)(tile - tile_q * a.tiles_p) * BP;
    const int64_t k0 = split * a.k_per_split;
    const int64_t k1 = k0 + a.k_per_split < a.nk ? k0 + a.k_per_split : a.nk;
    const int64_t len = k1 - k0;
    const int64_t nkt = (len + KE - 1) / KE;
    auto left_of = [&](int64_t kt) { const int64_t l = len - kt * KE; return l < KE ? (int)l : KE; };

    OP P;
    OQ Q;
    P.init(a.p, a.p_stride, p0, a.np, k0, wave, lane);
    Q.init(a.q, a.q_stride, q0, a.nq, k0, wave, lane);

    f32x16 acc[FQ][FP];
#pragma unroll
    for (int i = 0; i < FQ; i++)
#pragma unroll
        for (int j = 0; j < FP; j++) acc[i][j] = f32x16{};
    float row_sums[DB ? FQ : 1];
#pragma unroll
    for (int i = 0; i < (DB ? FQ : 1); i++) row_sums[i] = 0.f;
    const bool sum_rows = DB && a.db != nullptr && p0 == 0 && wp == 0;

    const int swz = plain_swizzle<KB>(l32);
    auto load_p = [&](const char* buf, int s, int j) __attribute__((always_inline)) -> FV {
        if constexpr (PT) return F::template turned<BP>(buf, wp * FP + j, lane, s);
        else return F::template plain<KB>(buf, wp * TP + 32 * j + l32, swz, half, s);
    };
    auto load_q = [&](const char* buf, int s, int i) __attribute__((always_inline)) -> FV {
        if constexpr (QT) return F::template turned<BQ>(buf + OP::BYTES, wq * FQ + i, lane, s);
        else return F::template plain<KB>(buf + OP::BYTES, wq * TQ + 32 * i + l32, swz, half, s);
    };
    FV fp[FP], fq[FQ];
    auto load = [&](const char* buf, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FQ; i++) fq[i] = load_q(buf, s, i);
#pragma unroll
        for (int j = 0; j < FP; j++) fp[j] = load_p(buf, s, j);
    };
    auto add_rows = [&]() __attribute__((always_inline)) {
        if constexpr (DB) {
            if (sum_rows) {
#pragma unroll
                for (int i = 0; i < FQ; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) row_sums[DB ? i : 0] += (float)fq[i][e];
            }
        }
    };
    auto multiply = [&]() __attribute__((always_inline)) {
        add_rows();
#pragma unroll
        for (int j = 0; j < FP; j++)
#pragma unroll
            for (int i = 0; i < FQ; i++) acc[i][j] = F::mfma(fp[j], fq[i], acc[i][j]);
    };
    // The products of the operands in registers, each P operand replaced by step s of `buf` as soon as it has been used: the
    // LDS reads of a step run under the matrix work of the one before it.
    auto multiply_and_load = [&](const char* buf, int s) __attribute__((always_inline)) {
        add_rows();
        FV qn[FQ];
#pragma unroll
        for (int i = 0; i < FQ; i++) qn[i] = load_q(buf, s, i);
#pragma unroll
        for (int j = 0; j < FP; j++) {
#pragma unroll
            for (int i = 0; i < FQ; i++) acc[i][j] = F::mfma(fp[j], fq[i], acc[i][j]);
            fp[j] = load_p(buf, s, j);
        }
#pragma unroll
        for (int i = 0; i < FQ; i++) fq[i] = qn[i];
    };

    if constexpr (VEC) {
        auto issue = [&](int64_t kt, char* buf) __attribute__((always_inline)) {
            P.issue(kt, left_of(kt), buf);
            Q.issue(kt, left_of(kt), buf + OP::BYTES);
        };
#pragma unroll
        for (int s = 0; s < STAGES; s++)
            if (s < nkt) issue(s, lds + s * STAGE);
        if (nkt >= STAGES) wait_vm<(STAGES - 1) * COPIES>();
        else wait_vm<0>();
        lds_barrier();
        load(lds, 0);
        char* cur = lds;
        for (int64_t kt = 0; kt + 1 < nkt; kt++) {
            char* next = cur + STAGE == lds + STAGES * STAGE ? lds : cur + STAGE;
#pragma unroll
            for (int s = 1; s < STEPS; s++) multiply_and_load(cur, s);
            // stage kt + 1 has landed when at most the copies of the later stages are still out ...
            if (kt + STAGES <= nkt) wait_vm<(STAGES - 2) * COPIES>();
            else wait_vm<0>();
            lds_barrier();      // ... for every wavefront, and all hold the rest of stage kt in registers: its place is free
            if (kt + STAGES < nkt) issue(kt + STAGES, cur);
            multiply_and_load(next, 0);
            cur = next;
        }
#pragma unroll
        for (int s = 1; s < STEPS; s++) multiply_and_load(cur, s);
        multiply();
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
            load(buf, 0);
#pragma unroll
            for (int s = 1; s < STEPS; s++) multiply_and_load(buf, s);
            multiply();
        }
    }

    if constexpr (DB) {
        if (sum_rows) {
#pragma unroll
            for (int i = 0; i < FQ; i++) {
                const float t = xor32_add(row_sums[DB ? i : 0]);
                const int64_t q = q0 + wq * TQ + 32 * i + l32;
                if (half == 0 && q < a.nq) {
                    if (a.splits > 1) a.part_db[(int64_t)split * a.nq + q] = t;
                    else reinterpret_cast<E16*>(a.db)[q] = (E16)t;
                }
            }
        }
    }
    lds_barrier();          // nobody reads operands any more: their memory takes the results
    typedef Results<TP> RS;
    RS r;
    r.init(lds + wave * 32 * TP * 4, lane);
    const int64_t qw = q0 + wq * TQ;        // uniform: first row of this wavefront
    const int pw = p0 + wp * TP, p = pw + 8 * r.cl;
    // Is row r0 + rl of the 32 this lane's business?  (q: the uniform part of its index in the output)
    auto mine_row = [&](int r0, int64_t q) __attribute__((always_inline)) {
        return r.rl < RS::RPI && p < a.np && (32 % RS::RPI == 0 || r0 + r.rl < 32) && q + r.rl < a.nq;
    };
    const uint32_t at = (uint32_t)r.rl * (uint32_t)a.np + (uint32_t)p;
    if (a.splits > 1) {
        float* out = a.part + (int64_t)split * a.nq * a.np;
        const bool whole = a.np % 8 == 0;
#pragma unroll
        for (int i = 0; i < FQ; i++) {
            r.put(acc[i]);
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += RS::RPI) {
                const int64_t q = qw + 32 * i + r0;
                if (!mine_row(r0, q)) continue;
                float v[8];
                r.get(r0 + r.rl, v);
                float* o = out + q * a.np + at;
                if (whole) {
                    *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
                    *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (p + e < a.np) o[e] = v[e];
                }
            }
            asm volatile("" ::: "memory");
        }
        return;
    }
    auto finish = [&](auto tag) __attribute__((always_inline)) {
        typedef decltype(tag) OT;
        typedef OT V8 __attribute__((ext_vector_type(8)));
        if (a.out_vec) {
            store_results<DT, OT, TP, TQ, ACT>(a, r, acc, qw, pw);
            return;
        }
        Columns<DT, OT> columns;
        columns.init(a, p);
        const uint32_t res_at = (uint32_t)r.rl * (uint32_t)(a.residual_stride / 2) + (uint32_t)p;
#pragma unroll
        for (int i = 0; i < FQ; i++) {
            r.put(acc[i]);
#pragma unroll 1
            for (int r0 = 0; r0 < 32; r0 += RS::RPI) {
                const int64_t q = qw + 32 * i + r0;
                if (!mine_row(r0, q)) continue;
                float v[8];
                r.get(r0 + r.rl, v);
                columns.apply(a, v, q + r.rl);
                settle8(v);
                const int n = a.np - p;
                V8 res, t;
                if (a.residual != nullptr) {
                    const OT* src = reinterpret_cast<const OT*>(a.residual + q * a.residual_stride) + res_at;
                    if (n >= 8) __builtin_memcpy(&res, src, 16);
                    else
#pragma unroll
                        for (int j = 0; j < 8; j++) res[j] = src[min(j, n - 1)];
                }
                auto store = [&](OT* to) __attribute__((always_inline)) {
#pragma unroll
                    for (int j = 0; j < 8; j++) t[j] = (OT)v[j];
                    if (n >= 8) __builtin_memcpy(to, &t, 16);
                    else
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (j < n) to[j] = t[j];
                };
                if (a.z != nullptr) store(reinterpret_cast<OT*>(a.z) + q * a.np + at);
                act8<ACT>(v, a.act);
                settle8(v);
                if (a.residual != nullptr) {
#pragma unroll
                    for (int j = 0; j < 8; j++) v[j] += (float)res[j];
                }
                settle8(v);
                store(reinterpret_cast<OT*>(a.out) + q * a.np + at);
            }
            asm volatile("" ::: "memory");
        }
    };
    if constexpr (DT == FWA2_E4M3) {
        if (a.out_bf16) finish((__bf16)0.f);
        else finish((_Float16)0.f);
    } else {
        finish((E16)0.f);
    }
}

// ---- few rows ---------------------------------------------------------------------------------------------------
// Single tokens, a pooled image: the call reads the weights once and is over; what counts is how soon every load is on its
// way.  A workgroup owns 16 output columns of 16 MQ rows and its wavefronts split the contraction; operands go from memory
// straight into the registers of 16-row products (no staging, no barrier until the end), partial sums meet in LDS and are
// added in a fixed order.  Its limit is that every workgroup gathers its rows of x anew (takes_rows has the figures).
template <int DT> struct Frag16 {           // v_mfma_f32_16x16x32
    typedef typename Elem<DT>::V8 V;
    static constexpr int BYTES = 64;        // of a row per product
    static __device__ __forceinline__ V load(const char* row, int64_t at, int64_t left, int g) {
        // beyond the end: the start of the row is read and zeros are used (a select, where a branch would wait)
        const V v = *reinterpret_cast<const V*>(row + (16 * g < left ? at + 16 * g : 0));
        return 16 * g < left ? v : zero8<V>();
    }
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) { return Elem<DT>::mfma16(a, b, c); }
};
template <> struct Frag16<FWA2_E4M3> {      // v_mfma_f32_16x16x128
    typedef i32x8 V;
    static constexpr int BYTES = 128;
    static __device__ __forceinline__ V load(const char* row, int64_t at, int64_t left, int g) {
        const bool in_a = 16 * g < left, in_b = 64 + 16 * g < left;
        const u32x4 a = *reinterpret_cast<const u32x4*>(row + (in_a ? at + 16 * g : 0));
        const u32x4 b = *reinterpret_cast<const u32x4*>(row + (in_b ? at + 64 + 16 * g : 0));
        V v;
#pragma unroll
        for (int i = 0; i < 4; i++) { v[i] = in_a ? (int)a[i] : 0; v[4 + i] = in_b ? (int)b[i] : 0; }
        return v;
    }
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
    }
};
constexpr int kRowsWaves = 8;

template <int DT, int MQ>       // MQ: groups of 16 rows
__global__ void __launch_bounds__(64 * kRowsWaves) linear_rows_kernel(const LinArgs a) {
    typedef Frag16<DT> F;
    constexpr int EB = LinElem<DT>::bytes, U = MQ == 1 ? 8 : 4;
    __shared__ float sums[kRowsWaves][MQ][16][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int l16 = lane & 15, g = lane >> 4;
    const int p0 = blockIdx.x * 16, q0 = blockIdx.y * (16 * MQ);
    const char* prow = a.p + (int64_t)min(p0 + l16, a.np - 1) * a.p_stride;
    const char* qrow[MQ];
#pragma unroll
    for (int i = 0; i < MQ; i++) qrow[i] = a.q + (int64_t)min(q0 + 16 * i + l16, (int)a.nq - 1) * a.q_stride;
    f32x4 acc[MQ];
#pragma unroll
    for (int i = 0; i < MQ; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // what the epilogue needs besides the sums is asked for first: value t of this thread is (row, column)
    // (t / 16, t % 16) of the workgroup's, t = threadIdx.x + k blockDim.x with at least 256 threads
    typedef typename std::conditional<DT == FWA2_E4M3, uint16_t, typename Elem<DT == FWA2_E4M3 ? FWA2_F16 : DT>::E>::type RT;
    RT bias = {}, res[MQ];
    float p_scale = 1.f, q_scale[MQ];
    const int p = min(p0 + (int)(threadIdx.x & 15), a.np - 1);
    if (a.bias != nullptr) bias = reinterpret_cast<const RT*>(a.bias)[p];
    if (DT == FWA2_E4M3) p_scale = a.p_scale[p];
#pragma unroll
    for (int k = 0; k < MQ; k++) {
        const int q = min(q0 + ((int)(threadIdx.x + k * blockDim.x) >> 4), (int)a.nq - 1);
        res[k] = {};
        q_scale[k] = 1.f;
        if (a.residual != nullptr) res[k] = reinterpret_cast<const RT*>(a.residual + q * a.residual_stride)[p];
        if (DT == FWA2_E4M3) q_scale[k] = a.q_scale[q];
    }
    const int64_t bytes = a.nk * EB;
    const int64_t steps = (bytes + F::BYTES - 1) / F::BYTES;
    // every `waves`-th product is this wavefront's: neighbouring wavefronts read neighbouring stretches
    for (int64_t s = wave; s < steps; s += (int64_t)waves * U) {
        typename F::V fp[U], fq[U][MQ];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t at = (s + (int64_t)u * waves) * F::BYTES;     // beyond the end: zeros
            fp[u] = F::load(prow, at, bytes - at, g);
#pragma unroll
            for (int i = 0; i < MQ; i++) fq[u][i] = F::load(qrow[i], at, bytes - at, g);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < MQ; i++) acc[i] = F::mfma(fp[u], fq[u][i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < MQ; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) sums[wave][i][l16][4 * g + r] = acc[i][r];      // [row][column]
    __syncthreads();
    auto finish = [&](auto tag) __attribute__((always_inline)) {
        typedef decltype(tag) OT;
#pragma unroll
        for (int k = 0; k < MQ; k++) {
            const int t = threadIdx.x + k * blockDim.x, q = t >> 4;
            if (t >= MQ * 256 || q0 + q >= a.nq || p0 + (t & 15) >= a.np) continue;
            float v = 0.f;
            for (int w = 0; w < waves; w++) v += sums[w][q >> 4][q & 15][t & 15];
            const float b = (float)__builtin_bit_cast(OT, bias);
            if constexpr (DT == FWA2_E4M3) v = v * (q_scale[k] * p_scale) + b;
            else v += b;
            asm("" : "+v"(v));
            const int64_t at = (int64_t)(q0 + q) * a.np + p;
            if (a.z != nullptr) reinterpret_cast<OT*>(a.z)[at] = (OT)v;
            v = act_of(v, a.act);
            asm("" : "+v"(v));
            if (a.residual != nullptr) v += (float)__builtin_bit_cast(OT, res[k]);
            asm("" : "+v"(v));
            reinterpret_cast<OT*>(a.out)[at] = (OT)v;
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
// dW, db = sums of partial rows, rounded once.  A workgroup owns 256 values of dW (64 of db: there are few and each has many
// partials); its W wavefronts take every W-th partial (a fixed assignment) and their sums are added in order.
// (16 wavefronts for many partials, 4 for few.)
template <class E, int W>
__global__ void __launch_bounds__(64 * W) linear_sum_kernel(const float* part, int parts, const float* part_db, int parts_db,
                                                          int64_t cells, int nq, E* out, E* db) {
    __shared__ float s[W][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t blocks = (cells + 255) / 256;
    if (blockIdx.x >= blocks) {         // the workgroups behind those of dW sum db
        const int i = (int)(blockIdx.x - blocks) * 64 + lane;
        const float* src = part_db + min(i, nq - 1);
        float t = 0.f;
#pragma unroll 8
        for (int k = wave; k < parts_db; k += W) t += src[(int64_t)k * nq];
        s[wave][lane] = t;
        __syncthreads();
        if (threadIdx.x < 64 && i < nq) {
            t = 0.f;
            for (int k = 0; k < W; k++) t += s[k][lane];
            db[i] = (E)t;
        }
        return;
    }
    const int64_t i0 = (int64_t)blockIdx.x * 256 + 4 * lane;
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    if (cells % 4 == 0) {
        if (i0 < cells) {
#pragma unroll 8
            for (int k = wave; k < parts; k += W) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(part + (int64_t)k * cells + i0);
#pragma unroll
                for (int j = 0; j < 4; j++) t[j] += v[j];
            }
        }
    } else {
        // (values beyond the last repeat it, so that the loads need no branch)
#pragma unroll 4
        for (int k = wave; k < parts; k += W)
#pragma unroll
            for (int j = 0; j < 4; j++) t[j] += part[(int64_t)k * cells + (i0 + j < cells ? i0 + j : cells - 1)];
    }
#pragma unroll
    for (int j = 0; j < 4; j++) s[wave][4 * lane + j] = t[j];
    __syncthreads();
    if (threadIdx.x < 256) {
        const int64_t i = i0 - 4 * lane + threadIdx.x;
        if (i < cells) {
            float v = 0.f;
            for (int k = 0; k < W; k++) v += s[k][threadIdx.x];
            out[i] = (E)v;
        }
    }
}

// dz = dy act'(z), contiguous, and the column sums of dz before its rounding (part_db, one partial row per blockIdx.y).
// A workgroup owns up to 512 columns (8 per lane, `lanes` lanes a row, a power of two) and a stretch of rows; bound by its
// three streams (16384 x 1536: 32 us, 4.7 TB/s).
//
// dz leaves in the element type because it is an operand of the matrix products behind, which take 16 bits: with the
// result's own rounding dx and dW are then 0.0024 off in bf16 (2-norm, 16384 x 384 -> 1536 with GELU), where sums of unrounded
// dz rounded once would be 0.0017 off.  z is kept in it too: in 32 bits it would move 100 MB more beside that case's 243.
constexpr int kActRows = 256;      // at most so many stretches of rows: their partial sums stay small
template <class E, int ACT, bool VEC>
__global__ void __launch_bounds__(256) act_backward_kernel(const E* dy, int64_t dy_stride, const E* z, E* dz, int64_t rows,
                                                           int n, int lanes, int64_t rows_per_block, float* part_db) {
    typedef E V8 __attribute__((ext_vector_type(8)));
    __shared__ float sums[256][9];
    const int cl = threadIdx.x % lanes, rl = threadIdx.x / lanes, step = 256 / lanes;
    const int c = (blockIdx.x * lanes + cl) * 8;
    const int64_t r0 = blockIdx.y * rows_per_block, r1 = r0 + rows_per_block < rows ? r0 + rows_per_block : rows;
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; j++) t[j] = 0.f;
    if (c < n) {
#pragma unroll 4
        for (int64_t row = r0 + rl; row < r1; row += step) {
            const E* a = dy + row * dy_stride + c;
            const E* b = z + row * n + c;
            E* o = dz + row * n + c;
            if (VEC) {
                const V8 g = *reinterpret_cast<const V8*>(a), v = *reinterpret_cast<const V8*>(b);
                V8 r;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    float d = (float)g[j] * slope_of((float)v[j], ACT);
                    t[j] += d;
                    r[j] = (E)d;
                }
                *reinterpret_cast<V8*>(o) = r;
            } else {
                V8 g, v, r;
                if (c + 8 <= n) {       // whole chunks in one access of whatever alignment the rows have
                    __builtin_memcpy(&g, a, 16);
                    __builtin_memcpy(&v, b, 16);
                } else {                // the last one element by element, from clamped places
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        g[j] = a[min(j, n - 1 - c)];
                        v[j] = b[min(j, n - 1 - c)];
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float d = (float)g[j] * slope_of((float)v[j], ACT);
                    t[j] += d;
                    r[j] = (E)d;
                }
                if (c + 8 <= n) {
                    __builtin_memcpy(o, &r, 16);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (c + j < n) o[j] = r[j];
                }
            }
        }
    }
    if (part_db == nullptr) return;
#pragma unroll
    for (int j = 0; j < 8; j++) sums[threadIdx.x][j] = t[j];
    __syncthreads();
    for (int i = threadIdx.x; i < lanes * 8; i += 256) {
        const int col = blockIdx.x * lanes * 8 + i;
        if (col >= n) continue;
        float v = 0.f;
        for (int k = 0; k < step; k++) v += sums[k * lanes + (i >> 3)][i & 7];
        part_db[(int64_t)blockIdx.y * n + col] = v;
    }
}
struct ActPlan {
    int lanes, blocks_x, blocks_y;
    int64_t rows_per_block;
};
static ActPlan plan_act(int64_t rows, int n, int cus) {
    ActPlan pl;
    const int chunks = (n + 7) / 8;
    pl.lanes = 1;
    while (pl.lanes < 64 && pl.lanes < chunks) pl.lanes *= 2;
    pl.blocks_x = (chunks + pl.lanes - 1) / pl.lanes;
    int64_t y = (8 * (int64_t)cus + pl.blocks_x - 1) / pl.blocks_x;
    if (y > kActRows) y = kActRows;
    const int64_t step = 4 * (256 / pl.lanes), most = (rows + step - 1) / step;     // at least 4 rows per lane
    if (y > most) y = most;
    pl.rows_per_block = (rows + y - 1) / y;
    pl.blocks_y = (int)((rows + pl.rows_per_block - 1) / pl.rows_per_block);
    return pl;
}
#endif

// ---- launch ---------------------------------------------------------------------------------------------------
// The tile a product runs on, and how its contraction is split.
enum Tile { T64, T128S, T128, T192P, T192Q, T192, T256, T256P };
struct TileShape {
    int bp, bq, kb, per_cu;     // columns, rows, bytes of the contraction per stage, resident workgroups of a CU
};
static constexpr TileShape kTiles[] = {
    {64, 64, 128, 3},     // T64:    too few output tiles of any other size to fill the chip; 3 stages, few waits per contraction
    {128, 128, 64, 4},    // T128S:  short contractions: loads and stores bound the call, many workgroups hide each other's
    {128, 128, 128, 2},   // T128
    {192, 128, 128, 2},   // T192P:  column counts that waste less of 192 than of 128 (and equal ones: fewer operand reads)
    {128, 192, 128, 2},   // T192Q:  the same for the rows; weight gradients only, as is
    {192, 192, 128, 1},   // T192:   both
    {256, 256, 128, 1},   // T256:   large products, 8 wavefronts: LDS reads per product fall with the tile's edge
    {256, 128, 64, 2},    // T256P:  contractions not quite as short: half as many tiles' first loads to wait for
};
struct LinPlan {
    Tile tile;
    int splits;
    int64_t k_per_split, tiles;
    int tiles_p;
};

// The rule, with what it was measured on (MI355X, us, bf16, launches back to back whose operands and results move through
// 1 GB, so that the caches hold none of them; rows x contraction -> columns):
//   262144 x   96 ->  384 gelu       T128S  85, T128  92, T192P  91, T256 109, T256P  94, T64 133
//    65536 x  192 ->  768 gelu, z    T128S  64, T128  69,                      T256P  59
//    65536 x  192 ->  768 (dx)       T128S  42, T128  44,                      T256P  39
//    16384 x  384 -> 1536 gelu, z    T128S  42, T128  36, T192P  37, T256  46,           T64  49
//    16384 x 1536 ->  384 (dx)       T128S  35, T128  30, T192P  30, T256  42,           T64  41
//    65536 x  768 ->  192 residual   T128S  54, T128  40, T192P  32, T256  34,           T64  52
//     4096 x  768 -> 1536 gelu, z    T128S  24, T128  21, T192P  22,                     T64  26
//     4096 x 1536 ->  768 residual   T128S  31, T128  26, T192P  29,                     T64  23     (T192P: half the CUs)
//    16384 x  384 ->  384            T128S  14, T128  12, T192P  12,                     T64  15
//    16384 x  384 ->   96 residual   T128S  11, T128  10, T192P  11,                     T64   7
//     2048 x 1024 -> 1024            T128S  17, T128  13,                                T64  10
//      512 x 4096 -> 1024            T128S  56, T128  42,                                T64  24
//     8192 x 4096 -> 4096 residual   T128S 378, T128 313, T192P 286, T256 238,           T64 593
// T256P on both sides of its borders (T128S or T128, whichever the rule would take / T256P; forward with gelu and z, dx):
//   contraction, 65536 rows, 768 columns:  88: 47 / 46, 28 / 24    96: 49 / 45, 30 / 24   104: 54 / 48, 34 / 27
//                                         192: 64 / 59, 42 / 39   200: 75 / 66, 51 / 43   208: 75 / 65, 51 / 43
//   workgroups, contraction 192:          192: 9.4 / 9.8, 9.1 / 9.7    384: 14 / 14, 13 / 14   (one row of tiles short of) 512:
//                                         19 / 15, 18 / 18   513: 19 / 22, 19 / 20   768: 25 / 24, 24 / 23   1023: 34 / 29, 32 / 28
//   columns, 65536 rows:                  256: 22 / 17   384: 26 / 27 (a third of its tiles' columns empty)   512: 31 / 27
// so it would pay from 88 to 208 elements as well; below two workgroups to a CU it does not.
// weight gradients (rows of dW x rows of the batch -> columns of dW), splits chosen as below, without the sum behind:
//      384 x 262144 ->  96           T128  56, T192Q  51, T192P  57, T192  56
//     1536 x  16384 -> 384           T128  41, T192Q  34, T192P  37, T192  36
//      192 x  65536 -> 768           T128  51, T192Q  37, T192P  40, T192  43
//     4096 x   8192 -> 4096          T128 332, T192Q 306, T192P 314, T192 314, T256 225
static LinPlan plan_product(int64_t nq, int np, int64_t nk, bool split, int elem_bytes, int cus) {
    auto up = [](int64_t n, int b) { return (n + b - 1) / b; };
    auto count = [&](Tile t) { return up(nq, kTiles[t].bq) * up(np, kTiles[t].bp); };
    auto wide = [&](int64_t n) { return up(n, 192) * 192 <= up(n, 128) * 128; };     // 192 wastes no more than 128
    LinPlan pl;
    const int64_t big = count(T256), rounds = up(big, cus);
    const bool small = nq <= 64 || np <= 64;
    if (!small && big >= cus && big * 10 >= rounds * cus * 8 && nk * elem_bytes >= 1024 &&
        (double)nq * np >= 0.8 * big * 256 * 256) {
        pl.tile = T256;             // whole rounds of full tiles and a contraction that hides the ends
    } else if (split) {
        pl.tile = small ? T64 : wide(np) && np > 128 ? (wide(nq) && nq > 128 ? T192 : T192P) : (wide(nq) && nq > 128 ? T192Q : T128);
    } else if (small || count(T128) * 10 < 6 * cus) {
        pl.tile = T64;
    } else if (nk * elem_bytes <= 384) {
        const bool whole = up(np, 256) * 2 <= up(np, 128) && count(T256P) >= 2 * cus;
        pl.tile = nk * elem_bytes > 192 && whole ? T256P : T128S;
    } else {
        pl.tile = wide(np) && np > 128 && count(T192P) >= cus ? T192P : T128;
    }
    const TileShape& sh = kTiles[pl.tile];
    const int ke = sh.kb / elem_bytes;
    pl.tiles_p = (int)up(np, sh.bp);
    pl.tiles = count(pl.tile);
    const int64_t stages = up(nk, ke);
    int64_t s = 1;
    if (split && pl.tile != T256) {
        // one round of workgroups (64-wide tiles: two), each with at least 4 stages
        s = (pl.tile == T64 ? 2 : 1) * (int64_t)cus * (pl.tile == T192P || pl.tile == T192Q ? 2 : 1) / pl.tiles;
        if (s > stages / 4) s = stages / 4;
        if (s < 1) s = 1;
    }
    const int64_t per = up(stages, (int)s);
    pl.k_per_split = per * ke;
    pl.splits = (int)up(stages, (int)per);
    return pl;
}

static uint64_t reciprocal40(uint32_t d) { return ((1ull << 40) + d - 1) / d; }

template <int DT, bool PT, bool QT, int ACT>
static void launch_product(LinArgs a, const LinPlan& pl, bool vec, hipStream_t st) {
    a.tiles = (uint32_t)pl.tiles; a.tiles_p = pl.tiles_p; a.splits = pl.splits; a.k_per_split = pl.k_per_split;
    a.by_tiles = reciprocal40(a.tiles); a.by_tiles_p = reciprocal40(a.tiles_p);
    const int64_t total = pl.tiles * pl.splits;
    const dim3 grid((unsigned)(8 * ((total + 7) / 8)));
    constexpr bool TURNED = PT && QT;
#define FWA2_GO(BP, BQ, WP, WQ, KB, ST, WAVES) \
    hipLaunchKernelGGL((linear_kernel<DT, PT, QT, BP, BQ, WP, WQ, KB, ST, true, ACT, WAVES>), grid, dim3(64 * WP * WQ), 0, st, a)
    if (!vec) {
        // rows off 16-byte boundaries: through registers, on two tile sizes
        if (kTiles[pl.tile].bp == 64) hipLaunchKernelGGL((linear_kernel<DT, PT, QT, 64, 64, 2, 2, 64, 2, false, -1, 1>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((linear_kernel<DT, PT, QT, 128, 128, 2, 2, 64, 2, false, -1, 1>), grid, dim3(256), 0, st, a);
        return;
    }
    switch (pl.tile) {
        case T64: FWA2_GO(64, 64, 2, 2, 128, 3, 3); break;
        case T128S:
            if constexpr (!TURNED) FWA2_GO(128, 128, 2, 2, 64, 2, 3);
            break;
        case T128: FWA2_GO(128, 128, 2, 2, 128, 2, 2); break;
        case T192P: FWA2_GO(192, 128, 2, 2, 128, 2, 2); break;
        case T192Q:
            if constexpr (TURNED) FWA2_GO(128, 192, 2, 2, 128, 2, 2);
            break;
        case T192:
            if constexpr (TURNED) FWA2_GO(192, 192, 2, 2, 128, 2, 1);
            break;
        case T256: FWA2_GO(256, 256, 2, 4, 128, 2, 2); break;
        case T256P:
            if constexpr (!TURNED) FWA2_GO(256, 128, 2, 2, 64, 2, 2);
            break;
    }
#undef FWA2_GO
}

// Which products linear_rows_kernel takes: up to 16 rows, and any number whose workgroups find a CU each; beyond that the
// gathering of x costs more than the 64 x 64 tiles' stages, one after the other, do.  Measured (bf16, us, tiles / this
// kernel, launches back to back with weights that the caches do not hold):
//     1 x  768 ->  1536   9.2 / 5.0      64 x  768 -> 1536   6.8 /  4.7      256 x 1536 ->  384  10.8 /  6.8
//     1 x 4096 ->  4096  28.3 / 9.1      64 x 4096 -> 1024  26.8 / 10.8      128 x 4096 -> 1024  27.1 / 14.7
//     1 x 1024 -> 16384  10.1 / 8.4      16 x 1024 -> 16384 11.0 / 11.5       16 x  384 -> 8192   4.7 /  4.3
// and beyond the rule:                   32 x 1024 -> 16384 11.0 / 16.1      256 x  768 -> 1536   6.8 /  9.4
//                                        64 x 4096 ->  4096 28.8 / 26.0      128 x 4096 -> 4096  29.1 / 46.6
static bool takes_rows(int64_t nq, int np, int cus) {
    return nq <= 16 || ((nq + 31) / 32) * (int64_t)((np + 15) / 16) <= cus;
}
// 16 rows to a workgroup while there is a CU for each, 32 otherwise (64 x 4096 -> 1024: 10.9 / 14.5 us; -> 4096: 32.8 / 25.8);
// 8 wavefronts, 4 where there are many workgroups (1 x 1024 -> 16384: 8.4 us with 4, 9.9 with 8; 1 x 4096 -> 4096: 12.0 / 9.1).
template <int DT>
static void launch_rows(const LinArgs& a, int cus, hipStream_t st) {
    const int64_t columns = (a.np + 15) / 16, groups = (a.nq + 15) / 16;
    const dim3 block(64 * (columns > 2 * cus ? 4 : kRowsWaves));
    if (a.nq <= 16 || columns * groups <= cus) hipLaunchKernelGGL((linear_rows_kernel<DT, 1>), dim3(columns, groups), block, 0, st, a);
    else hipLaunchKernelGGL((linear_rows_kernel<DT, 2>), dim3(columns, (groups + 1) / 2), block, 0, st, a);
}

// The activations a product is compiled for; the others are decided at run time, row by row of the epilogue.  The form without
// an activation writes no z, which is then the same as y but for the residual: who asks for it gets the run-time form.
template <int DT>
static void launch_forward(const LinArgs& a, const LinPlan& pl, bool vec, int cus, hipStream_t st) {
    if (vec && takes_rows(a.nq, a.np, cus)) {
        launch_rows<DT>(a, cus, st);
        return;
    }
    if (a.act == FWA2_ACT_NONE && a.z == nullptr) launch_product<DT, false, false, FWA2_ACT_NONE>(a, pl, vec, st);
    else if (a.act == FWA2_ACT_GELU) launch_product<DT, false, false, FWA2_ACT_GELU>(a, pl, vec, st);
    else launch_product<DT, false, false, -1>(a, pl, vec, st);
}

// Tiles for operands that go through registers: 128 wide when those fill the chip twice (their loads are waited for stage by
// stage, so there have to be several workgroups to a CU), 64 otherwise.  Measured (us, 64 / 128 wide, operands not in the
// caches): 1225 x 588 -> 333 13.9 / 18.9 and its weight gradient 11.3 / 13.4; 4099 x 585 -> 1161 27.1 / 23.7, 43.4 / 51.0;
// 16389 x 585 -> 1161 96.7 / 64.2.
static LinPlan plan_unaligned(int64_t nq, int np, int64_t nk, bool split, int elem_bytes, int cus) {
    LinPlan pl;
    auto count = [&](int b) { return ((nq + b - 1) / b) * ((np + b - 1) / b); };
    pl.tile = count(128) >= 2 * cus ? T128S : T64;
    const int b = kTiles[pl.tile].bp;
    pl.tiles_p = (np + b - 1) / b;
    pl.tiles = count(b);
    const int64_t ke = 64 / elem_bytes, stages = (nk + ke - 1) / ke;
    int64_t s = split ? 4 * (int64_t)cus / pl.tiles : 1;
    if (s > stages / 4) s = stages / 4;
    if (s < 1) s = 1;
    const int64_t per = (stages + s - 1) / s;
    pl.k_per_split = per * ke;
    pl.splits = (int)((stages + per - 1) / per);
    return pl;
}
static LinPlan plan(int64_t nq, int np, int64_t nk, bool split, int elem_bytes, int cus, bool vec) {
    return vec ? plan_product(nq, np, nk, split, elem_bytes, cus) : plan_unaligned(nq, np, nk, split, elem_bytes, cus);
}

static inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// rows of `bytes`-sized elements on 16-byte boundaries, whole chunks
static inline bool rows16(const void* p, int64_t stride, int64_t len, int bytes) {
    return al16(p) && stride * bytes % 16 == 0 && len * bytes % 16 == 0;
}

// Results too large to be found in the 256 MB memory-side cache by whoever reads them next leave with non-temporal stores: plain
// ones fill the L2s with lines that wait to be written back, behind which the operands of the next tiles queue.  Measured
// (us, plain / non-temporal), with two sets of operands in turn, which the cache keeps where the results do not push them out,
// and with operands that no cache holds: 262144 x 96 -> 384 with GELU 90 / 73 and 90 / 85, without 75 / 45 and 77 / 73;
// 65536 x 192 -> 768 38 / 34 and 41 / 40, with GELU and z 59 / 51 and 62 / 60; 16384 x 384 -> 1536 with both 37 / 36 and
// 43 / 38.  An MLP whose second product reads the 201 MB of the first: 178 / 184 forward, but 804 / 762 forward and backward.
static bool stream_results(int64_t rows, int columns, bool z) { return (double)rows * columns * (z ? 4 : 2) >= (64 << 20); }

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
    a.stream_out = stream_results(p->rows, p->out_features, p->z != nullptr);
    a.out_vec = p->out_features % 8 == 0 && al16(p->y) && al16(p->z) && al16(p->bias) && (!p->residual || rows16(p->residual, p->residual_stride, 8, 2));
    return a;
}

#if FWA2_HALF == 3
void linear_forward_e4m3(const fwa2_linear* p, int cus, hipStream_t st) {
    const bool vec = rows16(p->x, p->x_stride, p->in_features, 1) && rows16(p->weight, p->weight_stride, p->in_features, 1);
    launch_forward<FWA2_E4M3>(forward_args(p), plan(p->rows, p->out_features, p->in_features, false, 1, cus, vec), vec, cus, st);
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
    launch_forward<FWA2_LIN_DT>(forward_args(p), plan(p->rows, p->out_features, p->in_features, false, 2, cus, vec), vec, cus, st);
}
static size_t dz_bytes(int64_t m, int n) { return ((size_t)m * n * 2 + 255) / 256 * 256; }
static size_t act_bytes(const fwa2_linear* p, int cus) {
    if (p->activation == FWA2_ACT_NONE || p->dbias == nullptr) return 0;
    return ((size_t)plan_act(p->rows, p->out_features, cus).blocks_y * p->out_features * sizeof(float) + 255) / 256 * 256;
}
void FWA2_LIN_FN(linear_backward)(const fwa2_linear* p, int cus, hipStream_t st) {
    typedef Elem<FWA2_LIN_DT>::E E;
    const int64_t m = p->rows;
    const int n = p->out_features, k = p->in_features;
    const char* dz = reinterpret_cast<const char*>(p->dy);
    int64_t dz_stride = p->dy_stride;
    char* ws = reinterpret_cast<char*>(p->workspace);
    float* part_act = nullptr;      // of dbias, from the unrounded dz
    ActPlan act = {};
    if (p->activation != FWA2_ACT_NONE) {
        act = plan_act(m, n, cus);
        if (p->dbias != nullptr) part_act = reinterpret_cast<float*>(ws + dz_bytes(m, n));
        const dim3 grid(act.blocks_x, act.blocks_y), block(256);
        const bool vec = rows16(p->dy, p->dy_stride, n, 2) && al16(p->z);
        const E *dy = reinterpret_cast<const E*>(p->dy), *z = reinterpret_cast<const E*>(p->z);
#define FWA2_GO(ACT, VEC) hipLaunchKernelGGL((act_backward_kernel<E, ACT, VEC>), grid, block, 0, st, dy, p->dy_stride, z, \
                                             reinterpret_cast<E*>(ws), m, n, act.lanes, act.rows_per_block, part_act)
        auto go = [&](auto aligned) {
            constexpr bool VEC = decltype(aligned)::value;
            if (p->activation == FWA2_ACT_GELU) FWA2_GO(FWA2_ACT_GELU, VEC);
            else if (p->activation == FWA2_ACT_GELU_TANH) FWA2_GO(FWA2_ACT_GELU_TANH, VEC);
            else if (p->activation == FWA2_ACT_SILU) FWA2_GO(FWA2_ACT_SILU, VEC);
            else FWA2_GO(FWA2_ACT_RELU, VEC);
        };
        if (vec) go(std::true_type());
        else go(std::false_type());
#undef FWA2_GO
        dz = ws;
        dz_stride = n;
        ws += dz_bytes(m, n) + act_bytes(p, cus);
    }
    const bool dz_vec = rows16(dz, dz_stride, n, 2);
    if (p->dx != nullptr) {
        LinArgs a = {};
        a.q = dz; a.q_stride = dz_stride * 2;
        a.p = reinterpret_cast<const char*>(p->weight); a.p_stride = p->weight_stride * 2;
        a.nq = m; a.np = k; a.nk = n;
        a.out = p->dx;
        a.stream_out = stream_results(m, k, false);
        a.out_vec = k % 8 == 0 && al16(p->dx);
        const bool vec = dz_vec && rows16(p->weight, p->weight_stride, k, 2);
        launch_product<FWA2_LIN_DT, true, false, FWA2_ACT_NONE>(a, plan(m, k, n, false, 2, cus, vec), vec, st);
    }
    if (p->dweight != nullptr) {
        LinArgs a = {};
        a.q = dz; a.q_stride = dz_stride * 2;
        a.p = reinterpret_cast<const char*>(p->x); a.p_stride = p->x_stride * 2;
        a.nq = n; a.np = k; a.nk = m;
        a.out = p->dweight;
        a.db = part_act ? nullptr : p->dbias;
        a.out_vec = k % 8 == 0 && al16(p->dweight);
        const bool vec = dz_vec && rows16(p->x, p->x_stride, k, 2);
        const LinPlan pl = plan(n, k, m, true, 2, cus, vec);
        const int64_t cells = (int64_t)n * k;
        a.part = reinterpret_cast<float*>(ws);
        a.part_db = a.part + (int64_t)pl.splits * cells;
        launch_product<FWA2_LIN_DT, true, true, FWA2_ACT_NONE>(a, pl, vec, st);
        const int64_t summed = pl.splits > 1 ? cells : 0;
        const bool sum_db = p->dbias != nullptr && (part_act || pl.splits > 1);
        if (summed || sum_db) {
            const int64_t blocks = (summed + 255) / 256 + (sum_db ? (n + 63) / 64 : 0);
            const float* part_db = part_act ? part_act : a.part_db;
            const int parts_db = part_act ? act.blocks_y : pl.splits;
            E *dw = reinterpret_cast<E*>(p->dweight), *db = reinterpret_cast<E*>(p->dbias);
            if (pl.splits > 32 || !summed)
                hipLaunchKernelGGL((linear_sum_kernel<E, 16>), dim3((unsigned)blocks), dim3(1024), 0, st, a.part, pl.splits, part_db, parts_db, summed, n, dw, db);
            else
                hipLaunchKernelGGL((linear_sum_kernel<E, 4>), dim3((unsigned)blocks), dim3(256), 0, st, a.part, pl.splits, part_db, parts_db, summed, n, dw, db);
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
    size_t need = p->activation != FWA2_ACT_NONE ? dz_bytes(p->rows, p->out_features) + act_bytes(p, cus) : 0;
    if (p->dweight != nullptr) {
        // whichever way the operands turn out to be read
        int splits = 1;
        for (bool vec : {false, true}) {
            const LinPlan pl = plan(p->out_features, p->in_features, p->rows, true, 2, cus, vec);
            if (pl.splits > splits) splits = pl.splits;
        }
        if (splits > 1) need += (size_t)splits * p->out_features * ((size_t)p->in_features + 1) * sizeof(float);
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
