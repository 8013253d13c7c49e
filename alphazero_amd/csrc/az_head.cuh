// Loss of a linear layer over many classes, with its gradient, without ever holding the logits (az_linear_ce_*).
//
//   z = x W^T + b            [rows, classes]
//   lse_i = log sum_j exp z_ij,  p_ij = exp(z_ij - lse_i),  H_i = lse_i - sum_j p_ij z_ij
//   L_i = T_i lse_i - sum_j pi_ij z_ij - c H_i,   T_i = sum_j pi_ij   (an index target is pi = one at that class)
//   G_ij = dL_i/dz_ij = T_i p_ij - pi_ij + c p_ij (log p_ij + H_i)
//   dx = G W,  dW = G^T x,  db_j = sum_i G_ij
//
// Forward: one product whose tiles end in a few sums per row (Part), joined per row by a second kernel. Backward: the classes in pieces;
// per piece the logits are made again, turned into G (16 bits, in both orientations), and two products take it to dx and dW. Bound
// by the matrix instructions: 2 N V D forward, 6 N V D backward. 8192 rows, 4096 features, 131072 classes, bfloat16: logits and their
// sums 6.5 to 6.9 ms by card (1.35 PFLOP/s), G 7.4 to 7.7 ms (of which 0.9 ms are its 4.3 GB), dx and dW 13.1 to 13.3 ms (1.35 PFLOP/s),
// copies of W^T 0.4 ms (5.3 TB/s), joining 0.03 ms.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/azamd.h"
#include "az_gemm.cuh"
#include "az_types.cuh"

namespace az {
int fail(int code, const std::string& msg);

// One translation unit per element type (az_head_f32.hip, az_head_bf16.hip, az_head_f16.hip): they take half a minute each to compile.
#define AZ_HEAD_TYPE(NAME)                                                                                                                   \
    int ce_forward_##NAME(const az_linear_ce_args&, float* kept, float* loss, float* ce, float* ent, char* ws, hipStream_t);                  \
    int ce_backward_##NAME(const az_linear_ce_args&, const float* kept, const float* grad, void* gx, void* gw, void* gb, char* ws, hipStream_t);
AZ_HEAD_TYPE(f32)
AZ_HEAD_TYPE(bf16)
AZ_HEAD_TYPE(f16)
#undef AZ_HEAD_TYPE

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// ------------------------------------------------------------------------------------------------ operands
__device__ __forceinline__ float larger(float top, float v) { return v > top || v != v ? v : top; }      // a NaN stays

// Copies a [rows, cols] matrix (any row stride, any alignment) into rows of `pitch` bytes, zeros behind the last column. float32 is
// scaled by a power of two, each row by its own (its reciprocal goes to `own`), and split into two planes. Rows that do not count become
// zeros. Bound by memory; only operands that the tile loop cannot read in place come here (float32, rows that do not start at
// multiples of 16 bytes).
struct PackJob {
    const void* src;
    int64_t src_pitch;    // elements
    int32_t rows, cols;
    char* dst;
    int64_t pitch, plane;   // bytes
    float* own;             // float32
    const int64_t* target;  // null: every row counts
    int64_t ignore;
    // Lanes of a row that is scaled by itself: as many as it has pieces, up to a wave, or a workgroup from 4096 columns on (forward pass of
    // 64 x 64 -> 131000: 51 us, with a wave for each row 101; of 64 x 65536 -> 64: 78 against 180).
    __host__ __device__ int lanes() const { return pitch <= 128 ? 8 : pitch <= 256 ? 16 : pitch <= 512 ? 32 : pitch < 8192 ? 64 : 256; }
    __host__ __device__ int64_t blocks() const { return own ? (rows + 256 / lanes() - 1) / (256 / lanes()) : (rows * (pitch >> 4) + 255) / 256; }
    __device__ __forceinline__ bool counts(int64_t r) const { return !(target && target[r] == ignore); }
};

// Eight neighbours from element `at` on, `left` of them in the row (the others zero). They may start anywhere.
__device__ __forceinline__ void load8(const float* src, int64_t at, int left, float (&v)[8]) {
    if (left >= 8) __builtin_memcpy(v, src + at, 32);
    else
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? src[at + e] : 0.0f;
}
// The same as 16-bit planes; float32 times `scale`.
template <int DT>
__device__ __forceinline__ void load_planes(const void* src, int64_t at, int left, float scale, uint16_t (&h)[2][8]) {
    if constexpr (DT == DT_F32) {
        float v[8];
        load8((const float*)src, at, left, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) split2(v[e] * scale, h[0][e], h[1][e]);
    } else {
        if (left >= 8) __builtin_memcpy(h[0], (const uint16_t*)src + at, 16);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) h[0][e] = e < left ? ((const uint16_t*)src)[at + e] : (uint16_t)0;
    }
}

template <int DT>
__device__ __forceinline__ void pack_block(const PackJob& j, int64_t block, float* tops) {
    constexpr int NP = DT == DT_F32 ? 2 : 1;
    const int pieces = (int)(j.pitch >> 4);
    __align__(16) uint16_t h[2][8];
    auto put = [&](int64_t r, int piece, float scale) {
        load_planes<DT>(j.src, r * j.src_pitch + piece * 8, j.counts(r) ? j.cols - piece * 8 : 0, scale, h);
#pragma unroll
        for (int p = 0; p < NP; ++p) *(uint4*)(j.dst + p * j.plane + r * j.pitch + piece * 16) = *(const uint4*)h[p];
    };
    if constexpr (DT == DT_F32) {
        const int lanes = j.lanes(), lane = threadIdx.x & (lanes - 1);
        const int64_t r = block * (256 / lanes) + threadIdx.x / lanes;
        if (r >= j.rows) return;
        const bool counts = j.counts(r);
        float first[8], top = 0.0f;        // a lane's first piece stays in registers, what a row has beyond comes again from L2
        load8((const float*)j.src, r * j.src_pitch + lane * 8, counts ? j.cols - lane * 8 : 0, first);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = larger(top, fabsf(first[e]));
        if (counts)
            for (int i = lane + lanes; i < pieces; i += lanes) {
                float v[8];
                load8((const float*)j.src, r * j.src_pitch + i * 8, j.cols - i * 8, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = larger(top, fabsf(v[e]));
            }
        for (int o = 1; o < 64 && o < lanes; o *= 2) top = larger(top, __shfl_xor(top, o));
        if (lanes == 256) {
            if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 4; ++w) top = larger(top, tops[w]);
        }
        const float un = unscale_of(top), scale = 1.0f / un;
        if (lane == 0) j.own[r] = un;
        if (lane < pieces) {
#pragma unroll
            for (int e = 0; e < 8; ++e) split2(first[e] * scale, h[0][e], h[1][e]);
#pragma unroll
            for (int p = 0; p < NP; ++p) *(uint4*)(j.dst + p * j.plane + r * j.pitch + lane * 16) = *(const uint4*)h[p];
        }
        for (int i = lane + lanes; i < pieces; i += lanes) put(r, i, scale);
    } else {
        const int64_t at = block * 256 + threadIdx.x;
        if (at < (int64_t)j.rows * pieces) put(at / pieces, (int)(at % pieces), 1.0f);
    }
}

// The same, transposed: dst row c = column c of the source, rows behind the last one (up to the pitch, a multiple of 128 bytes) zero. The
// products' sums run over the source's rows here, so all of float32 is divided by what the largest row is (`all`): every value keeps 22
// bits down to 2^-27 of the largest, and what is left above 2^-49 of it below that. Rows that do not count become zeros, so that
// whatever a padded row holds - NaN included - stays out of dW. 64 x 64 elements per
// workgroup through LDS.
struct TurnJob {
    const void* src;
    int64_t src_pitch;
    int32_t rows, cols;
    char* dst;
    int64_t pitch, plane;
    const float* all;
    const int64_t* target;
    int64_t ignore;
    __host__ __device__ int64_t blocks() const { return (int64_t)((cols + 63) / 64) * (pitch / 128); }
};

template <int DT>
__device__ __forceinline__ void turn_block(const TurnJob& j, int64_t block, uint16_t (*tile)[64][66]) {
    constexpr int NP = DT == DT_F32 ? 2 : 1;
    const int across = (j.cols + 63) / 64;
    const int64_t r0 = block / across * 64;
    const int c0 = (int)(block % across) * 64;
    const float scale = DT == DT_F32 ? 1.0f / *j.all : 1.0f;
    __align__(16) uint16_t h[2][8];
    for (int i = threadIdx.x; i < 64 * 8; i += 256) {
        const int r = i >> 3, c = (i & 7) * 8;
        const bool in = r0 + r < j.rows && !(j.target && j.target[r0 + r] == j.ignore);
        load_planes<DT>(j.src, (r0 + r) * j.src_pitch + c0 + c, in ? j.cols - c0 - c : 0, scale, h);
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int e = 0; e < 8; e += 2) *(uint32_t*)&tile[p][r][c + e] = (uint32_t)h[p][e] | (uint32_t)h[p][e + 1] << 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 8; i += 256) {
        const int c = i >> 3, piece = i & 7;
        if (c0 + c >= j.cols) continue;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[0][e] = tile[p][piece * 8 + e][c];
            *(uint4*)(j.dst + p * j.plane + (int64_t)(c0 + c) * j.pitch + (r0 + piece * 8) * 2) = *(const uint4*)h[0];
        }
    }
}

// All copies that a piece needs in one launch: they are independent and mostly small.
struct PackArgs {
    PackJob w, x;
    TurnJob wt, xt;
    int64_t end_w, end_x, end_wt;     // workgroups up to each
};

template <int DT>
__global__ __launch_bounds__(256) void k_pack(PackArgs a) {
    __shared__ __align__(16) uint16_t tile[DT == DT_F32 ? 2 : 1][64][66];
    const int64_t id = blockIdx.x;
    if (id < a.end_w) pack_block<DT>(a.w, id, (float*)tile);
    else if (id < a.end_x) pack_block<DT>(a.x, id - a.end_w, (float*)tile);
    else if (id < a.end_wt) turn_block<DT>(a.wt, id - a.end_x, tile);
    else turn_block<DT>(a.xt, id - a.end_wt, tile);
}

// ------------------------------------------------------------------------------------------------ shared arguments
// A softmax is summed as 2^t, t = z log2(e) - reference. The reference of a part of a row is its largest z log2(e) rounded to a whole
// number: then one fused multiply-add gives t with a single rounding, and references differ by whole numbers, so joining parts
// multiplies by exact powers of two. Beyond |z| = 2^17 (masks of a type's lowest value, say) the products would overflow; there the
// reference is the largest z itself. One float tells which: half of the whole number (below 2^17), or the z.
struct Reference {
    float off, whole;      // t = (z - off) * log2(e) - whole
    __device__ __forceinline__ explicit Reference(float v) : off(fabsf(v) < 131072.0f ? 0.0f : v), whole(fabsf(v) < 131072.0f ? 2.0f * v : 0.0f) {}
    __device__ __forceinline__ float t(float z) const { return __builtin_fmaf(z - off, LOG2E, -whole); }
};
__device__ __forceinline__ float reference_of(float top) { return fabsf(top) < 131072.0f ? 0.5f * rintf(top * LOG2E) : top; }
// References in one order, and the difference a - b in units of t.
__device__ __forceinline__ float reference_size(float v) { return fabsf(v) < 131072.0f ? v * (2.0f * LN2) : v; }
__device__ __forceinline__ float reference_minus(float a, float b) {
    return fabsf(a) < 131072.0f && fabsf(b) < 131072.0f ? 2.0f * (a - b) : (reference_size(a) - reference_size(b)) * LOG2E;
}

// The backward pass makes the logits again, by other kernels than the forward pass where these are faster, and so with other roundings: in
// logits of millions they leave more than the distance to the sum. No p is above one all the same: t goes up to this, from 1 / sum 2^t.
// (A logit that is no number is lost here, but in 1 / sum it is not.)
__device__ __forceinline__ float most_of(float inv) { return -__builtin_amdgcn_logf(inv); }

// Sums of a part of a row: its reference (-inf: no class that can be), sum 2^t, sum 2^t t, sum pi t, sum pi.
struct Part {
    float ref, l, s, dot, pi;
};
// Adds a part to one whose reference is already the largest of all.
__device__ __forceinline__ void join_part(Part& o, const Part& v) {
    if (v.ref == -INFINITY) {
        o.l += v.l;       // nothing, or the NaN of a logit that is none
        o.dot += v.dot;
    } else {
        const float d = reference_minus(v.ref, o.ref), e = __builtin_amdgcn_exp2f(d);
        o.l += v.l * e;
        o.s += e == 0.0f ? 0.0f : (v.s + v.l * d) * e;
        o.dot += v.pi == 0.0f ? v.dot : v.dot + v.pi * d;
    }
    o.pi += v.pi;
}

struct Rows {               // what a row's target says
    const int64_t* index;   // [rows] or null
    const float* dense;     // [rows, classes] with row stride dense_pitch, or null
    int64_t dense_pitch;
    int64_t ignore;
    int32_t rows, classes;
    float entropy;          // c
};

// The walk over the features in `pieces` of `per` steps; with more than one, k_ce_walk leaves their products in part, [pieces][tiles] of what
// the lanes of a tile hold.
struct Walk {
    int32_t pieces, per;
    f32x4* part;
};

struct StatArgs {
    MmOperand w, x;
    Rows t;
    const void* bias;
    int32_t kbytes;
    const float *un_w, *un_x;   // float32: what the operands were divided by, per class of the piece and per row
    int32_t v0;             // first class of the piece that w starts at
    int32_t tile0, tiles;   // first tile of the piece, tiles of all classes
    f32x4* part;            // [rows][tiles] ref, l, s, dot
    float* tpart;           // dense: [rows][tiles][2] sum pi, sum |pi|
    float* zt;              // index: [rows] logit of the target
    int32_t tiles_p, tiles_q;
    Walk walk;
};

// The small tile's products before anything is done to them, a piece of the features per workgroup: where rows and classes make few
// tiles, one walk over the features would leave most of the chip idle (forward, 64 x 8192 -> 60 float32: 159 us in one walk, 41 in pieces;
// 128 x 4096 -> 4096 bfloat16: 36 and 31).
template <class T, int DT>
__global__ __launch_bounds__(T::THREADS) void k_ce_walk(MmOperand w, MmOperand x, int kbytes, int tiles_p, int tiles_q, Walk walk) {
    __shared__ __align__(16) char lds[T::LDS];
    constexpr bool SPLIT = DT == DT_F32;
    int piece, tp, tq;
    mm_place_piece(blockIdx.x, walk.pieces, tiles_p, tiles_q, piece, tp, tq);
    const int steps = ((kbytes + 127) >> 7) * (SPLIT ? MM_SEGMENTS : 1), begin = piece * walk.per;
    typename T::acc_t acc[T::FP][T::FQ];
    mm_tile<T>(w, x, (int64_t)tp * T::BP, (int64_t)tq * T::BQ, kbytes, begin, begin + walk.per < steps ? begin + walk.per : steps, SPLIT ? MM_SEGMENTS : 1, lds, acc);
    f32x4* const o = walk.part + (((int64_t)piece * tiles_q + tq) * tiles_p + tp) * (T::FP * T::FQ * T::THREADS) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < T::FP; ++i)
#pragma unroll
        for (int j = 0; j < T::FQ; ++j) o[(i * T::FQ + j) * T::THREADS] = acc[i][j];
}

// The tile's logits in acc.
template <class T, int DT, class A>
__device__ __forceinline__ void logits(const A& a, int64_t p0, int64_t q0, char* lds, typename T::acc_t (&acc)[T::FP][T::FQ]) {
    constexpr bool SPLIT = DT == DT_F32;
    if (T::BP == 64 && a.walk.pieces > 1) {
        const int64_t tile = T::FP * T::FQ * T::THREADS, all = tile * a.tiles_p * a.tiles_q;
        const f32x4* const o = a.walk.part + (q0 / T::BQ * a.tiles_p + p0 / T::BP) * tile + threadIdx.x;
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int j = 0; j < T::FQ; ++j) acc[i][j] = o[(i * T::FQ + j) * T::THREADS];
#pragma unroll 4
        for (int k = 1; k < a.walk.pieces; ++k)
#pragma unroll
            for (int i = 0; i < T::FP; ++i)
#pragma unroll
                for (int j = 0; j < T::FQ; ++j) acc[i][j] += o[k * all + (i * T::FQ + j) * T::THREADS];
    } else {
        mm_tile<T>(a.w, a.x, p0, q0, a.kbytes, 0, ((a.kbytes + 127) >> 7) * (SPLIT ? MM_SEGMENTS : 1), SPLIT ? MM_SEGMENTS : 1, lds, acc);
    }
#ifdef __HIP_DEVICE_COMPILE__
    const int lane = mm_lane_after(), wave = threadIdx.x >> 6, wp = wave / T::WQ, wq = wave % T::WQ;
    const int ml = wp * T::TP + (lane >> 4) * 4;
    const int64_t here = a.w.rows - p0;       // classes of the piece from the tile's first one on
    if constexpr (SPLIT) {
        float un[T::FQ];
#pragma unroll
        for (int j = 0; j < T::FQ; ++j) {
            const int64_t n = q0 + wq * T::TQ + j * 16 + (lane & 15);
            un[j] = a.un_x[n < a.x.rows ? n : a.x.rows - 1];
        }
        const AxisView un_w(a.un_w + p0, here);
#pragma unroll
        for (int i = 0; i < T::FP; ++i) {
            const f32x4 u = un_w.four(ml + i * 16);
#pragma unroll
            for (int j = 0; j < T::FQ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] = acc[i][j][r] * u[r] * un[j];
        }
    }
    if (a.bias) {
        const AxisView bias((const char*)a.bias + (a.v0 + p0) * (DT == DT_F32 ? 4 : 2), here * (DT == DT_F32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float b = bias.one<DT>(ml + i * 16 + r);
#pragma unroll
                for (int j = 0; j < T::FQ; ++j) acc[i][j][r] += b;
            }
    }
#endif
}

// A row's target weights for the classes that a lane holds, from class `at` on, `left` of which exist. A tile without the last class (`full`)
// loads 16 bytes at a time and asks nothing; a question for each of them, held in a scalar register each, made the 256 tile spill
// (8192 x 1024 -> 4001 float16: forward 114 us, now 99, backward 353,
// now 305). Rows behind the last one get the last one's, which nobody uses.
template <class T>
__device__ __forceinline__ void target_weights(const Rows& t, int64_t n, int64_t at, int left, bool full, f32x4 (&pi)[T::FP]) {
    const float* const p = t.dense + (n < t.rows ? n : t.rows - 1) * t.dense_pitch + at;
    asm volatile("" : "+v"(left));        // the questions are not kept from one row of the lane for the next
    if (full) {
#pragma unroll
        for (int i = 0; i < T::FP; ++i) __builtin_memcpy(&pi[i], p + i * 16, 16);
    } else {
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) pi[i][r] = i * 16 + r < left ? p[i * 16 + r] : 0.0f;
    }
}

// ------------------------------------------------------------------------------------------------ forward
template <class T, int DT, bool DENSE, bool ENT>
__global__ __launch_bounds__(T::THREADS) void k_ce_stats(StatArgs a) {
    __shared__ __align__(16) char lds[T::LDS];
    int tp, tq;
    mm_place(blockIdx.x, a.tiles_p, a.tiles_q, tp, tq);
    const int64_t p0 = (int64_t)tp * T::BP, q0 = (int64_t)tq * T::BQ;
    typename T::acc_t acc[T::FP][T::FQ];
    logits<T, DT>(a, p0, q0, lds, acc);
    const int lane = mm_lane_after(), wave = threadIdx.x >> 6, wp = wave / T::WQ, wq = wave % T::WQ;
    const int left = a.t.classes - a.v0 - (int)p0 - wp * T::TP - (lane >> 4) * 4;   // classes from this lane's first one on
    if (p0 + T::BP > a.t.classes - a.v0) {          // the last tile
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (i * 16 + r >= left)
#pragma unroll
                    for (int j = 0; j < T::FQ; ++j) acc[i][j][r] = -INFINITY;
    }
    f32x4* const joint = (f32x4*)lds;                       // [WP][BQ]
    float* const jt = (float*)(lds + T::WP * T::BQ * 16);   // [WP][BQ][2]
#pragma unroll
    for (int j = 0; j < T::FQ; ++j) {
        const int64_t n = q0 + wq * T::TQ + j * 16 + (lane & 15);
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[i][j][r]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float ref = reference_of(top);
        const Reference at(top == -INFINITY ? 0.0f : ref);
        float l = 0.0f, s = 0.0f, dot = 0.0f, pi_sum = 0.0f, pi_abs = 0.0f;
        if (!DENSE && n < a.t.rows) {
            const int64_t hit = a.t.index[n] - (a.v0 + p0 + wp * T::TP + (lane >> 4) * 4);
            if (hit >= 0 && hit < T::TP && hit < left) {
#pragma unroll
                for (int i = 0; i < T::FP; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (hit == i * 16 + r) a.zt[n] = acc[i][j][r];
            }
        }
        f32x4 pi[T::FP];
        if constexpr (DENSE) target_weights<T>(a.t, n, a.v0 + p0 + wp * T::TP + (lane >> 4) * 4, left, p0 + T::BP <= a.t.classes - a.v0, pi);
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float t = at.t(acc[i][j][r]);
                const float e = __builtin_amdgcn_exp2f(t);
                l += e;
                if constexpr (ENT) s += e == 0.0f ? 0.0f : e * t;   // 0 * -inf of a class that cannot be
                if constexpr (DENSE) {
                    const float v = pi[i][r];
                    pi_sum += v;
                    pi_abs += fabsf(v);
                    dot += v == 0.0f ? 0.0f : v * t;
                }
            }
#pragma unroll
        for (int o = 16; o < 64; o *= 2) {
            l += __shfl_xor(l, o);
            if constexpr (ENT) s += __shfl_xor(s, o);
            if constexpr (DENSE) {
                dot += __shfl_xor(dot, o);
                pi_sum += __shfl_xor(pi_sum, o);
                pi_abs += __shfl_xor(pi_abs, o);
            }
        }
        if (lane < 16) {
            const int q = wp * T::BQ + wq * T::TQ + j * 16 + lane;
            joint[q] = f32x4{ref, l, s, dot};
            if constexpr (DENSE) {
                jt[2 * q] = pi_sum;
                jt[2 * q + 1] = pi_abs;
            }
        }
    }
    __syncthreads();
    for (int q = threadIdx.x; q < T::BQ; q += T::THREADS) {
        if (q0 + q >= a.t.rows) break;
        Part v[T::WP];
        float ta = 0.0f;
        Part o = {-INFINITY, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < T::WP; ++w) {
            const f32x4 u = joint[w * T::BQ + q];
            v[w] = Part{u[0], u[1], u[2], u[3], DENSE ? jt[2 * (w * T::BQ + q)] : 0.0f};
            if (DENSE) ta += jt[2 * (w * T::BQ + q) + 1];
            if (reference_size(v[w].ref) > reference_size(o.ref)) o.ref = v[w].ref;
        }
#pragma unroll
        for (int w = 0; w < T::WP; ++w) join_part(o, v[w]);
        const int64_t at = (q0 + q) * a.tiles + a.tile0 + tp;
        a.part[at] = f32x4{o.ref, o.l, o.s, o.dot};
        if constexpr (DENSE) {
            a.tpart[2 * at] = o.pi;
            a.tpart[2 * at + 1] = ta;
        }
    }
}

struct JoinArgs {
    Rows t;
    const f32x4* part;
    const float* tpart;
    const float* zt;
    int32_t tiles, reduction;
    float *ref, *inv, *mean, *tsum, *scalars;   // kept for the backward pass: reference, 1 / l, s / l, sum pi
    float *ce, *ent, *tabs;                     // per row
    float *loss, *out_ce, *out_ent;          // results, per row or one; the last two may be null
    const float *un_x, *un_w;                // float32: what operands were divided by, by row and class or by workgroup; or null
    int32_t count_x, count_w;
};

__device__ __forceinline__ Part part_at(const JoinArgs& a, int64_t at) {
    const f32x4 u = a.part[at];
    return Part{u[0], u[1], u[2], u[3], a.t.dense ? a.tpart[2 * at] : 0.0f};
}

// LANES lanes per row, each over its share of the row's tiles. 8192 rows of 512 tiles: 24 us (67 MB).
template <int LANES>
__device__ __forceinline__ void join_row(const JoinArgs& a, int64_t n, int lane) {
    const int64_t first = n * a.tiles;
    Part v = {-INFINITY, 0.0f, 0.0f, 0.0f, 0.0f};
    float top = -INFINITY, ta = 0.0f;      // top: the largest reference's place in the order
    auto larger = [&](float ref) {
        if (reference_size(ref) > top) {
            top = reference_size(ref);
            v.ref = ref;
        }
    };
#pragma unroll 4
    for (int i = lane; i < a.tiles; i += LANES) larger(a.part[first + i][0]);
#pragma unroll
    for (int o = 1; o < LANES; o *= 2) larger(__shfl_xor(v.ref, o));
#pragma unroll 4
    for (int i = lane; i < a.tiles; i += LANES) {
        join_part(v, part_at(a, first + i));
        if (a.t.dense) ta += a.tpart[2 * (first + i) + 1];
    }
#pragma unroll
    for (int o = 1; o < LANES; o *= 2) {
        v.l += __shfl_xor(v.l, o);
        v.s += __shfl_xor(v.s, o);
        v.dot += __shfl_xor(v.dot, o);
        v.pi += __shfl_xor(v.pi, o);
        ta += __shfl_xor(ta, o);
    }
    if (lane) return;
    const bool none = v.ref == -INFINITY;      // every logit of the row is -inf: no softmax exists
    const float bits = none ? NAN : __builtin_amdgcn_logf(v.l), inv = 1.0f / v.l, mean = v.s * inv;   // log2 of the sum
    const float h = none ? NAN : LN2 * (bits - mean);
    float ce;
    bool counts = true;
    if (a.t.dense) {
        ce = LN2 * (v.pi * bits - v.dot);
        a.tsum[n] = v.pi;
        a.tabs[n] = ta;
    } else {
        const int64_t t = a.t.index[n];
        counts = t != a.t.ignore;
        ce = t >= 0 && t < a.t.classes ? LN2 * (bits - Reference(v.ref).t(a.zt[n])) : NAN;   // a class that does not exist: nobody overlooks it
    }
    a.ref[n] = v.ref;
    a.inv[n] = inv;
    a.mean[n] = mean;
    a.ent[n] = h;
    a.ce[n] = ce;
    if (a.reduction == AZ_REDUCE_NONE) {
        a.loss[n] = counts ? (a.t.entropy != 0.0f ? ce - a.t.entropy * h : ce) : 0.0f;
        if (a.out_ce) a.out_ce[n] = counts ? ce : 0.0f;
        if (a.out_ent) a.out_ent[n] = counts ? h : 0.0f;
    }
}

// Sums over the rows by one workgroup of 1024, in a fixed order and in 64 bits (a row is 4 to 20 bytes here).
__device__ __forceinline__ void reduce_rows(const JoinArgs& a) {
    __shared__ double sums[2][16];
    __shared__ float tops[16];
    __shared__ int numbers[16];
    __shared__ float uns[2][16];
    double ce = 0.0, h = 0.0;
    float top = 0.0f;
    int count = 0;
    for (int n = threadIdx.x; n < a.t.rows; n += 1024) {
        if (a.t.index && a.t.index[n] == a.t.ignore) continue;
        ++count;
        ce += a.ce[n];
        h += a.ent[n];
        if (a.t.dense && a.tabs[n] < INFINITY) top = fmaxf(top, a.tabs[n]);     // a row of infinite weights spoils itself only
    }
    float ux = 0.0f, uw = 0.0f;        // the largest: the backward pass divides its transposed copies by it
    if (a.un_x) {
        for (int n = threadIdx.x; n < a.count_x; n += 1024) ux = fmaxf(ux, a.un_x[n]);
#pragma unroll 4
        for (int m = threadIdx.x; m < a.count_w >> 2; m += 1024) {
            const f32x4 v = ((const f32x4*)a.un_w)[m];
            uw = fmaxf(fmaxf(uw, fmaxf(v[0], v[1])), fmaxf(v[2], v[3]));
        }
        if (const int m = (a.count_w & ~3) + threadIdx.x; m < a.count_w) uw = fmaxf(uw, a.un_w[m]);
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            ux = fmaxf(ux, __shfl_xor(ux, o));
            uw = fmaxf(uw, __shfl_xor(uw, o));
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        ce += __shfl_xor(ce, o);
        h += __shfl_xor(h, o);
        top = fmaxf(top, __shfl_xor(top, o));
        count += __shfl_xor(count, o);
    }
    if ((threadIdx.x & 63) == 0) {
        const int w = threadIdx.x >> 6;
        sums[0][w] = ce;
        sums[1][w] = h;
        tops[w] = top;
        numbers[w] = count;
        uns[0][w] = ux;
        uns[1][w] = uw;
    }
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 16; ++w) {
        ce += sums[0][w];
        h += sums[1][w];
        top = fmaxf(top, tops[w]);
        count += numbers[w];
    }
    if (a.un_x) {
        for (int w = 1; w < 16; ++w) {
            ux = fmaxf(ux, uns[0][w]);
            uw = fmaxf(uw, uns[1][w]);
        }
        a.scalars[2] = ux;
        a.scalars[3] = uw;
    }
    a.scalars[0] = (float)count;
    // |G| <= 2 sum |pi| + |c| (1/e + log classes)
    a.scalars[1] = (a.t.dense ? 2.0f * top : 1.0f) + fabsf(a.t.entropy) * (0.4f + logf((float)a.t.classes));
    if (a.reduction == AZ_REDUCE_NONE) return;
    const double d = a.reduction == AZ_REDUCE_MEAN ? (double)count : 1.0;
    a.loss[0] = (float)((ce - (a.t.entropy != 0.0f ? a.t.entropy * h : 0.0)) / d);
    if (a.out_ce) a.out_ce[0] = (float)(ce / d);
    if (a.out_ent) a.out_ent[0] = (float)(h / d);
}

// A wave per row where a row has many tiles, four lanes where it has few.
__global__ __launch_bounds__(256) void k_ce_join(JoinArgs a) {
    if (a.tiles > 32) {
        const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
        if (n < a.t.rows) join_row<64>(a, n, threadIdx.x & 63);
    } else {
        const int64_t n = (int64_t)blockIdx.x * 64 + (threadIdx.x >> 2);
        if (n < a.t.rows) join_row<4>(a, n, threadIdx.x & 3);
    }
}
__global__ __launch_bounds__(1024) void k_ce_reduce(JoinArgs a) { reduce_rows(a); }
// Few rows with few tiles: both in one launch.
__global__ __launch_bounds__(1024) void k_ce_join_reduce(JoinArgs a) {
    for (int64_t n = threadIdx.x >> 2; n < a.t.rows; n += 256) join_row<4>(a, n, threadIdx.x & 3);
    __threadfence_block();
    __syncthreads();
    reduce_rows(a);
}

// ------------------------------------------------------------------------------------------------ backward
// How G is held in 16 bits. The factor of a row (the caller's gradient, over the number of rows in a mean) stays out of what is
// rounded wherever it can: rounded with it, the -1 at every row's target would be off by the same relative amount in every row, and
// that would not average out. With one factor for all rows it multiplies the products' results. With a factor for each row it does so
// for dx, and for dW, whose sum runs over the rows, G^T holds factor / largest factor.
// float16 (and the two planes of float32) has too few exponents for small p: there G is held times the power of two that takes its
// bound to at most 2^14, so that values down to 2^-27 of the bound keep all their bits.
__device__ __forceinline__ float hold_scale(const float* scalars) {
    return ldexpf(1.0f, 14 - (ilogbf(fmaxf(scalars[1], 1e-30f)) + 1));
}

// Largest |gradient| of the rows, for one gradient per row.
__global__ __launch_bounds__(1024) void k_ce_largest(const float* grad, Rows t, float* out) {
    __shared__ float tops[16];
    float top = 0.0f;
    auto see = [&](float g) { top = g > top || g != g ? g : top; };      // a NaN stays
    for (int n = threadIdx.x; n < t.rows; n += 1024)
        if (!(t.index && t.index[n] == t.ignore)) see(fabsf(grad[n]));      // the gradient of a row that does not count may be anything
#pragma unroll
    for (int o = 1; o < 64; o *= 2) see(__shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 16; ++w) see(tops[w]);
    *out = top;
}

// The factors that the results of the products with G get.
struct Factor {
    const float *grad, *scalars, *largest;   // largest: one gradient per row
    int32_t mean, half;                      // half: G is held times hold_scale
    const float* un;                         // float32: what the other operand was divided by, or null
    const int64_t* index;                    // rows that do not count get 0, whatever their gradient
    int64_t ignore;
};
__device__ __forceinline__ float factor_all(const Factor& f) {            // dW, db, and dx with one factor
    float v = f.largest ? *f.largest : f.grad[0];
    if (f.mean) v = f.scalars[0] > 0.0f ? v / f.scalars[0] : 0.0f;     // no row counts: G is zero
    if (f.un) v *= *f.un;
    return f.half ? v / hold_scale(f.scalars) : v;
}
__device__ __forceinline__ float factor_row(const Factor& f, int64_t n) {  // dx with one factor per row
    if (f.index && f.index[n] == f.ignore) return 0.0f;
    const float v = f.un ? f.grad[n] * *f.un : f.grad[n];
    return f.half ? v / hold_scale(f.scalars) : v;
}

struct GradArgs {
    MmOperand w, x;
    Rows t;
    const void* bias;
    int32_t kbytes;
    const float *un_w, *un_x;
    int32_t v0;
    int32_t tiles_p, tiles_q;
    Walk walk;
    const float *ref, *inv, *mean, *tsum;
    Factor f;
    int32_t two;           // 16 bits: G in two planes
    char* g;               // [rows][g_pitch] per plane, or null (no dx wanted)
    int64_t g_pitch, g_plane;
    char* gt;              // [classes of the piece][gt_pitch] per plane, or null (no dW wanted)
    int64_t gt_pitch, gt_plane;
    float* db;             // [tiles_q][db_pitch] sums over a tile's rows, or null
    int64_t db_pitch;
};

// Two waves to a SIMD: with float32, target weights and entropy the 128 tile would else take one register too many for them.
template <class T, int DT, bool DENSE, bool ENT>
__global__ __launch_bounds__(T::THREADS, 2) void k_ce_grad(GradArgs a) {
    __shared__ __align__(16) char lds[T::LDS];
    int tp, tq;
    mm_place(blockIdx.x, a.tiles_p, a.tiles_q, tp, tq);
    const int64_t p0 = (int64_t)tp * T::BP, q0 = (int64_t)tq * T::BQ;
    typename T::acc_t acc[T::FP][T::FQ];
    logits<T, DT>(a, p0, q0, lds, acc);
    const int lane = mm_lane_after(), wave = threadIdx.x >> 6, wp = wave / T::WQ, wq = wave % T::WQ;
    const int ml = (int)p0 + wp * T::TP + (lane >> 4) * 4;        // class of the piece
    const int left = a.t.classes - a.v0 - ml;
    const float hold = a.f.half ? hold_scale(a.f.scalars) : 1.0f;
    float share[T::FQ];        // of a row's factor in the largest
#pragma unroll
    for (int j = 0; j < T::FQ; ++j) {
        const int64_t n = q0 + wq * T::TQ + j * 16 + (lane & 15);
        const bool row = n < a.t.rows;
        int64_t target = 0;
        float ref = 0.0f, inv = 0.0f, mean = 0.0f, total = 1.0f, f = hold;
        bool counts = false;
        share[j] = 1.0f;
        if (row) {
            ref = a.ref[n];
            inv = a.inv[n];
            if constexpr (ENT) mean = a.mean[n];
            if constexpr (DENSE) total = a.tsum[n];
            else target = a.t.index[n];
            counts = DENSE || target != a.t.ignore;
            if (a.f.largest) share[j] = counts && (*a.f.largest > 0.0f || *a.f.largest != *a.f.largest) ? a.f.grad[n] / *a.f.largest : 0.0f;
            if (!DENSE && (target < 0 || target >= a.t.classes)) f = NAN;
        }
        const Reference at(ref);
        const float most = most_of(inv);
        f32x4 pi[T::FP];
        if constexpr (DENSE) target_weights<T>(a.t, n, a.v0 + ml, left, p0 + T::BP <= a.t.classes - a.v0, pi);
        const float scale = (DENSE ? total * inv : inv) * f, c = a.t.entropy * LN2 * inv * f;
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float t = fminf(at.t(acc[i][j][r]), most);
                const float e = __builtin_amdgcn_exp2f(t);
                float g = e * scale;
                if constexpr (DENSE) g -= pi[i][r] * f;
                if constexpr (ENT) g += e == 0.0f ? 0.0f : c * e * (t - mean);
                acc[i][j][r] = counts ? g : 0.0f;
            }
        if constexpr (!DENSE) {
            const int64_t hit = target - a.v0 - ml;
            if (counts && hit >= 0 && hit < T::TP) {
#pragma unroll
                for (int i = 0; i < T::FP; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (hit == i * 16 + r) acc[i][j][r] -= f;
            }
        }
    }
    if (p0 + T::BP > a.t.classes - a.v0) {          // classes behind the last one
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (i * 16 + r >= left)
#pragma unroll
                    for (int j = 0; j < T::FQ; ++j) acc[i][j][r] = 0.0f;
    }
    if (a.db) {
        float* const joint = (float*)lds;      // [WQ][BP]
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float s = 0.0f;
#pragma unroll
                for (int j = 0; j < T::FQ; ++j) s += acc[i][j][r] * share[j];
#pragma unroll
                for (int o = 1; o < 16; o *= 2) s += __shfl_xor(s, o);
                if ((lane & 15) == 0) joint[wq * T::BP + wp * T::TP + i * 16 + (lane >> 4) * 4 + r] = s;
            }
        __syncthreads();
        for (int p = threadIdx.x; p < T::BP; p += T::THREADS) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < T::WQ; ++w) s += joint[w * T::BP + p];
            if (p0 + p < a.db_pitch) a.db[tq * a.db_pitch + p0 + p] = s;
        }
        __syncthreads();
    }
    auto emit = [&](auto which) {
        constexpr int P = decltype(which)::value;
        auto bits = [&](int i, int j, float by) {
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v[r] = acc[i][j][r] * by;
                if constexpr (P == 1 && DT == DT_BF16) v[r] -= (float)(__bf16)v[r];
                else if constexpr (P == 1) v[r] = (v[r] - (float)(_Float16)v[r]) * 2048.0f;      // G is finite in float16: hold_scale
            }
            return pack4<DT == DT_BF16 ? DT_BF16 : DT_F16>(v[0], v[1], v[2], v[3]);
        };
        if (a.g) {
            mm_stage<T>(lds, [&](int i, int j) { return bits(i, j, 1.0f); });
            __syncthreads();
            mm_unstage<T, T::BQ, T::BP>(lds, a.g + P * a.g_plane + q0 * a.g_pitch + p0 * 2, a.g_pitch, a.t.rows - q0, a.g_pitch - p0 * 2);
            __syncthreads();
        }
        if (a.gt) {
            mm_stage_turned<T>(lds, [&](int i, int j) { return bits(i, j, share[j]); });
            __syncthreads();
            mm_unstage<T, T::BP, T::BQ>(lds, a.gt + P * a.gt_plane + p0 * a.gt_pitch + q0 * 2, a.gt_pitch, a.w.rows - p0, a.gt_pitch - q0 * 2);
            __syncthreads();
        }
    };
    emit(std::integral_constant<int, 0>{});
    if constexpr (DT == DT_F32 || T::BP < 256) {
        if (DT == DT_F32 || a.two) {
            mm_opaque<T>(acc);       // the planes are made one after another: both would not fit the registers
            emit(std::integral_constant<int, 1>{});
        }
    }
}

struct OutArgs {
    MmOperand p, q;
    int32_t kbytes, tiles_p, tiles_q;
    int32_t splits, per;   // the walk over k in `splits` pieces of `per` steps
    float* part;           // [splits][q rows][p rows] with more than one: k_ce_out_join adds them
    void* out;             // [q rows][p rows]
    float* sum;            // running sums over the pieces of the classes, or null
    int32_t first, last, by_row;
    Factor f;
};

// SEGMENTS of the walk: three for float32, two for 16 bits with G in two planes.
template <class T, int DT, int SEGMENTS>
__device__ __forceinline__ void out_tile(const OutArgs& a, int id, char* lds) {
    const int tiles = a.tiles_p * a.tiles_q, split = id / tiles;
    int tp, tq;
    mm_place(id - split * tiles, a.tiles_p, a.tiles_q, tp, tq);
    const int64_t p0 = (int64_t)tp * T::BP, q0 = (int64_t)tq * T::BQ;
    typename T::acc_t acc[T::FP][T::FQ];
    const int steps = ((a.kbytes + 127) >> 7) * SEGMENTS, begin = split * a.per;
    mm_tile<T>(a.p, a.q, p0, q0, a.kbytes, begin, begin + a.per < steps ? begin + a.per : steps, SEGMENTS, lds, acc);
    const int lane = mm_lane_after(), wave = threadIdx.x >> 6, wp = wave / T::WQ, wq = wave % T::WQ;
    const int64_t width = a.p.rows;
    const bool first = a.first || a.splits > 1, last = a.last && a.splits == 1;
    float* const sum = a.splits > 1 ? a.part + (int64_t)split * a.q.rows * width : a.sum;
    const float all = a.by_row || !last ? 0.0f : factor_all(a.f);
#pragma unroll
    for (int j = 0; j < T::FQ; ++j) {
        const int64_t n = q0 + wq * T::TQ + j * 16 + (lane & 15);
        const bool row = n < a.q.rows;
        const float post = !row || !last ? 0.0f : a.by_row ? factor_row(a.f, n) : all;
#pragma unroll
        for (int i = 0; i < T::FP; ++i) {
            const int64_t m = p0 + wp * T::TP + i * 16 + (lane >> 4) * 4;
            const int64_t at = n * width + m;
            if (row && m + 4 <= width) {        // four together, wherever a row starts
                if (!first) {
                    f32x4 before;
                    __builtin_memcpy(&before, sum + at, 16);
                    acc[i][j] += before;
                }
                if (!last) __builtin_memcpy(sum + at, &acc[i][j], 16);
            } else if (row) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m + r < width) {
                        if (!first) acc[i][j][r] += sum[at + r];
                        if (!last) sum[at + r] = acc[i][j][r];
                    }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] *= post;
            if constexpr (DT == DT_F32) {       // 16 bytes per lane already
                if (last && row) {
                    float* o = (float*)a.out + at;
                    if (m + 4 <= width) {
                        __builtin_memcpy(o, &acc[i][j], 16);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (m + r < width) o[r] = acc[i][j][r];
                    }
                }
            }
        }
    }
    if constexpr (DT != DT_F32) {
        if (!last) return;
        mm_stage<T>(lds, [&](int i, int j) { return pack4<DT>(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]); });
        __syncthreads();
        mm_unstage<T, T::BQ, T::BP>(lds, (char*)a.out + (q0 * width + p0) * 2, width * 2, a.q.rows - q0, (width - p0) * 2);
    }
}

// Adds the pieces of split walks, in their order: one thread per result.
template <int DT>
__global__ __launch_bounds__(256) void k_ce_out_join(OutArgs a, OutArgs b, int64_t blocks_a) {
    const bool one = (int64_t)blockIdx.x < blocks_a;
    const OutArgs& o = one ? a : b;
    const int64_t at = ((int64_t)blockIdx.x - (one ? 0 : blocks_a)) * 256 + threadIdx.x, size = (int64_t)o.p.rows * o.q.rows;
    if (at >= size) return;
    float v = 0.0f;
#pragma unroll 4
    for (int i = 0; i < o.splits; ++i) v += o.part[i * size + at];
    if (!o.first) v += o.sum[at];
    if (!o.last) o.sum[at] = v;
    else store_scalar<DT>(o.out, at, v * (o.by_row ? factor_row(o.f, at / o.p.rows) : factor_all(o.f)));
}

struct BiasArgs {
    const float* part;     // [tiles][pitch]
    int64_t pitch, at;
    int32_t tiles, classes;
    void* out;
    Factor f;
};

template <int DT>
__device__ __forceinline__ void bias_block(const BiasArgs& a, int64_t m) {
    if (m >= a.classes) return;
    float s = 0.0f;
    for (int t = 0; t < a.tiles; ++t) s += a.part[t * a.pitch + m];
    store_scalar<DT>(a.out, a.at + m, s * factor_all(a.f));
}

// dx, dW and db of a piece in one launch: they share nothing but G, and small ones fill the chip together.
template <class T, int DT, int SEGMENTS>
__global__ __launch_bounds__(T::THREADS) void k_ce_out(OutArgs a, OutArgs b, BiasArgs c, int blocks_a, int blocks_b) {
    __shared__ __align__(16) char lds[T::LDS];
    const int id = blockIdx.x;
    if (id < blocks_a) out_tile<T, DT, SEGMENTS>(a, id, lds);
    else if (id < blocks_a + blocks_b) out_tile<T, DT, SEGMENTS>(b, id - blocks_a, lds);
    else bias_block<DT>(c, (int64_t)(id - blocks_a - blocks_b) * T::THREADS + threadIdx.x);
}

}  // namespace
}  // namespace az
#include "az_head_few.cuh"
namespace az {
namespace {

// ------------------------------------------------------------------------------------------------ host side
// float32 goes as planes of float16. Four stages for the small tile: its workgroups wait for memory more than they compute (eight gain
// nothing for few tiles and cost a resident workgroup for many: 4096 x 722 -> 362 20.5 against 14.8 us).
template <int KIND> struct TilesOf {
    typedef MmTile<256, 256, 2, 4, 2, KIND> Big;
    typedef MmTile<128, 128, 2, 2, 2, KIND> Mid;
    typedef MmTile<64, 64, 2, 2, 4, KIND> Small;
};
template <int DT> struct Tiles : TilesOf<MM_F16> {};
template <> struct Tiles<DT_BF16> : TilesOf<MM_BF16> {};

int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

struct Layout {       // of the workspace, and the pieces of the classes
    bool few = false;   // the kernels of az_head_few.cuh
    int grid = 0, chunks = 0, chunk = 0;      // of those: workgroups; chunks of the classes, classes of a chunk
    bool split;              // float32
    bool pack_w, pack_x;     // operands copied into rows of whole 16 bytes
    int planes, g_planes;         // 16-bit planes of an operand, and of G
    int edge_most = 256;          // largest tile of the backward pass
    int64_t kpitch;     // bytes of an operand's row as the tile loop reads it (when packed)
    int64_t piece;      // classes of a piece
    int pieces;
    int64_t bytes = 0;
    int64_t xp = -1, wp = -1, ux = -1, uw = -1, part = -1, tpart = -1, zt = -1, ce = -1, tabs = -1, walk = -1;          // forward
    int64_t xt = -1, wt = -1, g = -1, gt = -1, db = -1, sum = -1, largest = -1, px = -1, pw = -1, fg = -1;                 // backward
    int64_t take(int64_t n) {
        const int64_t at = bytes;
        bytes += round_up(n, 256);
        return at;
    }
};

bool in_place(const void* p, int64_t pitch, int64_t cols) { return ((uintptr_t)p & 15) == 0 && (pitch & 7) == 0 && (cols & 7) == 0 && pitch * 2 <= MM_MAX_PITCH; }

void operand_layout(const az_linear_ce_args& a, Layout& l) {
    l.split = a.dtype == AZ_DT_F32;
    l.planes = l.split ? 2 : 1;
    // Where a handful of values is most of G, the rounding of each to 16 bits shows in the gradients. Their error against what the rounding of
    // the gradients themselves makes: 1.6 with up to 40 rows, 1.45 with 100; beyond, with target weights 1.4 at 362
    // classes, 1.36 at 600, 1.25 at 2000, 1.05 to 1.15 at 20000, with class indices 1.2 at 512, 1.1 to 1.18 at 4000, 1.01 to 1.13 at
    // 20000 to 32000 (less in bfloat16). With two planes of G it is 1.0 everywhere.
    // They cost, in both passes together, 8 to 20 % with up to 128 rows (64 x 4096 -> 4096 bfloat16 77 and 91 us, 64 x 722 -> 362 34 and
    // 39), 7 to 17 % with up to 512 classes (256 x 162 -> 82 float16 36.8 and 39.4, 4096 x 722 -> 362 80 and 89, 16384 x 722 -> 362 176
    // and 201, 16384 x 256 -> 512 115 and 131), and from 13 % to twice the time beyond (4096 x 256 -> 2048 87 and 103, 1024 x 1024 -> 4096 99
    // and 127, 1024 x 2048 -> 32000 687 and 1403), where it is the caller's choice.
    const bool two = !l.split && (a.rows <= 128 || a.classes <= 512 || (a.reduction & AZ_PRECISE_GRADIENT));
    l.g_planes = l.split || two ? 2 : 1;
    if (two) l.edge_most = 128;
    l.pack_w = l.split || !in_place(a.weight, a.weight_pitch, a.features);
    l.pack_x = l.split || !in_place(a.x, a.x_pitch, a.features);
    l.kpitch = round_up(a.features, 8) * 2;
}

int64_t logit_steps(const az_linear_ce_args& a) { return (a.features + 63) / 64 * (a.dtype == AZ_DT_F32 ? MM_SEGMENTS : 1); }

// Tile edge of the logits of nv classes, and pieces of the walk over the features (small tiles only). In microseconds: a step of a workgroup
// that has a compute unit for itself takes about half of what it takes two (1024 x 2048 -> 1000 bfloat16, 256 tiles: one walk 28, two
// pieces 30), joining costs a launch and 16 KB per piece that one workgroup reads. At most 512 workgroups, two on each compute unit, so the sums never take more than 8 MB.
constexpr int64_t WALK_BYTES = int64_t(512) * 64 * 64 * 4;
struct LogitPlan {
    int edge, pieces, per;
};
LogitPlan logit_plan(const az_linear_ce_args& a, int64_t nv, int edge = 0) {
    const int64_t steps = logit_steps(a), tiles = ((nv + 63) / 64) * ((a.rows + 63) / 64);
    LogitPlan p{edge ? edge : mm_tile_edge(nv, a.rows, steps), 1, (int)steps};
    if ((edge && edge != 64) || tiles > 256) return p;
    double least = steps * 0.4 + 4.0;      // of small tiles, which is what few tiles always are
    if (p.edge != 64) return p;
    for (int64_t n = 2; n * tiles <= 512 && n * 2 <= steps; ++n) {
        const int64_t per = (steps + n - 1) / n;
        const double t = per * (n * tiles <= 256 ? 0.4 : 0.8) + 4.0 + 8.0 + n * 0.25;
        if (t < least) {
            least = t;
            p = {64, (int)((steps + per - 1) / per), (int)per};
        }
    }
    return p;
}
int forward_edge(const az_linear_ce_args& a) { return logit_plan(a, a.classes).edge; }

// Waves of a workgroup that split the features of the same classes: each keeps eight turns of loads, unless more splitting makes a
// workgroup for every half compute unit.
int few_share(const az_linear_ce_args& a) {
    const int64_t turns = a.features / (a.dtype == AZ_DT_F32 ? 16 : 32);
    int share = 1;
    while (share < 16 && (share * 16 <= turns || (share * 2 <= turns && a.classes * share < 512 * 16 * FEW_CLASSES))) share *= 2;
    return share;
}
// Workgroups of the streaming kernel: two per compute unit, each with a stretch of classes.
int few_grid(const az_linear_ce_args& a) {
    const int64_t groups = (a.classes + 16 / few_share(a) * FEW_CLASSES - 1) / (16 / few_share(a) * FEW_CLASSES);
    return (int)(groups < 512 ? groups : 512);
}

// Where the kernels of az_head_few.cuh, which stream the weight as it lies, take the place of the tiles. Measured with 1 to 32 rows.
// Forward, 16 bits: tiles read a weight in place as fast (16 x 4096 -> 4096: 26 us against 31, 16 x 1024 -> 32000: 30 against 52); only
// copying a large one costs more (16 x 4095 -> 32000: 212 against 185; 16 x 2047 -> 16000: 54 against 68).
// Forward, float32, where tiles always copy: streaming (16 x 4096 -> 4096: 43 us against 72) unless long features and few classes leave it
// few workgroups (16 x 8192 -> 60: 59 against 40). 24 rows 101 us against 238 (2048 -> 32000), 48 rows, which need more accumulators
// than it has registers, 246 against 240.
bool few_forward(const az_linear_ce_args& a) {
    if (a.dtype == AZ_DT_F32) return a.rows <= 32 && (a.features <= 1024 || a.features <= 4 * a.classes);
    return a.rows <= 16 && !in_place(a.weight, a.weight_pitch, a.features) && a.classes * a.features > (int64_t(1) << 26);
}
// Backward: streaming saves the turned copies of the weight and G, its sums over the classes grow with the rows (streaming against tiles, us).
// 16 bits: 4096 -> 8000 4 rows 49, 100, 16 rows 71, 100; 2048 -> 4000 8 rows 37, 46, 16 rows 46, 46; 4096 -> 1000 4 rows 30, 38, 16 rows 45, 38;
// 1024 -> 200 4 rows 23, 19; copied 2047 -> 16000 1 row 114, 142, 16 rows 142, 140. float32: 2048 -> 4000 16 rows 51, 75; 2048 -> 1000
// 4 rows 29, 40, 16 rows 43, 40; 1024 -> 200 1 row 19, 23, 8 rows 27, 24.
bool few_backward(const az_linear_ce_args& a) {
    const int64_t size = a.classes * a.features;
    if (a.rows > FEW_GRAD_ROWS || a.features > 16 * a.classes || a.features < 256) return false;      // 256 lanes take 4 features each
    if (a.dtype == AZ_DT_F32) return size >= a.rows * (3 << 16);
    return size >= a.rows << 19 && (size >= int64_t(1) << 24 || in_place(a.weight, a.weight_pitch, a.features));
}

Layout forward_layout(const az_linear_ce_args& a) {
    Layout l;
    if (few_forward(a)) {
        l.few = true;
        l.grid = few_grid(a);
        l.part = l.take(a.rows * l.grid * 16);
        l.ce = l.take(a.rows * 8);
        if (a.target_dense) {
            l.tpart = l.take(a.rows * l.grid * 8);
            l.tabs = l.take(a.rows * 4);
        } else {
            l.zt = l.take(a.rows * 4);
        }
        if (a.dtype == AZ_DT_F32) {
            l.ux = l.take(l.grid * 4);
            l.uw = l.take(l.grid * 4);
        }
        return l;
    }
    operand_layout(a, l);
    const int64_t edge = forward_edge(a), tiles = (a.classes + edge - 1) / edge;
    // A launch holds fewer than 2^32 threads, a tile 512 at most; a packed piece of the weight stays below 512 MB. Pieces start at tiles.
    int64_t piece = (int64_t(1) << 22) / ((a.rows + edge - 1) / edge) * edge;
    if (l.pack_w) {
        const int64_t w = (int64_t(1) << 29) / (l.kpitch * l.planes) / 256 * 256;
        if (w < piece) piece = w;
    }
    l.piece = piece < 256 ? 256 : piece;
    if (l.piece > a.classes) l.piece = a.classes;
    l.pieces = (int)((a.classes + l.piece - 1) / l.piece);
    if (l.pack_x) l.xp = l.take(a.rows * l.kpitch * l.planes);
    if (l.pack_w) l.wp = l.take(l.piece * l.kpitch * l.planes);
    if (l.split) {
        l.ux = l.take(a.rows * 4);
        l.uw = l.take(a.classes * 4);
    }
    if (edge == 64) l.walk = l.take(WALK_BYTES);
    l.part = l.take(a.rows * tiles * 16);
    l.ce = l.take(a.rows * 8);       // cross entropy, entropy
    if (a.target_dense) {
        l.tpart = l.take(a.rows * tiles * 8);
        l.tabs = l.take(a.rows * 4);
    } else {
        l.zt = l.take(a.rows * 4);
    }
    return l;
}

// How dx = G W and dW = G^T x of a piece of nv classes go over the chip: one tile size for both, and walks over k split where they are so
// long, or so few, that the chip would wait for the last ones. A workgroup's walk is at most half of what a compute unit does in all,
// but not below 8 steps, where fetching the first stage costs as much as the products. Split walks write and read their sums once
// more. The tile with the least time is taken.
struct OutPlan {
    int edge;
    struct Job {
        int tiles_p, tiles_q, splits, per;
    } x, w;
};
OutPlan out_plan(const az_linear_ce_args& a, const Layout& l, int64_t nv) {
    OutPlan best{};
    double least = 1e300;
    const int walks = l.split ? MM_SEGMENTS : l.g_planes;
    const int64_t steps_x = round_up(nv, 64) / 64 * walks, steps_w = round_up(a.rows, 64) / 64 * walks;
    for (const MmTileCost& c : MM_TILE_COSTS) {
        if (c.edge > l.edge_most) continue;
        OutPlan o;
        o.edge = c.edge;
        auto tiles = [&](int64_t n) { return (int)((n + o.edge - 1) / o.edge); };
        o.x = {tiles(a.features), tiles(a.rows), 1, (int)steps_x};
        o.w = {tiles(a.features), tiles(nv), 1, (int)steps_w};
        const int64_t total = steps_x * o.x.tiles_p * o.x.tiles_q + steps_w * o.w.tiles_p * o.w.tiles_q;
        const int64_t cap = total / 512 > 8 ? total / 512 : 8;
        double sums = 0.0;
        auto split = [&](OutPlan::Job& j, int64_t steps, int64_t results) {
            if (steps <= 2 * cap) return;
            j.per = (int)cap;
            j.splits = (int)((steps + cap - 1) / cap);
            sums += j.splits * (double)results * 8.0;
        };
        split(o.x, steps_x, a.rows * a.features);
        split(o.w, steps_w, nv * a.features);
        const int64_t items = (int64_t)o.x.tiles_p * o.x.tiles_q * o.x.splits + (int64_t)o.w.tiles_p * o.w.tiles_q * o.w.splits;
        const int64_t longest = o.x.per > o.w.per ? o.x.per : o.w.per;
        const double all = (total * c.step + items * c.rest) / (256 * c.at_once), one = longest * c.step + c.rest;
        const double t = (all > one ? all : one) + (sums > 0.0 ? 5.0 + sums / 4.5e6 : 0.0);
        if (t < least) {
            least = t;
            best = o;
        }
    }
    return best;
}

Layout backward_layout(const az_linear_ce_args& a) {
    Layout l;
    if (few_backward(a)) {
        l.few = true;
        l.grid = few_grid(a);
        l.fg = l.take(a.classes * 16 * 4);
        // chunks of the classes: about two workgroups per compute unit, but not below 32 classes, where the sums of dx would weigh more
        // than the weights
        const int64_t wide = (a.features + 1023) / 1024;
        int64_t chunks = 512 / wide < 1 ? 1 : 512 / wide;
        if (chunks > (a.classes + 31) / 32) chunks = (a.classes + 31) / 32;
        l.chunk = (int)((a.classes + chunks - 1) / chunks);
        l.chunks = (int)((a.classes + l.chunk - 1) / l.chunk);
        l.sum = l.take((int64_t)l.chunks * a.rows * a.features * 4);
        return l;
    }
    operand_layout(a, l);
    const int64_t np = round_up(a.rows, 64);
    // G and its transpose of a piece stay at about 1 GB: then the sums of dx that travel between pieces cost a few per cent. So does its part of
    // the weight, transposed and perhaps copied (256 x 4096 -> 262144 bfloat16: one piece 3.64 ms, two 3.74, four 4.02).
    int64_t piece = (int64_t(1) << 30) / (np * 4 * l.g_planes) / 256 * 256;
    const int64_t w = (int64_t(1) << 30) / (l.kpitch * l.planes * (l.pack_w ? 2 : 1)) / 256 * 256;
    if (w < piece) piece = w;
    l.piece = piece < 256 ? 256 : piece;
    if (l.piece > a.classes) l.piece = a.classes;
    l.pieces = (int)((a.classes + l.piece - 1) / l.piece);
    const int64_t vp = round_up(l.piece, 64);
    if (l.pack_x) l.xp = l.take(a.rows * l.kpitch * l.planes);
    if (l.pack_w) l.wp = l.take(l.piece * l.kpitch * l.planes);
    if (l.split) {
        l.ux = l.take(a.rows * 4);
        l.uw = l.take(l.piece * 4);
    }
    l.xt = l.take(a.features * np * 2 * l.planes);
    l.wt = l.take(a.features * vp * 2 * l.planes);
    l.g = l.take(a.rows * vp * 2 * l.g_planes);
    l.gt = l.take(l.piece * np * 2 * l.g_planes);
    l.db = l.take((a.rows + 63) / 64 * l.piece * 4);      // the smallest tiles make the most sums
    if (l.pieces > 1) l.sum = l.take(a.rows * a.features * 4);
    // sums of split walks, for the piece that splits most
    int64_t nx = 0, nw = 0;
    for (int i = 0; i < l.pieces; i += l.pieces > 1 ? l.pieces - 1 : 1) {
        const int64_t nv = i + 1 < l.pieces ? l.piece : a.classes - (l.pieces - 1) * l.piece;
        const OutPlan o = out_plan(a, l, nv);
        if (o.x.splits > 1 && o.x.splits * a.rows * a.features * 4 > nx) nx = o.x.splits * a.rows * a.features * 4;
        if (o.w.splits > 1 && o.w.splits * nv * a.features * 4 > nw) nw = o.w.splits * nv * a.features * 4;
    }
    l.walk = l.take(WALK_BYTES);
    l.px = l.take(nx);
    l.pw = l.take(nw);
    l.largest = l.take(16);
    return l;
}

int check_args(const az_linear_ce_args* a) {
    if (!a) return fail(AZ_ERR_ARG, "null argument");
    if (a->dtype != AZ_DT_F32 && a->dtype != AZ_DT_BF16 && a->dtype != AZ_DT_F16) return fail(AZ_ERR_ARG, "dtype is float32, bfloat16 or float16");
    if (a->rows < 1 || a->features < 1 || a->classes < 1) return fail(AZ_ERR_ARG, "rows, features and classes are at least 1");
    if (a->rows > (1 << 30) || a->classes > (1 << 30)) return fail(AZ_ERR_ARG, "rows and classes are at most 2^30");
    if (a->features * 2 > MM_MAX_PITCH - 16 || a->rows * 2 > MM_MAX_PITCH - 128) return fail(AZ_ERR_ARG, "features and rows are at most 4194000");
    if (a->rows * a->features > (int64_t(1) << 34)) return fail(AZ_ERR_ARG, "rows times features are at most 2^34");
    if (!a->x || !a->weight || !a->target) return fail(AZ_ERR_ARG, "null argument");
    if (a->x_pitch < a->features || a->weight_pitch < a->features || (a->target_dense && a->target_pitch < a->classes))
        return fail(AZ_ERR_ARG, "a row stride is smaller than the row");
    if ((a->reduction & ~AZ_PRECISE_GRADIENT) < AZ_REDUCE_NONE || (a->reduction & ~AZ_PRECISE_GRADIENT) > AZ_REDUCE_SUM) return fail(AZ_ERR_ARG, "reduction is none, mean or sum");
    return AZ_OK;
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? AZ_OK : fail(AZ_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

int reduction_of(const az_linear_ce_args& a) { return a.reduction & ~AZ_PRECISE_GRADIENT; }

Rows rows_of(const az_linear_ce_args& a) {
    Rows t;
    t.index = a.target_dense ? nullptr : (const int64_t*)a.target;
    t.dense = a.target_dense ? (const float*)a.target : nullptr;
    t.dense_pitch = a.target_pitch;
    t.ignore = a.ignore_index;
    t.rows = (int)a.rows;
    t.classes = (int)a.classes;
    t.entropy = a.entropy_coeff;
    return t;
}

template <int DT>
void pack(PackArgs& a, hipStream_t st) {
    a.end_w = a.w.blocks();
    a.end_x = a.end_w + a.x.blocks();
    a.end_wt = a.end_x + a.wt.blocks();
    const int64_t n = a.end_wt + a.xt.blocks();
    if (n) hipLaunchKernelGGL((k_pack<DT>), dim3((unsigned)n), dim3(256), 0, st, a);
}

// The pieces of the walk over the features, where there are more than one.
template <int DT, class S>
int walk(const LogitPlan& plan, S& s, char* part, hipStream_t st) {
    s.walk = {plan.pieces, plan.per, (f32x4*)part};
    if (plan.pieces == 1) return AZ_OK;
    typedef typename Tiles<DT>::Small T;
    hipLaunchKernelGGL((k_ce_walk<T, DT>), dim3((unsigned)(s.tiles_p * s.tiles_q * plan.pieces)), dim3(T::THREADS), 0, st, s.w, s.x, s.kbytes, s.tiles_p, s.tiles_q, s.walk);
    return launched("k_ce_walk");
}

template <class T, int DT>
void launch_stats(const StatArgs& s, bool dense, bool ent, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)s.tiles_p * s.tiles_q)), block(T::THREADS);
    if (dense && ent) hipLaunchKernelGGL((k_ce_stats<T, DT, true, true>), grid, block, 0, st, s);
    else if (dense) hipLaunchKernelGGL((k_ce_stats<T, DT, true, false>), grid, block, 0, st, s);
    else if (ent) hipLaunchKernelGGL((k_ce_stats<T, DT, false, true>), grid, block, 0, st, s);
    else hipLaunchKernelGGL((k_ce_stats<T, DT, false, false>), grid, block, 0, st, s);
}

template <class T, int DT>
void launch_grad(const GradArgs& s, bool dense, bool ent, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)s.tiles_p * s.tiles_q)), block(T::THREADS);
    if (dense && ent) hipLaunchKernelGGL((k_ce_grad<T, DT, true, true>), grid, block, 0, st, s);
    else if (dense) hipLaunchKernelGGL((k_ce_grad<T, DT, true, false>), grid, block, 0, st, s);
    else if (ent) hipLaunchKernelGGL((k_ce_grad<T, DT, false, true>), grid, block, 0, st, s);
    else hipLaunchKernelGGL((k_ce_grad<T, DT, false, false>), grid, block, 0, st, s);
}

FewArgs few_args(const az_linear_ce_args& a) {
    FewArgs f{};
    f.w = a.weight;
    f.x = a.x;
    f.bias = a.bias;
    f.w_pitch = a.weight_pitch;
    f.x_pitch = a.x_pitch;
    f.cols = (int)a.features;
    f.share = few_share(a);
    f.t = rows_of(a);
    return f;
}

// The operands of a piece's logits, in place or as copies that `p` is to make (x with the first piece).
template <int DT, class S>
void operands(const az_linear_ce_args& a, const Layout& l, int piece, int64_t nv, const char* w, char* ws, PackArgs& p, S& s) {
    s.w = MmOperand{w, a.weight_pitch * 2, 0, (int)nv};
    s.x = MmOperand{(const char*)a.x, a.x_pitch * 2, 0, (int)a.rows};
    if (l.pack_w) {
        p.w = PackJob{w, a.weight_pitch, (int)nv, (int)a.features, ws + l.wp, l.kpitch, l.piece * l.kpitch, (float*)s.un_w, nullptr, 0};
        s.w = MmOperand{ws + l.wp, l.kpitch, l.piece * l.kpitch, (int)nv};
    }
    if (l.pack_x) {
        if (piece == 0)
            p.x = PackJob{a.x, a.x_pitch, (int)a.rows, (int)a.features, ws + l.xp, l.kpitch, a.rows * l.kpitch, (float*)s.un_x, s.t.index, a.ignore_index};
        s.x = MmOperand{ws + l.xp, l.kpitch, a.rows * l.kpitch, (int)a.rows};
    }
}

struct Kept {      // what the forward pass leaves for the backward one
    float *ref, *inv, *mean, *tsum, *scalars;
    Kept(float* p, int64_t rows) : ref(p), inv(p + rows), mean(p + 2 * rows), tsum(p + 3 * rows), scalars(p + 4 * rows) {}     // 4 of them
};

template <int DT>
int join(const az_linear_ce_args& a, const Layout& l, const StatArgs& s, float* kept, float* loss, float* ce, float* ent, char* ws, hipStream_t st) {
    const Kept k(kept, a.rows);
    const JoinArgs j{s.t, s.part, s.tpart, s.zt, s.tiles, reduction_of(a), k.ref, k.inv, k.mean, k.tsum, k.scalars, (float*)(ws + l.ce), (float*)(ws + l.ce) + a.rows,
                     a.target_dense ? (float*)(ws + l.tabs) : nullptr, loss, ce, ent,
                     l.ux >= 0 ? (float*)(ws + l.ux) : nullptr, l.uw >= 0 ? (float*)(ws + l.uw) : nullptr,
                     l.few ? l.grid : (int)a.rows, l.few ? l.grid : (int)a.classes};
    if (a.rows <= 512 && s.tiles <= 32) {
        hipLaunchKernelGGL(k_ce_join_reduce, dim3(1), dim3(1024), 0, st, j);
    } else {
        const int per = s.tiles > 32 ? 4 : 64;
        hipLaunchKernelGGL(k_ce_join, dim3((unsigned)((a.rows + per - 1) / per)), dim3(256), 0, st, j);
        hipLaunchKernelGGL(k_ce_reduce, dim3(1), dim3(1024), 0, st, j);
    }
    return launched("k_ce_join");
}

template <int DT>
int forward(const az_linear_ce_args& a, float* kept, float* loss, float* ce, float* ent, char* ws, hipStream_t st) {
    const Layout l = forward_layout(a);
    const int edge = forward_edge(a);
    StatArgs s{};
    s.t = rows_of(a);
    if (l.few) {
        FewArgs f = few_args(a);
        s.part = f.part = (f32x4*)(ws + l.part);
        s.tpart = f.tpart = a.target_dense ? (float*)(ws + l.tpart) : nullptr;
        s.zt = f.zt = a.target_dense ? nullptr : (float*)(ws + l.zt);
        s.tiles = l.grid;
        if (DT == DT_F32) {
            f.un_x = (float*)(ws + l.ux);
            f.un_w = (float*)(ws + l.uw);
        }
        const dim3 grid((unsigned)l.grid), block(1024);
        if constexpr (DT == DT_F32) {
            if (a.rows <= 16) hipLaunchKernelGGL((k_ce_few<DT, 1, false>), grid, block, 0, st, f);
            else hipLaunchKernelGGL((k_ce_few<DT, 2, false>), grid, block, 0, st, f);
        } else {
            hipLaunchKernelGGL((k_ce_few<DT, 1, false>), grid, block, 0, st, f);
        }
        if (const int rc = launched("k_ce_few")) return rc;
        return join<DT>(a, l, s, kept, loss, ce, ent, ws, st);
    }
    s.bias = a.bias;
    s.un_x = l.split ? (float*)(ws + l.ux) : nullptr;
    s.part = (f32x4*)(ws + l.part);
    s.tpart = a.target_dense ? (float*)(ws + l.tpart) : nullptr;
    s.zt = a.target_dense ? nullptr : (float*)(ws + l.zt);
    s.tiles = (int)((a.classes + edge - 1) / edge);
    s.tiles_q = (int)((a.rows + edge - 1) / edge);
    s.kbytes = (int)l.kpitch;     // of an operand read in place too: its rows are whole 16 bytes
    for (int i = 0; i < l.pieces; ++i) {
        const int64_t v0 = i * l.piece, nv = a.classes - v0 < l.piece ? a.classes - v0 : l.piece;
        const char* w = (const char*)a.weight + v0 * a.weight_pitch * (l.split ? 4 : 2);
        PackArgs p{};
        s.un_w = l.split ? (float*)(ws + l.uw) + v0 : nullptr;
        operands<DT>(a, l, i, nv, w, ws, p, s);
        pack<DT>(p, st);
        s.v0 = (int)v0;
        s.tile0 = (int)(v0 / edge);
        s.tiles_p = (int)((nv + edge - 1) / edge);
        const bool d = a.target_dense, e = a.entropy_coeff != 0.0f || ent;
        if (const int rc = walk<DT>(logit_plan(a, nv, edge), s, ws + l.walk, st)) return rc;
        if (edge == 256) launch_stats<typename Tiles<DT>::Big, DT>(s, d, e, st);
        else if (edge == 128) launch_stats<typename Tiles<DT>::Mid, DT>(s, d, e, st);
        else launch_stats<typename Tiles<DT>::Small, DT>(s, d, e, st);
        if (const int rc = launched("k_ce_stats")) return rc;
    }
    return join<DT>(a, l, s, kept, loss, ce, ent, ws, st);
}

template <int DT>
int backward(const az_linear_ce_args& a, const Kept& kept, const float* grad, void* gx, void* gw, void* gb, char* ws, hipStream_t st) {
    const Layout l = backward_layout(a);
    if (l.few) {
        FewArgs f = few_args(a);
        f.ref = kept.ref;
        f.inv = kept.inv;
        f.mean = kept.mean;
        f.tsum = kept.tsum;
        f.grad = grad;
        f.scalars = kept.scalars;
        f.each = reduction_of(a) == AZ_REDUCE_NONE;
        f.mean_of = reduction_of(a) == AZ_REDUCE_MEAN;
        f.g = (float*)(ws + l.fg);
        hipLaunchKernelGGL((k_ce_few<DT, 1, true>), dim3((unsigned)l.grid), dim3(1024), 0, st, f);
        if (const int rc = launched("k_ce_few")) return rc;
        const FewOutArgs o{a.weight, a.x, a.weight_pitch, a.x_pitch, (int)a.features, l.chunk, f.t, f.g, gx ? (float*)(ws + l.sum) : nullptr, gw, gb};
        const dim3 grid((unsigned)((a.features + 1023) / 1024), (unsigned)l.chunks), block(256);
        if (a.rows <= 1) hipLaunchKernelGGL((k_ce_few_out<DT, 1>), grid, block, 0, st, o);
        else if (a.rows <= 2) hipLaunchKernelGGL((k_ce_few_out<DT, 2>), grid, block, 0, st, o);
        else if (a.rows <= 4) hipLaunchKernelGGL((k_ce_few_out<DT, 4>), grid, block, 0, st, o);
        else if (a.rows <= 8) hipLaunchKernelGGL((k_ce_few_out<DT, 8>), grid, block, 0, st, o);
        else hipLaunchKernelGGL((k_ce_few_out<DT, 16>), grid, block, 0, st, o);
        const int64_t size = a.rows * a.features;
        if (gx) hipLaunchKernelGGL((k_ce_few_join<DT>), dim3((unsigned)((size + 255) / 256)), dim3(256), 0, st, o.part, l.chunks, size, gx);
        return launched("k_ce_few_out");
    }
    const int esize = l.split ? 4 : 2;
    const int64_t np = round_up(a.rows, 64);
    const bool each = reduction_of(a) == AZ_REDUCE_NONE;
    const float *un_x = l.split ? kept.scalars + 2 : nullptr, *un_w = l.split ? kept.scalars + 3 : nullptr;
    const Factor f{grad, kept.scalars, each ? (const float*)(ws + l.largest) : nullptr, reduction_of(a) == AZ_REDUCE_MEAN, DT != DT_BF16, nullptr, a.target_dense ? nullptr : (const int64_t*)a.target,
                   a.ignore_index};
    if (each) hipLaunchKernelGGL(k_ce_largest, dim3(1), dim3(1024), 0, st, grad, rows_of(a), (float*)(ws + l.largest));
    GradArgs s{};
    s.t = rows_of(a);
    s.bias = a.bias;
    s.un_x = l.split ? (float*)(ws + l.ux) : nullptr;      // the logits are those of the forward pass again, to the bit of their scales
    s.un_w = l.split ? (float*)(ws + l.uw) : nullptr;
    s.kbytes = (int)l.kpitch;     // of an operand read in place too: its rows are whole 16 bytes
    s.ref = kept.ref;
    s.inv = kept.inv;
    s.mean = kept.mean;
    s.tsum = kept.tsum;
    s.f = f;
    s.two = !l.split && l.g_planes == 2;
    s.g = gx ? ws + l.g : nullptr;
    s.gt = gw ? ws + l.gt : nullptr;
    s.gt_pitch = np * 2;
    s.gt_plane = l.piece * np * 2;
    s.db = gb ? (float*)(ws + l.db) : nullptr;
    for (int i = 0; i < l.pieces; ++i) {
        const int64_t v0 = i * l.piece, nv = a.classes - v0 < l.piece ? a.classes - v0 : l.piece;
        const char* w = (const char*)a.weight + v0 * a.weight_pitch * esize;
        const int64_t vpi = round_up(nv, 64);    // k of dx in this piece
        PackArgs p{};
        operands<DT>(a, l, i, nv, w, ws, p, s);
        if (gx) p.wt = TurnJob{w, a.weight_pitch, (int)nv, (int)a.features, ws + l.wt, vpi * 2, a.features * vpi * 2, un_w, nullptr, 0};
        if (gw && i == 0) p.xt = TurnJob{a.x, a.x_pitch, (int)a.rows, (int)a.features, ws + l.xt, np * 2, a.features * np * 2, un_x, s.t.index, a.ignore_index};
        pack<DT>(p, st);
        s.g_pitch = vpi * 2;
        s.g_plane = a.rows * vpi * 2;
        s.v0 = (int)v0;
        s.db_pitch = nv;
        LogitPlan logit = logit_plan(a, nv);
        if (logit.edge > l.edge_most) logit.edge = l.edge_most;
        const int edge = logit.edge;
        s.tiles_p = (int)((nv + edge - 1) / edge);
        s.tiles_q = (int)((a.rows + edge - 1) / edge);
        const bool d = a.target_dense, e = a.entropy_coeff != 0.0f;
        if (const int rc = walk<DT>(logit, s, ws + l.walk, st)) return rc;
        if (edge == 256) launch_grad<typename Tiles<DT>::Big, DT>(s, d, e, st);
        else if (edge == 128) launch_grad<typename Tiles<DT>::Mid, DT>(s, d, e, st);
        else launch_grad<typename Tiles<DT>::Small, DT>(s, d, e, st);
        if (const int rc = launched("k_ce_grad")) return rc;
        const OutPlan plan = out_plan(a, l, nv);
        OutArgs ox{}, ow{};
        ox.p = MmOperand{ws + l.wt, vpi * 2, a.features * vpi * 2, (int)a.features};
        ox.q = MmOperand{ws + l.g, vpi * 2, a.rows * vpi * 2, (int)a.rows};
        ox.kbytes = (int)(vpi * 2);
        ox.out = gx;
        ox.sum = l.pieces > 1 ? (float*)(ws + l.sum) : nullptr;
        ox.first = i == 0;
        ox.last = i == l.pieces - 1;
        ox.by_row = each;
        ox.f = f;
        ox.f.un = un_w;
        ox.part = (float*)(ws + l.px);
        ow.p = MmOperand{ws + l.xt, np * 2, a.features * np * 2, (int)a.features};
        ow.q = MmOperand{ws + l.gt, np * 2, l.piece * np * 2, (int)nv};
        ow.kbytes = (int)(np * 2);
        ow.out = (char*)gw + v0 * a.features * esize;
        ow.first = ow.last = 1;
        ow.f = f;
        ow.f.un = un_x;
        ow.part = (float*)(ws + l.pw);
        auto size = [](OutArgs& o, const OutPlan::Job& j, bool wanted) {
            o.tiles_p = j.tiles_p;
            o.tiles_q = j.tiles_q;
            o.splits = j.splits;
            o.per = j.per;
            return wanted ? (int64_t)j.tiles_p * j.tiles_q * j.splits : 0;
        };
        const int64_t bx = size(ox, plan.x, gx), bw = size(ow, plan.w, gw);
        BiasArgs ob{s.db, s.db_pitch, v0, s.tiles_q, gb ? (int)nv : 0, gb, f};
        // the longer walks first
        const bool swap = plan.w.per > plan.x.per;
        const OutArgs &longer = swap ? ow : ox, &second = swap ? ox : ow;
        const int64_t ba = swap ? bw : bx, bs = swap ? bx : bw;
        auto run = [&](auto tile, auto segments) {
            typedef decltype(tile) T;
            const int64_t bb = (ob.classes + T::THREADS - 1) / T::THREADS;
            hipLaunchKernelGGL((k_ce_out<T, DT, decltype(segments)::value>), dim3((unsigned)(ba + bs + bb)), dim3(T::THREADS), 0, st, longer, second, ob, (int)ba, (int)bs);
        };
        const std::integral_constant<int, DT == DT_F32 ? MM_SEGMENTS : 1> usual;
        const std::integral_constant<int, DT == DT_F32 ? MM_SEGMENTS : 2> two;
        if (plan.edge == 256) run(typename Tiles<DT>::Big{}, usual);
        else if (plan.edge == 128 && s.two) run(typename Tiles<DT>::Mid{}, two);
        else if (plan.edge == 128) run(typename Tiles<DT>::Mid{}, usual);
        else if (s.two) run(typename Tiles<DT>::Small{}, two);
        else run(typename Tiles<DT>::Small{}, usual);
        if (const int rc = launched("k_ce_out")) return rc;
        const int64_t jx = bx && ox.splits > 1 ? (a.rows * a.features + 255) / 256 : 0, jw = bw && ow.splits > 1 ? (nv * a.features + 255) / 256 : 0;
        if (jx + jw) hipLaunchKernelGGL((k_ce_out_join<DT>), dim3((unsigned)(jx + jw)), dim3(256), 0, st, ox, ow, jx);
    }
    return launched("k_ce_out_join");
}

}  // namespace
}  // namespace az

#define AZ_HEAD_UNIT(NAME, DT)                                                                                                              \
    namespace az {                                                                                                                          \
    int ce_forward_##NAME(const az_linear_ce_args& a, float* kept, float* loss, float* ce, float* ent, char* ws, hipStream_t st) {            \
        return forward<DT>(a, kept, loss, ce, ent, ws, st);                                                                                 \
    }                                                                                                                                       \
    int ce_backward_##NAME(const az_linear_ce_args& a, const float* kept, const float* grad, void* gx, void* gw, void* gb, char* ws,          \
                           hipStream_t st) {                                                                                                \
        return backward<DT>(a, Kept(const_cast<float*>(kept), a.rows), grad, gx, gw, gb, ws, st);                                            \
    }                                                                                                                                       \
    }
