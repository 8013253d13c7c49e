// Tile loop of the matrix products of the head operators (az_head.cuh, az_int8.hip): C[p][q] = sum_k P[p][k] * Q[q][k], both
// operands with k contiguous, 16-bit floats or 8-bit integers, accumulated in 32 bits.
//
// A workgroup owns BP x BQ results and walks k in steps of 128 bytes (64 16-bit or 128 8-bit values). A step's BP + BQ rows of
// 128 bytes go from global memory to LDS without passing through registers (buffer_load_dwordx4 ... lds, 1 KB = 8 rows per wave
// and instruction), into STAGES stages of which all but the one in use are on their way. The load writes a wave's 64 x 16 bytes
// contiguously, so the bank permutation is made on the global side: the lane that writes 16-byte piece c of row r fetches piece
// c ^ (r & 7), and a fragment read (16 rows, one piece each) then touches all banks evenly. Reads behind the last row or the last k of
// a matrix are turned into zeros by the buffer descriptor's range check, so ragged sizes need no other code.
//
// Measured with the 256 x 256 tile of 8 waves: 8192 x 8192 results over 4096 bfloat16 1.43 PFLOP/s, over 8192 int8 2.2 to 2.6 POP/s by
// card (power). A step takes 2912 cycles at the 2.05 GHz that the power limit leaves, 2048 of them the matrix instruction's; without the
// fetches the loop reaches 1.83, without the fragment reads 1.6 PFLOP/s. 64-byte steps in 3 to 5 stages: 1.36. Four waves of 128 x 128,
// which read a third less from LDS, have nobody to hide their waits: 1.25. Left to the compiler's order of reads and products: 1.41.
//
// P is the matrix instruction's row operand: lane l then holds results p = 4 * (l >> 4) + 0..3 of column q = l & 15 of each
// 16 x 16 tile, i.e. four neighbouring p of one q. Callers put the axis that is contiguous in their output (classes, features)
// on P, and a softmax over P is mostly inside a lane.
//
// float32 operands come as two float16 planes, v = h + m / 2048 (split2), scaled by powers of two beforehand. k is walked three times,
// first with the plane pairs (h, m) and (m, h), whose sum is then divided by 2048, then with (h, h); (m, m) / 2^22 is below
// 2^-24 of the result and left out. Each product keeps 22 bits or more, of values down to 2^-27 of the largest with the same scale; the
// sum is float32's: 2.5 PFLOP/s / 3 against the 0.16 PFLOP/s of the float32 matrix instructions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "az_types.cuh"

namespace az {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum { MM_BF16 = 0, MM_F16 = 1, MM_I8 = 2 };

struct MmOperand {
    const char* base;    // 16-byte aligned
    int64_t pitch;       // bytes between rows, a multiple of 16, at most MM_MAX_PITCH
    int64_t plane;       // bytes between the planes of a split float32 operand
    int32_t rows;
    int32_t short_by;    // bytes that the last row lacks of kbytes (whole 4 bytes, fewer than 16): they are not read and count as zero
};
constexpr int64_t MM_MAX_PITCH = (int64_t(1) << 31) / 256 - 16;   // 256 rows of a tile stay below 2^31 bytes

template <int KIND> struct MmAcc { typedef f32x4 type; };
template <> struct MmAcc<MM_I8> { typedef i32x4 type; };

template <int KIND>
__device__ __forceinline__ typename MmAcc<KIND>::type mm_mfma(i32x4 a, i32x4 b, typename MmAcc<KIND>::type c) {
    if constexpr (KIND == MM_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else if constexpr (KIND == MM_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

template <int BP_, int BQ_, int WP_, int WQ_, int STAGES_, int KIND_>
struct MmTile {
    static constexpr int BP = BP_, BQ = BQ_, WP = WP_, WQ = WQ_, STAGES = STAGES_, KIND = KIND_;
    static constexpr int WAVES = WP * WQ, THREADS = WAVES * 64;
    static constexpr int TP = BP / WP, TQ = BQ / WQ;          // a wave's share
    static constexpr int FP = TP / 16, FQ = TQ / 16;
    static constexpr int LP = BP / 8 / WAVES, LQ = BQ / 8 / WAVES;   // 1 KB loads of a wave per stage
    static constexpr int STAGE = (BP + BQ) * 128;
    static constexpr int LDS = STAGES * STAGE;
    static_assert(LDS <= 160 * 1024 && BP * BQ * 2 <= LDS && (STAGES - 1) * (LP + LQ) < 64, "LDS, the results' image in it, the counter of loads");
    static_assert(BP % (8 * WAVES) == 0 && BQ % (8 * WAVES) == 0 && TP % 16 == 0 && TQ % 16 == 0, "tile shape");
    typedef typename MmAcc<KIND>::type acc_t;
};

// Planes of segment s of 3: (h, m) (m, h) (h, h).
// With planes of Q only (P is 16-bit by itself) it is walked twice: m, then h. Planes of bfloat16 keep their exponent, m is not scaled.
constexpr int MM_SEGMENTS = 3;

// One tile: acc[i][j] = results p = p0 + wp * TP + 16 i + 4 (lane >> 4) + 0..3, q = q0 + wq * TQ + 16 j + (lane & 15), where
// wave = wp * WQ + wq. kbytes: bytes of k per row (a multiple of 16). k_first / k_last: the 128-byte steps [k_first, k_last) of
// the walk of ceil(kbytes / 128) steps for each of `segments` (1, 2 or 3) that this workgroup takes. All lanes of the workgroup call it; on
// return every wave has read its last fragment and passed a barrier, so the LDS may be used for something else.
template <class T>
__device__ __forceinline__ void mm_tile(const MmOperand& P, const MmOperand& Q, int64_t p0, int64_t q0, int kbytes, int k_first, int k_last,
                                        int segments, char* lds, typename T::acc_t (&acc)[T::FP][T::FQ]) {
#ifdef __HIP_DEVICE_COMPILE__   // the buffer resource type exists on the device only
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave / T::WQ, wq = wave % T::WQ;
    const int ksteps = (kbytes + 127) >> 7;
    const int row8 = lane >> 3, piece = (lane & 7) ^ row8;
    const int pp = (int)P.pitch, qp = (int)Q.pitch;
    int offp[T::LP], offq[T::LQ];
#pragma unroll
    for (int i = 0; i < T::LP; ++i) offp[i] = ((wave + i * T::WAVES) * 8 + row8) * pp + piece * 16;
#pragma unroll
    for (int i = 0; i < T::LQ; ++i) offq[i] = ((wave + i * T::WAVES) * 8 + row8) * qp + piece * 16;
    const char* const pbase = P.base + p0 * P.pitch;
    const char* const qbase = Q.base + q0 * Q.pitch;
    // bytes from the tile's first row to the end of the matrix' last row; below zero (an empty tile) reads nothing
    const int64_t pext = ((int64_t)P.rows - p0 - 1) * P.pitch + kbytes - P.short_by, qext = ((int64_t)Q.rows - q0 - 1) * Q.pitch + kbytes - Q.short_by;
    int ks = segments > 1 ? k_first / ksteps : 0;      // segment and step within it of the next stage to fetch
    int kk = k_first - ks * ksteps;
    int left = k_last - k_first;                // stages still to fetch

    // A stage past the last one is fetched too, out of range of an empty matrix: zeros arrive and the loop needs no branch.
    auto fetch = [&](int stage) {
        const int k = kk << 7;
        const char* pb = pbase + k;
        const char* qb = qbase + k;
        if (segments == 3) pb += (ks == 1) * P.plane;
        if (segments > 1) qb += (ks == 0) * Q.plane;
        const int64_t pn = pext - k, qn = qext - k;
        const bool none = left <= 0;
        const int pr = pn < 0 || none ? 0 : (pn > 0x7fffffff ? 0x7fffffff : (int)pn), qr = qn < 0 || none ? 0 : (qn > 0x7fffffff ? 0x7fffffff : (int)qn);
        const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void*)pb, 0, pr, 0x00020000);
        const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void*)qb, 0, qr, 0x00020000);
        // pieces behind the row's end would read the next row: sent out of range instead
        const int past = k + piece * 16 >= kbytes ? (int)0x80000000 : 0;
        char* dst = lds + stage + wave * 1024;
#pragma unroll
        for (int i = 0; i < T::LP; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rp, (__attribute__((address_space(3))) void*)(dst + i * T::WAVES * 1024), 16, offp[i] | past, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < T::LQ; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, (__attribute__((address_space(3))) void*)(dst + T::BP * 128 + i * T::WAVES * 1024), 16, offq[i] | past, 0, 0, 0);
        --left;
        if (++kk == ksteps) {
            kk = 0;
            ++ks;
        }
    };
    // fragment reads: 16 rows x 16 bytes, half h of the step; piece h * 4 + (lane >> 4) of row r sits at piece ^ (r & 7)
    const int frow = lane & 15, fq4 = lane >> 4;
    const int sw0 = ((fq4 ^ (frow & 7)) * 16), sw1 = (((4 + fq4) ^ (frow & 7)) * 16);
    const int rdp = (wp * T::TP + frow) * 128, rdq = T::BP * 128 + (wq * T::TQ + frow) * 128;
    auto read = [&](int stage, int sw, i32x4 (&a)[T::FP], i32x4 (&b)[T::FQ]) {
        const char* s = lds + stage + sw;
#pragma unroll
        for (int j = 0; j < T::FQ; ++j) b[j] = *(const i32x4*)(s + rdq + j * 2048);
#pragma unroll
        for (int i = 0; i < T::FP; ++i) a[i] = *(const i32x4*)(s + rdp + i * 2048);
    };
    auto multiply = [&](const i32x4 (&a)[T::FP], const i32x4 (&b)[T::FQ]) {
#pragma unroll
        for (int i = 0; i < T::FP; ++i)
#pragma unroll
            for (int j = 0; j < T::FQ; ++j) acc[i][j] = mm_mfma<T::KIND>(a[i], b[j], acc[i][j]);
    };
    // all but the last `flying` stages' loads of this wave have landed and every fragment read has returned, for all waves; nothing is
    // moved across
    auto meet = [](auto flying) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(flying)::value * (T::LP + T::LQ)) : "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // half a step: fragment reads spread among the products (and, in the second half, the loads of the next stage)
    auto weave = [](auto loads) {
        constexpr int R = T::FP + T::FQ, M = T::FP * T::FQ, L = decltype(loads)::value, PER = M / R > 0 ? M / R : 1;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                       // a read
            if (i < L) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);            // a load
            __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);                     // products
        }
    };

#pragma unroll
    for (int i = 0; i < T::FP; ++i)
#pragma unroll
        for (int j = 0; j < T::FQ; ++j) acc[i][j] = typename T::acc_t{};
    const int n = k_last - k_first;
    if (n <= 0) return;
    i32x4 a0[T::FP], b0[T::FQ], a1[T::FP], b1[T::FQ];
#pragma unroll
    for (int i = 0; i < T::STAGES; ++i) fetch(i * T::STAGE);
    meet(std::integral_constant<int, T::STAGES - 1>{});
    read(0, sw0, a0, b0);
    int s = 0;
    const int turn = segments > 1 ? (segments - 1) * ksteps - k_first : -1;      // the step that the (h, h) segment starts with
    auto lower = [&] {
        if constexpr (T::KIND == MM_F16)
#pragma unroll
            for (int i = 0; i < T::FP; ++i)
#pragma unroll
                for (int j = 0; j < T::FQ; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] *= 1.0f / 2048.0f;
    };
    for (int t = 0; t < n; ++t) {
        if (t == turn) lower();
        read(s, sw1, a1, b1);
        multiply(a0, b0);
        weave(std::integral_constant<int, 0>{});
        meet(std::integral_constant<int, T::STAGES - 2>{});     // stage t + 1 is in LDS, stage t has been read by all
        fetch(s);
        s = s == (T::STAGES - 1) * T::STAGE ? 0 : s + T::STAGE;
        read(s, sw0, a0, b0);
        multiply(a1, b1);
        weave(std::integral_constant<int, T::LP + T::LQ>{});
        __builtin_amdgcn_sched_barrier(0);
    }
    meet(std::integral_constant<int, 0>{});
    if (segments > 1 && turn >= n) lower();      // a piece of the walk that ends before it
#endif
}

// ---- 16-bit results of a tile on their way to memory --------------------------------------------------------------------
// The lanes hold four neighbouring p of a q; written directly, an instruction would touch 16 rows with 32 bytes each. The tile goes
// through the LDS of its stages instead (all waves are past their last fragment read) and leaves in whole 16-byte pieces, 512
// bytes of a row after another. Piece c of image row r sits at c ^ r, so neither side meets a bank twice.
// bits(i, j) gives the four values of fragment (i, j) as two words.
template <class T, class F>
__device__ __forceinline__ void mm_stage(char* lds, F bits) {      // image [q][p]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wp = wave / T::WQ, wq = wave % T::WQ;
#pragma unroll
    for (int j = 0; j < T::FQ; ++j) {
        const int q = wq * T::TQ + j * 16 + (lane & 15);
#pragma unroll
        for (int i = 0; i < T::FP; ++i) {
            const int c = (wp * T::TP + i * 16) / 8 + (lane >> 5);
            *(uint2*)(lds + q * (T::BP * 2) + ((c ^ (q & (T::BP / 8 - 1))) * 16) + ((lane >> 4) & 1) * 8) = bits(i, j);
        }
    }
}
template <class T, class F>
__device__ __forceinline__ void mm_stage_turned(char* lds, F bits) {   // image [p][q]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wp = wave / T::WQ, wq = wave % T::WQ;
    const bool odd = lane & 1;
#pragma unroll
    for (int j = 0; j < T::FQ; ++j) {
        const int q = wq * T::TQ + j * 16 + (lane & 14);
#pragma unroll
        for (int i = 0; i < T::FP; ++i) {
            // neighbouring lanes hold neighbouring q: the even one takes both values of the first two p, the odd one of the last two
            const uint2 v = bits(i, j);
            const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(odd ? v.x : v.y), 0xB1, 0xF, 0xF, true);
            const uint32_t lo = odd ? got : v.x, hi = odd ? v.y : got;
            const int p = wp * T::TP + i * 16 + (lane >> 4) * 4 + (odd ? 2 : 0), c = q >> 3;
            char* at = lds + p * (T::BQ * 2) + (q & 7) * 2;
            *(uint32_t*)(at + ((c ^ (p & (T::BQ / 8 - 1))) * 16)) = (lo & 0xffffu) | (hi << 16);
            *(uint32_t*)(at + T::BQ * 2 + ((c ^ ((p + 1) & (T::BQ / 8 - 1))) * 16)) = (lo >> 16) | (hi & 0xffff0000u);
        }
    }
}
// An image of ROWS x COLS to dst: rows and bytes beyond `rows` / `bytes` are left out. Rows may start anywhere.
template <class T, int ROWS, int COLS>
__device__ __forceinline__ void mm_unstage(const char* lds, char* dst, int64_t pitch, int64_t rows, int64_t bytes) {
    constexpr int C = COLS / 8;
#pragma unroll
    for (int k = 0; k < ROWS * C / T::THREADS; ++k) {
        const int at = k * T::THREADS + threadIdx.x, r = at / C, c = at % C;
        if (r >= rows || c * 16 >= bytes) continue;
        const uint4 v = *(const uint4*)(lds + r * (COLS * 2) + ((c ^ (r & (C - 1))) * 16));
        char* o = dst + r * pitch + c * 16;
        if (c * 16 + 16 <= bytes) {
            __builtin_memcpy(o, &v, 16);
        } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c * 16 + e * 2 < bytes) *(uint16_t*)(o + e * 2) = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        }
    }
}

// The lane, as a value that the compiler knows nothing of: what is computed from it stays behind the tile loop, instead of taking
// registers through it.
__device__ __forceinline__ int mm_lane_after() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

template <class T>
__device__ __forceinline__ void mm_opaque(typename T::acc_t (&acc)[T::FP][T::FQ]) {
#pragma unroll
    for (int i = 0; i < T::FP; ++i)
#pragma unroll
        for (int j = 0; j < T::FQ; ++j) asm volatile("" : "+v"(acc[i][j]));
}

// Place of a workgroup in a walk over `total` of them: consecutive ids go round the 8 XCDs, so each XCD gets a contiguous stretch.
__device__ __forceinline__ int mm_stretch(int id, int total) {
    const int per = total >> 3, rest = total & 7, xcd = id & 7;
    return xcd * per + (xcd < rest ? xcd : rest) + (id >> 3);
}
// Workgroup id -> piece of k and tile, for few tiles whose walk over k is split: a stretch has whole pieces or parts of one, in which the
// tiles that read the same strip of the longer side follow each other.
__device__ __forceinline__ void mm_place_piece(int id, int pieces, int tiles_p, int tiles_q, int& piece, int& tp, int& tq) {
    const int tiles = tiles_p * tiles_q, l = mm_stretch(id, tiles * pieces), t = l % tiles;
    piece = l / tiles;
    const bool wide = tiles_p >= tiles_q;
    tp = wide ? t / tiles_q : t % tiles_p;
    tq = wide ? t % tiles_q : t / tiles_p;
}
// Workgroup id -> tile (p, q): consecutive ids go round the 8 XCDs, so each XCD gets a contiguous stretch of the walk, and the
// walk goes through groups of 8 p tiles with q outermost inside a group: the 32 tiles that an XCD works on at a time are about
// 8 x 4, which read 12 operand strips through its L2 instead of 33.
__device__ __forceinline__ void mm_place(int id, int tiles_p, int tiles_q, int& tp, int& tq) {
    const int l = mm_stretch(id, tiles_p * tiles_q);
    const int group = l / (8 * tiles_q), in = l - group * 8 * tiles_q;
    const int width = tiles_p - group * 8 < 8 ? tiles_p - group * 8 : 8;
    tp = group * 8 + in % width;
    tq = in / width;
}

// ---- host: which tile -----------------------------------------------------------------------------------------------------
// What the tiles were measured to take, in microseconds: a step (128 bytes of k), and a tile beside its steps (first loads, results), with as
// many of them on a compute unit at a time as its LDS holds. 4096 x 722 -> 362 float16 dense: 64 tiles 14.8 (logits) and 17.1 us (G), 128
// tiles 22.1 and 32.4; 7955 x 3877 -> 829: 128 tiles 79; 809 x 437 -> 20359: 256 tiles 37 and 54, 128 tiles 37 and 48.
struct MmTileCost {
    int edge, at_once;
    double step, rest;
};
constexpr MmTileCost MM_TILE_COSTS[3] = {{256, 1, 1.5, 8.0}, {128, 2, 1.1, 6.0}, {64, 2, 0.8, 4.0}};

// Tile edge for p x q results of sums over `steps` steps: rounds of tiles over the compute units, times a tile.
inline int mm_tile_edge(int64_t p, int64_t q, int64_t steps) {
    int best = 256;
    double least = 1e300;
    for (const MmTileCost& c : MM_TILE_COSTS) {
        const int64_t tiles = ((p + c.edge - 1) / c.edge) * ((q + c.edge - 1) / c.edge), round = 256 * c.at_once;
        const double t = (double)((tiles + round - 1) / round) * (steps * c.step + c.rest);
        if (t < least) {
            least = t;
            best = c.edge;
        }
    }
    return best;
}

}  // namespace az
