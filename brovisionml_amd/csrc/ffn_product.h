// C[m][n] = sum_k P(m, k) Q(n, k) on the matrix cores, with the feed-forward
// operators' epilogues: the kernel behind the forward products and, with one
// or both operands read across their rows, behind both gradients.
//
//   forward       P = x,  k along its rows      Q = W,  k along its rows
//   input's       P = dz, k along its rows      Q = W,  k across its rows
//   weight's      P = dz, k across its rows     Q = x,  k across its rows
//
// A workgroup of WM x WN waves owns a BM x BN tile of C; a wave its
// (BM / WM) x (BN / WN) part, in fp32 accumulators.  Per step the two
// operands' next 128 bytes of k go to LDS (two stages; the copy of step s + 1
// is in flight while step s is multiplied), from which every wave reads its
// rows as 16-byte matrix operands.  Q is the instruction's first operand, so
// that a lane holds neighbouring columns of one row of C.
//
// LDS layout, operand with k along its rows: 128 bytes a row, its 16-byte
// pieces permuted by the row (piece ^ key) so that the 16 rows a matrix
// operand reads at once fall into different banks.  The rows of Q go to the
// instruction's rows in an order that leaves a lane with 4 NB (gated: 2 NB)
// neighbouring columns of C, so that it stores 16 bytes at a time.
// Operand with k across its rows: one k a row, its pieces permuted by k; the
// transposing LDS read hands each lane four k of one column.
//
// Copies go straight from memory to LDS where every row begins on 16 bytes
// (DMA); otherwise through registers at any alignment.  Rows beyond the
// operand repeat its last one (their results are not stored); k beyond its
// end reads as zero: by the buffer descriptor's bound or by an offset past it.
#pragma once

#include <type_traits>

#include "ffn_common.h"

namespace bvml_ffn {

struct Product {
    const char* p;          // first operand, rows are C's rows
    const char* q;          // second operand, rows are C's columns
    long long ldp, ldq;     // bytes from row to row in memory
    int M, K;               // C's rows; the sum's length
    int R;                  // Q's columns of C: N, or 2N for the gated form
    int tiles_m, tiles_n;
    int steps;              // ceil(K / kStep): all of them
    int per_split;          // steps a workgroup takes (blockIdx.y: which)
    Epilogue e;
};

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

#define BVML_LDS(T, p) ((__attribute__((address_space(3))) T*)(p))

constexpr int kBufferWord3 = 0x00020000;      // gfx9 raw-buffer descriptor word 3
constexpr uint32_t kBufferEnd = 0x7fffffffu;  // the longest range a descriptor gets here
constexpr int kPastEnd = (int)0x80000000u;    // an offset past any of them: reads zeros

template <int kIn>
__device__ __forceinline__ v4f multiply16(v8s a, v8s b, v4f c) {
    if constexpr (kIn == kBF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a),
                                                       __builtin_bit_cast(v8b, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                      __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
// 128 products of 8-bit values a row; no block scales
__device__ __forceinline__ v4f multiply8(v8i a, v8i b, v4f c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

// Which 32-byte slot a k row's pieces move by: different for the 8 rows that
// a transposing read touches at once (k = q + 8 g, q < 4, g < 2).
template <int kCols>
__device__ __forceinline__ int slot_key(int k) {
    return kCols >= 128 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2);
}

// 16 bytes a lane from the buffer at `off` to LDS at `to` + 16 lane, counted by
// vmcnt; nothing comes back to a register.  In assembly, because the compiler
// makes every LDS read after the builtin wait for all of these copies, those
// into the other stage among them: the kernel waits where a stage is due.
__device__ __forceinline__ void copy_to_lds(v4i rsrc, int off, char* to) {
    const uint32_t at = (uint32_t)reinterpret_cast<uintptr_t>(BVML_LDS(char, to));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(at), "v"(off), "s"(rsrc)
                 : "memory", "m0");
}

// One operand's copy into an LDS tile of kRows x 128 bytes (or, transposed,
// kStep k rows of kRows 16-bit columns).
template <int kIn, int kRows, int kWaves, bool kT, bool kDma>
struct Copy {
    static constexpr int kSize = kIn == kE4M3 ? 1 : 2;
    static constexpr int kPiece = 16 / kSize;  // elements of 16 bytes
    static constexpr int kStep = 128 / kSize;  // k of one step
    static constexpr int kParts = kRows / 8 / kWaves;
    static constexpr int kChunks = kRows / 8;  // pieces of a transposed row
    static_assert(kRows % (8 * kWaves) == 0, "whole copies a wave");

    int off[kParts];    // per-lane byte offset from the tile's base
    int piece;          // k along rows: the lane's first k in the step
    v4i held[kDma ? 1 : kParts];

    // rows: how many the operand has from the tile's base on
    // key_shift: the row bit that is the key's third bit (0: row & 7)
    __device__ __forceinline__ void init(int w, int lane, long long ld, int rows, int key_shift,
                                         int t0, int t1) {
        if constexpr (!kT) {
            const int r0 = w * 8 + (lane >> 3);
            const int key = key_shift ? (r0 & 3) | (((w * 8) >> key_shift & 1) << 2) : r0 & 7;
            const int c = (lane & 7) ^ key;
            piece = c * kPiece;
#pragma unroll
            for (int t = 0; t < kParts; ++t) {
                if (t < t0 || t >= t1) continue;
                const int row = (t - t0) * kWaves * 8 + r0;
                off[t] = (int)((row < rows ? row : rows - 1) * ld) + c * 16;
            }
        } else {
            piece = 0;
#pragma unroll
            for (int t = 0; t < kParts; ++t) {
                const int pos = (t * kWaves + w) * 64 + lane;
                const int k = pos / kChunks;
                const int c = (pos % kChunks) ^ (slot_key<kRows>(k) << 1);
                // an offset past the end for columns beyond the operand
                off[t] = c * 8 < rows ? (int)(k * ld) + c * 16 : kPastEnd;
            }
        }
    }

    // Starts the copy of the step whose first k is k0 (left of them remain);
    // base points at the tile's first row (transposed: at row k0).
    __device__ __forceinline__ void start(const char* base, long long ld, int left, int rows,
                                          int w, int lane, char* to, int t0, int t1) {
        if constexpr (kDma) {
            uint32_t bytes = kBufferEnd;
            if constexpr (kT) {
                const long long have = (long long)left * ld;
                bytes = have < (long long)kBufferEnd ? (uint32_t)have : kBufferEnd;
            }
            const uint64_t at = reinterpret_cast<uint64_t>(base);
            const v4i rs = {(int)(uint32_t)at, (int)(uint32_t)(at >> 32) & 0xffff, (int)bytes,
                            kBufferWord3};
            const bool in = kT || piece < left;
#pragma unroll
            for (int t = 0; t < kParts; ++t) {
                if (t < t0 || t >= t1) continue;
                copy_to_lds(rs, in ? off[t] : kPastEnd, to + (t * kWaves + w) * 1024);
            }
        } else {
#pragma unroll
            for (int t = 0; t < kParts; ++t) {
                if (t < t0 || t >= t1) continue;
                int n;  // elements of the piece inside the operand
                if constexpr (kT) {
                    const int pos = (t * kWaves + w) * 64 + lane;
                    const int k = pos / kChunks;
                    const int c = (pos % kChunks) ^ (slot_key<kRows>(k) << 1);
                    n = k < left ? rows - c * 8 : 0;
                } else {
                    n = left - piece;
                }
                v4i v = {0, 0, 0, 0};
                const char* from = base + off[t];
                if (n >= kPiece) {
                    __builtin_memcpy(&v, from, 16);
                } else if (n > 0) {
                    if constexpr (kSize == 2) {
                        uint16_t h[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            h[i] = i < n ? reinterpret_cast<const uint16_t*>(from)[i]
                                         : (uint16_t)0;
                        __builtin_memcpy(&v, h, 16);
                    } else {
                        uint8_t h[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            h[i] = i < n ? reinterpret_cast<const uint8_t*>(from)[i] : (uint8_t)0;
                        __builtin_memcpy(&v, h, 16);
                    }
                }
                held[t] = v;
            }
        }
    }
    // Without DMA: what start() read, into LDS.
    __device__ __forceinline__ void commit(int w, int lane, char* to) {
        if constexpr (!kDma) {
#pragma unroll
            for (int t = 0; t < kParts; ++t)
                *reinterpret_cast<v4i*>(to + (t * kWaves + w) * 1024 + lane * 16) = held[t];
        }
    }
};

// The tile of workgroup `b` of n: consecutive tiles on one XCD (workgroups go
// round the 8 of them), so that its L2 serves the operand rows they share,
// and within that groups of kGroup row tiles by all column tiles.
constexpr int kXcds = 8;
constexpr int kGroup = 4;

__device__ __forceinline__ void tile_of(int b, int tm, int tn, int& m, int& n) {
    const int total = tm * tn, each = total / kXcds, more = total % kXcds;
    const int x = b % kXcds, i = b / kXcds;
    const int t = x * each + (x < more ? x : more) + i;
    const int per = kGroup * tn, g = t / per, in = t % per;
    const int rows = tm - g * kGroup < kGroup ? tm - g * kGroup : kGroup;
    m = g * kGroup + in % rows;
    n = in / rows;
}

template <int kIn, int BM, int BN, int WM, int WN, bool kPT, bool kQT, bool kGated, bool kDma>
__global__ __launch_bounds__(64 * WM * WN, 2) void product_kernel(Product a) {
    constexpr int kWaves = WM * WN;
    constexpr int MT = BM / WM, NT = BN / WN, MB = MT / 16, NB = NT / 16;
    constexpr int kSize = kIn == kE4M3 ? 1 : 2;
    constexpr int kStep = 128 / kSize;
    constexpr int kPBytes = BM * 128, kQBytes = BN * 128;
    // neighbouring columns of C a lane ends up with
    constexpr int kRun = kQT ? 4 : kGated ? 2 * NB : 4 * NB;
    constexpr int kVec = kRun < 8 ? kRun : 8;  // columns of one store
    constexpr int kKeyShift = kRun == 4 ? 0 : kRun == 8 ? 3 : kRun == 16 ? 4 : 5;
    static_assert(kQT || kKeyShift == 0 || kWaves % (1 << (kKeyShift - 2)) == 0, "one key a lane");
    static_assert(!(kGated && kQT) && !(kPT && kIn == kE4M3) && !(kQT && kIn == kE4M3), "");

    constexpr int kStage = kPBytes + kQBytes;
    static_assert((kStage & (kStage - 1)) == 0, "the other stage is one bit away");
    __shared__ __align__(1024) char lds[2 * kStage];

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = w / WN, wn = w % WN;
    int tm, tn;
    tile_of(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * (kGated ? BN / 2 : BN);
    const int step0 = blockIdx.y * a.per_split;
    const int step1 = step0 + a.per_split < a.steps ? step0 + a.per_split : a.steps;

    // ---- copies
    Copy<kIn, BM, kWaves, kPT, kDma> cp;
    Copy<kIn, BN, kWaves, kQT, kDma> cq;
    constexpr int PP = BM / 8 / kWaves, QP = BN / 8 / kWaves, QH = kGated ? QP / 2 : QP;
    static_assert(!kGated || QP % 2 == 0, "a copy belongs to the gate or to the other half");
    const int rows_p = a.M - m0;
    const int rows_q = (kGated ? a.R / 2 : a.R) - n0;
    cp.init(w, lane, a.ldp, rows_p, 0, 0, PP);
    cq.init(w, lane, a.ldq, rows_q, kKeyShift, 0, QH);
    if constexpr (kGated) cq.init(w, lane, a.ldq, rows_q, kKeyShift, QH, QP);
    const char* pb = kPT ? a.p + (long long)m0 * 2 : a.p + (long long)m0 * a.ldp;
    const char* qb = kQT ? a.q + (long long)n0 * 2 : a.q + (long long)n0 * a.ldq;
    const char* qb2 = kGated ? qb + (long long)(a.R / 2) * a.ldq : qb;

    auto start = [&](int step, char* to) {
        const int k0 = step * kStep, left = a.K - k0;
        const long long ap = kPT ? k0 * a.ldp : (long long)k0 * kSize;
        const long long aq = kQT ? k0 * a.ldq : (long long)k0 * kSize;
        cp.start(pb + ap, a.ldp, left, rows_p, w, lane, to, 0, PP);
        cq.start(qb + aq, a.ldq, left, rows_q, w, lane, to + kPBytes, 0, QH);
        if constexpr (kGated)
            cq.start(qb2 + aq, a.ldq, left, rows_q, w, lane, to + kPBytes, QH, QP);
    };
    auto commit = [&](char* to) {
        cp.commit(w, lane, to);
        cq.commit(w, lane, to + kPBytes);
    };

    // ---- where the lane's operands are in a stage
    const int g = lane >> 4, i16 = lane & 15;
    int pat[kPT ? MB : 1], qat[kQT ? NB : 1];
    if constexpr (kPT) {
        const int k = 8 * g + (i16 >> 2);
        const int c = (wm * MT) / 8 + ((i16 & 3) >> 1);
#pragma unroll
        for (int i = 0; i < MB; ++i)
            pat[i] = k * BM * 2 + (((c + 2 * i) ^ (slot_key<BM>(k) << 1)) << 4) + (i16 & 1) * 8;
    } else {
        pat[0] = (wm * MT + i16) * 128 + ((g ^ (i16 & 7)) << 4);
    }
    if constexpr (kQT) {
        const int k = 8 * g + (i16 >> 2);
        const int c = (wn * NT) / 8 + ((i16 & 3) >> 1);
#pragma unroll
        for (int j = 0; j < NB; ++j)
            qat[j] = kPBytes + k * BN * 2 + (((c + 2 * j) ^ (slot_key<BN>(k) << 1)) << 4) +
                     (i16 & 1) * 8;
    } else {
        const int row = (kGated ? wn * (NT / 2) : wn * NT) + kRun * (i16 >> 2) + (i16 & 3);
        qat[0] = kPBytes + row * 128 + ((g ^ (i16 & 7)) << 4);
    }

    v4f acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};

    // the j-th 16 rows of Q, k-along-rows layout, relative to qat
    auto qrow = [](int j) {
        return kGated && j >= NB / 2 ? (BN / 2 + 4 * (j - NB / 2)) * 128 : 4 * j * 128;
    };
    auto across = [](const char* at, int cols) {  // 8 k of a column
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(BVML_LDS(v4s, at));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(BVML_LDS(v4s, at + 8 * cols));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto both = [](const char* s, int at) {  // pieces g and g + 4 of a row
        const v4i lo = *reinterpret_cast<const v4i*>(s + at);
        const v4i hi = *reinterpret_cast<const v4i*>(s + (at ^ 64));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };

    // A step is kPhases groups of products, one k group (16 bits: 32 of the
    // 64) by one part of the wave's rows; each phase's operands are read from
    // LDS during the phase before, the first ones during the step before.
    constexpr bool k8 = kIn == kE4M3;
    constexpr int kKs = k8 ? 1 : 2, kParts = k8 ? (MB < 4 ? MB : 4) : 2;
    constexpr int kPhases = kKs * kParts, MP = MB / kParts;
    static_assert(MB % kParts == 0 && kPhases % 2 == 0, "");
    using Operand = std::conditional_t<k8, v8i, v8s>;
    Operand p[2][MP], q[2][NB];

    auto read_p = [&](const char* s, int ph, Operand (&to)[MP]) {
        const int kk = ph / kParts, i0 = ph % kParts * MP;
#pragma unroll
        for (int i = 0; i < MP; ++i) {
            if constexpr (k8)
                to[i] = both(s, pat[0] + (i0 + i) * 2048);
            else if constexpr (kPT)
                to[i] = across(s + pat[i0 + i] + kk * 32 * BM * 2, BM);
            else
                to[i] = *reinterpret_cast<const v8s*>(s + (pat[0] ^ (kk * 64)) + (i0 + i) * 2048);
        }
    };
    auto read_q = [&](const char* s, int kk, Operand (&to)[NB]) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            if constexpr (k8)
                to[j] = both(s, qat[0] + qrow(j));
            else if constexpr (kQT)
                to[j] = across(s + qat[j] + kk * 32 * BN * 2, BN);
            else
                to[j] = *reinterpret_cast<const v8s*>(s + (qat[0] ^ (kk * 64)) + qrow(j));
        }
    };
    auto multiply = [&](int ph, const Operand (&pp)[MP], const Operand (&qq)[NB]) {
        const int i0 = ph % kParts * MP;
#pragma unroll
        for (int i = 0; i < MP; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                if constexpr (k8)
                    acc[i0 + i][j] = multiply8(qq[j], pp[i], acc[i0 + i][j]);
                else
                    acc[i0 + i][j] = multiply16<kIn>(qq[j], pp[i], acc[i0 + i][j]);
            }
    };
    // every copy of this wave landed and its reads done, then every wave's
    auto arrive = [&]() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(kDma ? 0x0070 : 0xc07f);  // vmcnt(0) lgkmcnt(0) or lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // Step s works on the stage at `cur`; the next step's operands are in the
    // other one, and the step after that is copied over `cur` once every wave
    // has read it.  The last step reads the other stage for nothing; no copy
    // is in flight when the loop ends.
    if (step0 < step1) {
        start(step0, lds);
        commit(lds);
        arrive();
        if (step0 + 1 < step1) start(step0 + 1, lds + kStage);
        read_p(lds, 0, p[0]);
        read_q(lds, 0, q[0]);
        int cur = 0;
        for (int s = step0; s < step1; ++s) {
#pragma unroll
            for (int ph = 0; ph < kPhases; ++ph) {
                const int qi = k8 ? 0 : ph / kParts;
                if (ph + 1 < kPhases) {
                    read_p(lds + cur, ph + 1, p[(ph + 1) & 1]);
                    if ((ph + 1) % kParts == 0)
                        read_q(lds + cur, (ph + 1) / kParts, q[qi ^ 1]);
                } else {
                    if (!kDma) commit(lds + (cur ^ kStage));
                    arrive();
                    if (s + 2 < step1) start(s + 2, lds + cur);
                    cur ^= kStage;
                    read_p(lds + cur, 0, p[0]);
                    read_q(lds + cur, 0, q[k8 ? 1 : 0]);
                }
                __builtin_amdgcn_sched_barrier(0);
                multiply(ph, p[ph & 1], q[qi]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (k8) {
#pragma unroll
                for (int j = 0; j < NB; ++j) q[0][j] = q[1][j];
            }
        }
    }

    // ---- epilogue
    const Epilogue& e = a.e;
    const bool part = gridDim.y > 1;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int m = m0 + wm * MT + 16 * i + i16;
        if constexpr (kQT) {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int n = n0 + wn * NT + 16 * j + 4 * g;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = acc[i][j][r];
                if (part) {
                    if (m < a.M && n < a.R)
                        store_row<4>(e.part, kF32, ((long long)blockIdx.y * a.M + m) * a.R + n,
                                     a.R - n, v);
                } else {
                    finish<4>(e, m, n, v);
                }
            }
        } else if constexpr (kGated) {
#pragma unroll
            for (int j = 0; j < NB / 2; j += kVec / 4) {
                const int n = n0 + wn * (NT / 2) + kRun * g + 4 * j;
                float gv[kVec], uv[kVec];
#pragma unroll
                for (int r = 0; r < kVec; ++r) {
                    gv[r] = acc[i][j + r / 4][r % 4];
                    uv[r] = acc[i][NB / 2 + j + r / 4][r % 4];
                }
                if (part) {
                    if (m < a.M && n < e.N) {
                        const long long at = ((long long)blockIdx.y * a.M + m) * a.R + n;
                        store_row<kVec>(e.part, kF32, at, e.N - n, gv);
                        store_row<kVec>(e.part, kF32, at + e.N, e.N - n, uv);
                    }
                } else {
                    finish_gated<kVec>(e, m, n, gv, uv);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < NB; j += 2) {
                const int n = n0 + wn * NT + kRun * g + 4 * j;
                float v[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) v[r] = acc[i][j + r / 4][r % 4];
                if (part) {
                    if (m < a.M && n < a.R)
                        store_row<8>(e.part, kF32, ((long long)blockIdx.y * a.M + m) * a.R + n,
                                     a.R - n, v);
                } else {
                    finish<8>(e, m, n, v);
                }
            }
        }
    }
}

}  // namespace bvml_ffn
