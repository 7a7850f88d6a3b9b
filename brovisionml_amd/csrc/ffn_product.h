// C[m][n] = sum_k P(m, k) Q(n, k) on the matrix cores, with the feed-forward
// operators' epilogues: the kernel behind the forward products and, with one
// or both operands read across their rows, behind both gradients.
//
//   forward       P = x,  k along its rows      Q = W,  k along its rows
//   input's       P = dz, k along its rows      Q = W,  k across its rows
//   weight's      P = dz, k across its rows     Q = x,  k across its rows
//
// A workgroup of 2 x 2 waves owns a BM x BN tile of C; a wave a quarter of it,
// in fp32 accumulators of 32 x 32.  k goes by in steps of 128 bytes (64 16-bit
// or 128 8-bit elements: whole cache lines of every row), each multiplied in two
// halves.  kSlots LDS slots hold a step of both operands each.  While a half is
// multiplied the next half's operands are read from LDS into the other set of
// registers, and in a step's second half, when every wave has read its slot,
// the step kSlots later is copied over it; reads and copies are dealt out
// between the products, so that the matrix cores never wait for a burst of
// them.  One barrier a step.
//
// What bounds it: at 256 x 256 the matrix cores and the clock they leave
// (4096 x 4096 x 8192 at 1350 TFLOP/s; one address for all rows, so that
// nothing comes from memory, makes 4096 x 4096 x 5120 25% faster); at 128 x 128 the
// way from cache to LDS, 64 bytes a clock and CU (1130); below that the latency of
// a step.  4805 x 5120 x 1280, 380 tiles of 128 x 128, takes 66 us with its
// operands in the caches and 80 without, 256 x 128 tiles with three slots
// 64 to 75 and 83, 256 x 256 96 and 137.  8-bit 4805 x 1280 x 5120: 48 us.
//
// LDS layout, operand with k along its rows: 128 bytes a row, its eight
// 16-byte pieces permuted by the row (piece ^ key) so that the rows a matrix
// operand reads at once fall into different banks.  Q is the instruction's
// first operand, its rows taken in an order that leaves a lane with 16
// neighbouring columns of one row of C, so that it stores 16 bytes at a time.
// Operand with k across its rows: one k a row, its 64-byte runs permuted by
// k; the transposing LDS read hands each lane four k of one column.
//
// Copies go straight from memory to LDS where every row begins on 16 bytes
// (DMA); otherwise through registers at any alignment.  Rows beyond the
// operand repeat its last one (their results are not stored); k beyond its
// end reads as zero: by the buffer descriptor's bound or by an offset past it.
//
// 8-bit products: the matrix instruction adds eight neighbouring products at
// a time aligned to the largest of them and cut off 13 bits below it (measured);
// the sums of eights are fp32.  Beside the operands' own 4-bit rounding that
// is nothing, and the exact alternative, 16-bit products, has half the rate.
#pragma once

#include <type_traits>

#include "ffn_sums.h"

namespace bvml_ffn {

struct Product {
    const char* p;          // first operand, rows are C's rows
    const char* q;          // second operand, rows are C's columns
    long long ldp, ldq;     // bytes from row to row in memory
    int M, K;               // C's rows; the sum's length
    int R;                  // Q's columns of C: N, or 2N for the gated form
    int tiles_m, tiles_n;
    int steps;              // ceil(K / kStep)
    // The first `whole` tiles have a workgroup each; each of the others has
    // `splits`, for per_split steps each, which leave fp32 parts of the tile.
    int whole, splits, per_split;
    Epilogue e;
};

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

#define BVML_LDS(T, p) ((__attribute__((address_space(3))) T*)(p))

constexpr int kBufferWord3 = 0x00020000;      // gfx9 raw-buffer descriptor word 3
constexpr uint32_t kBufferEnd = 0x7fffffffu;  // the longest range a descriptor gets here
constexpr int kPastEnd = (int)0x80000000u;    // an offset past any of them: reads zeros

struct Operand {  // of a half: 32 bytes of k a lane
    v4i lo, hi;
};

// 32 x 32 of C += Q's 32 rows by P's: in 16 bits the half's products are two
// of 16 k each (kk), in 8 bits one of 64 (without block scales).
template <int kIn>
__device__ __forceinline__ v16f multiply(int kk, const Operand& q, const Operand& p, v16f c) {
    const v4i qk = kk == 0 ? q.lo : q.hi, pk = kk == 0 ? p.lo : p.hi;
    if constexpr (kIn == kBF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, qk),
                                                       __builtin_bit_cast(v8b, pk), c, 0, 0, 0);
    } else if constexpr (kIn == kF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, qk),
                                                      __builtin_bit_cast(v8h, pk), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
            __builtin_shufflevector(q.lo, q.hi, 0, 1, 2, 3, 4, 5, 6, 7),
            __builtin_shufflevector(p.lo, p.hi, 0, 1, 2, 3, 4, 5, 6, 7), c, 0, 0, 0, 0, 0, 0);
    }
}

// The few-rows kernel's: 16 x 16 of C.
template <int kIn>
__device__ __forceinline__ v4f multiply16(v4i q, v4i p, v4f c) {
    if constexpr (kIn == kBF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, q),
                                                       __builtin_bit_cast(v8b, p), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, q),
                                                      __builtin_bit_cast(v8h, p), c, 0, 0, 0);
}
__device__ __forceinline__ v4f multiply8(v8i q, v8i p, v4f c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(q, p, c, 0, 0, 0, 0, 0, 0);
}

// Which 64-byte run of a k row another one takes the place of: different for
// the 4 rows (2 rows of 128 bytes side by side) a transposing read touches.
template <int kCols>
__device__ __forceinline__ int run_key(int k) {
    return kCols >= 128 ? k & 3 : (k >> 1) & 1;
}
// A row's permutation of its eight pieces: the instruction's row bits 3 2 1.
// kRemap: Q, where the instruction's row 8 b + 4 h + e is the block's row
// 16 h + 4 b + e.
template <bool kRemap>
__device__ __forceinline__ int piece_key(int row) {
    return kRemap ? ((row >> 1) & 1) | ((row >> 3) & 2) | (row & 4) : (row >> 1) & 7;
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

// One operand's copy of a step into an LDS slot: kRows x 128 bytes or,
// transposed, kStep k rows of kRows 16-bit columns; in parts of 1 KB a wave.
template <int kIn, int kRows, int kWaves, bool kT, bool kRemap, bool kDma>
struct Copy {
    static constexpr int kSize = kIn == kE4M3 ? 1 : 2;
    static constexpr int kPiece = 16 / kSize;  // elements of 16 bytes
    static constexpr int kStep = 128 / kSize;  // k of one step
    static constexpr int kParts = kRows / 8 / kWaves;
    static constexpr int kChunks = kRows / 8;  // pieces of a transposed row
    static_assert(kRows % (8 * kWaves) == 0 && kWaves % 4 == 0, "whole copies; one key a lane");

    int off[kParts];  // per-lane byte offset from the tile's base
    int piece;        // k along rows: the lane's first k in the step
    v4i held[kDma ? 1 : kParts];
    // the step that is being copied
    v4i rsrc;
    const char* base;
    int left;
    long long have;  // transposed: bytes to the end

    static __device__ __forceinline__ int across_k(int t, int w, int lane) {
        return ((t * kWaves + w) * 64 + lane) / kChunks;
    }
    static __device__ __forceinline__ int across_col(int t, int w, int lane) {
        const int pos = (t * kWaves + w) * 64 + lane;
        return ((pos % kChunks) ^ (run_key<kRows>(pos / kChunks) << 2)) * 8;
    }

    // parts t0 .. t1 of the slot; rows: how many the operand has from the
    // base on
    __device__ __forceinline__ void init(int w, int lane, long long ld, int rows, int t0, int t1) {
        const int r0 = w * 8 + (lane >> 3);
        const int c = (lane & 7) ^ piece_key<kRemap>(r0);
        piece = kT ? 0 : c * kPiece;
#pragma unroll
        for (int t = 0; t < kParts; ++t) {
            if (t < t0 || t >= t1) continue;
            if constexpr (!kT) {
                const int row = (t - t0) * kWaves * 8 + r0;
                off[t] = (int)((row < rows ? row : rows - 1) * ld) + c * 16;
            } else {
                // an offset past the end for columns beyond the operand
                const int col = across_col(t, w, lane);
                off[t] = col < rows ? (int)(across_k(t, w, lane) * ld) + col * 2 : kPastEnd;
            }
        }
    }

    // The first step: its first k is at `from`, `remain` k before the end.
    __device__ __forceinline__ void aim(const char* from, long long ld, int remain) {
        base = from;
        left = remain;
        have = kT ? remain * ld : 0;
        describe();
    }
    // The one after it (past the end: zeros, without touching memory).
    __device__ __forceinline__ void next(long long ld) {
        base += kT ? kStep * ld : 128;
        left -= kStep;
        if constexpr (kT) have -= kStep * ld;
        describe();
    }
    __device__ __forceinline__ void describe() {
        if constexpr (kDma) {
            uint32_t bytes = kBufferEnd;
            if constexpr (kT)
                bytes = have < 0 ? 0u : have < (long long)kBufferEnd ? (uint32_t)have : kBufferEnd;
            const uint64_t at = reinterpret_cast<uint64_t>(base);
            rsrc = (v4i){(int)(uint32_t)at, (int)(uint32_t)(at >> 32) & 0xffff, (int)bytes,
                         kBufferWord3};
        }
    }
    // One part of it on its way.
    __device__ __forceinline__ void start(int t, int rows, int w, int lane, char* to) {
        if constexpr (kDma) {
            copy_to_lds(rsrc, kT || piece < left ? off[t] : kPastEnd, to + (t * kWaves + w) * 1024);
        } else {
            int n;  // elements of the piece inside the operand
            if constexpr (kT)
                n = across_k(t, w, lane) < left ? rows - across_col(t, w, lane) : 0;
            else
                n = left - piece;
            v4i v = {0, 0, 0, 0};
            const char* from = base + off[t];
            if (n >= kPiece) {
                __builtin_memcpy(&v, from, 16);
            } else if (n > 0) {
                if constexpr (kSize == 2) {
                    uint16_t h[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        h[i] = i < n ? reinterpret_cast<const uint16_t*>(from)[i] : (uint16_t)0;
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
    // Without DMA: what start() read, into LDS.
    __device__ __forceinline__ void commit(int w, int lane, char* to) {
        if constexpr (!kDma) {
#pragma unroll
            for (int t = 0; t < kParts; ++t)
                *reinterpret_cast<v4i*>(to + (t * kWaves + w) * 1024 + lane * 16) = held[t];
        }
    }
};

// Tile t of a product: groups of kGroup row tiles by all column tiles, so that
// neighbours share operand rows.
constexpr int kGroup = 4;
__device__ __forceinline__ void tile_of(int t, int tm, int tn, int& m, int& n) {
    const int per = kGroup * tn, g = t / per, in = t % per;
    const int rows = tm - g * kGroup < kGroup ? tm - g * kGroup : kGroup;
    m = g * kGroup + in % rows;
    n = in / rows;
}
// Workgroup b of n as a place in the tiles' order: consecutive tiles on one
// XCD (workgroups go round the 8 of them), whose L2 then serves them all.
constexpr int kXcds = 8;
__device__ __forceinline__ int place_of(int b, int n) {
    const int each = n / kXcds, more = n % kXcds, x = b % kXcds;
    return x * each + (x < more ? x : more) + b / kXcds;
}

// One workgroup's tile: workgroup b of the product's, LDS of kLdsBytes.
template <int kIn, int BM, int BN, int kSlots, bool kPT, bool kQT, bool kGated, bool kDma>
__device__ __forceinline__ void product_tile(const Product& a, const int b, char* const lds) {
    constexpr int WM = 2, WN = 2;
    constexpr int kWaves = WM * WN;
    constexpr int MT = BM / WM, NT = BN / WN, MB = MT / 32, NB = NT / 32;
    constexpr int kSize = kIn == kE4M3 ? 1 : 2;
    constexpr int kStep = 128 / kSize;
    constexpr int kPBytes = BM * 128, kSlot = (BM + BN) * 128;
    static_assert(!kGated || NB % 2 == 0, "");
    static_assert(!(kGated && kQT) && !((kPT || kQT) && kIn == kE4M3), "");

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = w / WN, wn = w % WN;
    int tm, tn, step0 = 0, step1 = a.steps;
    const bool part = b >= a.whole;
    if (!part) {
        tile_of(place_of(b, a.whole), a.tiles_m, a.tiles_n, tm, tn);
    } else {
        tile_of(a.whole + (b - a.whole) / a.splits, a.tiles_m, a.tiles_n, tm, tn);
        step0 = (b - a.whole) % a.splits * a.per_split;
        step1 = step0 + a.per_split < a.steps ? step0 + a.per_split : a.steps;
    }
    const int m0 = tm * BM, n0 = tn * (kGated ? BN / 2 : BN);

    // ---- copies
    using CopyP = Copy<kIn, BM, kWaves, kPT, false, kDma>;
    using CopyQ = Copy<kIn, BN, kWaves, kQT, true, kDma>;
    CopyP cp;
    CopyQ cq, cu;  // cu: the gated form's other half
    constexpr int PP = CopyP::kParts, QP = CopyQ::kParts, QH = kGated ? QP / 2 : QP;
    static_assert(!kGated || QP % 2 == 0, "a copy belongs to the gate or to the other half");
    const int rows_p = a.M - m0;
    const int rows_q = (kGated ? a.R / 2 : a.R) - n0;
    cp.init(w, lane, a.ldp, rows_p, 0, PP);
    cq.init(w, lane, a.ldq, rows_q, 0, QH);
    if constexpr (kGated) cu.init(w, lane, a.ldq, rows_q, QH, QP);
    const char* pb = kPT ? a.p + (long long)m0 * 2 : a.p + (long long)m0 * a.ldp;
    const char* qb = kQT ? a.q + (long long)n0 * 2 : a.q + (long long)n0 * a.ldq;

    {
        const int k = step0 * kStep, end = step1 < a.steps ? step1 * kStep : a.K;
        const long long at = kQT ? k * a.ldq : (long long)k * kSize;
        cp.aim(pb + (kPT ? k * a.ldp : (long long)k * kSize), a.ldp, end - k);
        cq.aim(qb + at, a.ldq, end - k);
        if constexpr (kGated) cu.aim(qb + (long long)(a.R / 2) * a.ldq + at, a.ldq, end - k);
    }
    auto next_step = [&]() {
        cp.next(a.ldp);
        cq.next(a.ldq);
        if constexpr (kGated) cu.next(a.ldq);
    };
    auto start = [&](int t, char* slot) {  // part t of PP + QP
        if (t < PP)
            cp.start(t, rows_p, w, lane, slot);
        else if (t - PP < QH)
            cq.start(t - PP, rows_q, w, lane, slot + kPBytes);
        else
            cu.start(t - PP, rows_q, w, lane, slot + kPBytes);
    };
    auto start_all = [&](char* slot) {
#pragma unroll
        for (int t = 0; t < PP + QP; ++t) start(t, slot);
    };
    auto commit = [&](char* slot) {
        if constexpr (!kDma) {
            cp.commit(w, lane, slot);
            if constexpr (kGated) {
#pragma unroll
                for (int t = QH; t < QP; ++t) cq.held[t] = cu.held[t];
            }
            cq.commit(w, lane, slot + kPBytes);
        }
    };

    // ---- where the lane's operands are in a slot
    const int hl = lane >> 5;
    int pat[kPT ? MB : 1], qat[kQT ? NB : 1];
    {
        // transposing reads: 16 lanes take 4 k rows by 16 columns, a lane the
        // address of 4 columns of one of them
        const int i16 = lane & 15, t = (lane >> 4) & 1;
        const int k = 8 * hl + (i16 >> 2), piece = i16 & 3;
        if constexpr (kPT) {
            const int c = wm * MT / 8 + 2 * t + (piece >> 1);
#pragma unroll
            for (int i = 0; i < MB; ++i)
                pat[i] = k * BM * 2 + (((c + 4 * i) ^ (run_key<BM>(k) << 2)) << 4) + (piece & 1) * 8;
        } else {
            const int row = wm * MT + (lane & 31);
            pat[0] = row * 128 + ((hl ^ piece_key<false>(row)) << 4);
        }
        if constexpr (kQT) {
            const int c = wn * NT / 8 + 2 * (piece & 1) + t;
#pragma unroll
            for (int j = 0; j < NB; ++j)
                qat[j] = kPBytes + k * BN * 2 + (((c + 4 * j) ^ (run_key<BN>(k) << 2)) << 4) +
                         (piece >> 1) * 8;
        } else {
            const int i = lane & 31;
            const int r = 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3);
            const int row = (kGated ? wn * (NT / 2) : wn * NT) + r;
            qat[0] = kPBytes + row * 128 + ((hl ^ piece_key<true>(row)) << 4);
        }
    }
    // the j-th 32 rows of Q, k-along-rows layout, relative to qat
    auto qrow = [](int j) {
        return (kGated && j >= NB / 2 ? BN / 2 + 32 * (j - NB / 2) : 32 * j) * 128;
    };
    auto along = [](const char* s, int at) -> Operand {  // pieces h and h + 2 of a half row
        return {*reinterpret_cast<const v4i*>(s + at), *reinterpret_cast<const v4i*>(s + (at ^ 32))};
    };
    auto four = [](const char* at) {  // 4 k of a column
        return __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16(BVML_LDS(v4s, at)));
    };
    auto across = [&](const char* at, int cols) -> Operand {  // the same k of a column
        return {__builtin_shufflevector(four(at), four(at + 8 * cols), 0, 1, 2, 3),
                __builtin_shufflevector(four(at + 32 * cols), four(at + 40 * cols), 0, 1, 2, 3)};
    };

    v16f acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    Operand p[2][MB], q[2][NB];  // by half

    // operand r of a half: p[0], q[0], q[1], ..., then the other rows of p
    auto read = [&](const char* s, int kk, int r, Operand (&pp)[MB], Operand (&qq)[NB]) {
        if (r == 0 || r > NB) {
            const int i = r == 0 ? 0 : r - NB;
            if constexpr (kPT)
                pp[i] = across(s + pat[i] + kk * 64 * BM, BM);
            else
                pp[i] = along(s + i * 4096, pat[0] ^ (kk * 64));
        } else {
            const int j = r - 1;
            if constexpr (kQT)
                qq[j] = across(s + qat[j] + kk * 64 * BN, BN);
            else
                qq[j] = along(s + qrow(j), qat[0] ^ (kk * 64));
        }
    };
    // The next step's copies of this wave landed (those of the steps after it
    // may be on their way) and its reads are done; then every wave's.
    constexpr int kCopies = PP + QP, kFlying = (kSlots - 2) * kCopies;
    static_assert(kFlying < 64, "what vmcnt can count");
    auto arrive = [&]() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(kDma ? 0x0070 | (kFlying & 15) | (kFlying >> 4 << 14) : 0xc07f);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // The products of a half in kGroups groups; between them the next half's
    // reads, in the groups' first half, and copies.
    constexpr int kKs = kIn == kE4M3 ? 1 : 2, kGroups = MB * NB;
    constexpr int kReads = MB + NB;
    static_assert(kDma || kSlots == 2, "one step in registers");

    if (step0 < step1) {
        // (past the last step a copy is zeros: every step counts the same)
        start_all(lds);
        commit(lds);
#pragma unroll
        for (int i = 1; i < kSlots - 1; ++i) {
            next_step();
            start_all(lds + i * kSlot);
        }
        arrive();
        next_step();
        start_all(lds + (kSlots - 1) * kSlot);
#pragma unroll
        for (int r = 0; r < kReads; ++r) read(lds, 0, r, p[0], q[0]);
        int cur = 0;
        for (int s = step0; s < step1; ++s) {
            const int next = cur == (kSlots - 1) * kSlot ? 0 : cur + kSlot;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                if (kk == 0) {
                    next_step();  // which the second half starts to copy
                } else {
                    commit(lds + next);
                    arrive();
                }
                const char* const from = lds + (kk == 0 ? cur : next);
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
#pragma unroll
                    for (int r = 0; r < kReads; ++r)
                        if (r * kGroups / (2 * kReads) == g)
                            read(from, kk ^ 1, r, p[kk ^ 1], q[kk ^ 1]);
                    if (kk == 1) {
#pragma unroll
                        for (int t = 0; t < kCopies; ++t)
                            if (t * kGroups / kCopies == g) start(t, lds + cur);
                    }
#pragma unroll
                    for (int x = g * kKs; x < (g + 1) * kKs; ++x) {
                        const int u = x / (MB * NB), i = x / NB % MB, j = x % NB;
                        acc[i][j] = multiply<kIn>(u, q[kk][j], p[kk][i], acc[i][j]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            cur = next;
        }
        // no copy may be in flight when the workgroup's LDS is given away
        if constexpr (kDma) __builtin_amdgcn_s_waitcnt(0x0f70);
    }

    // ---- epilogue, 32 rows of the wave's part at a time: the sums go through
    // LDS, so that a row of C is finished by neighbouring lanes, 8 columns
    // each, in a rolled loop.  (Straight from the registers it is thousands
    // of instructions that run once, and fetching them costs more than the
    // products: a 256 x 256 tile took 100 us.)
    __builtin_amdgcn_s_barrier();  // every wave has read its last operands
    asm volatile("" ::: "memory");
    constexpr int kPitch = NT + 4;  // floats; rows 16 bytes apart in the banks
    static_assert(32 * kPitch * 4 * kWaves <= kSlots * kSlot, "");
    float* const sums = reinterpret_cast<float*>(lds) + w * 32 * kPitch;
    const Epilogue& e = a.e;
    constexpr bool kPlain = kPT || kQT;  // a gradient: nothing but the store
    constexpr int kCols = kGated ? NT / 2 : NT, kLanes = kCols / 8;  // lanes of a row
    // the lane takes every kGap-th row, kTimes rows at once
    constexpr int kGap = 64 / kLanes, kTimes = 32 / kGap < 4 ? 32 / kGap : 4;
    const int type16 = kIn == kE4M3 ? e.out_type : kIn;
    const int y_type = e.out_type == kF32 ? kF32 : type16;
    const int row0 = lane / kLanes, col = lane % kLanes * 8, n = n0 + wn * kCols + col;
    const int c = e.N - n;
    // no ragged column and no row beyond the last in the tile
    const bool whole = n0 + (kGated ? BN / 2 : BN) <= e.N && m0 + BM <= a.M;
    Column<8> kv, ku;
    if (!kPlain && !part) {
        kv.load(e, n, c);
        if constexpr (kGated) ku.load(e, e.N + n, c);
    }
#pragma unroll 1
    for (int i = 0; i < MB; ++i) {
#pragma unroll
        for (int x = 0; x < MB; ++x) {
            if (x != i) continue;
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int y = 0; y < 16; y += 4)
                    *reinterpret_cast<v4f*>(sums + (lane & 31) * kPitch + 32 * j + 16 * hl + y) =
                        (v4f){acc[x][j][y], acc[x][j][y + 1], acc[x][j][y + 2], acc[x][j][y + 3]};
        }
        asm volatile("" ::: "memory");
#pragma unroll 1
        for (int from = row0; from < 32; from += kTimes * kGap) {
            const int first = m0 + wm * MT + 32 * i + from;
            // each step for all of the lane's rows before the next: one branch a step
            auto store = [&](void* to, int type, long long ld, int at, const float (&x)[kTimes][8]) {
                const int size = type == kF32 ? 4 : 2;
                char* p = static_cast<char*>(to) + ((long long)first * ld + at) * size;
                const long long step = kGap * ld * size;
                if (whole) {
#pragma unroll
                    for (int t = 0; t < kTimes; ++t, p += step) store_row<8>(p, type, 0, 8, x[t]);
                } else {
#pragma unroll
                    for (int t = 0; t < kTimes; ++t, p += step)
                        if (first + t * kGap < a.M && c > 0) store_row<8>(p, type, 0, c, x[t]);
                }
            };
            float r[kPlain || kGated ? 1 : kTimes][8];
            if constexpr (!kPlain && !kGated) {
                if (e.residual && !part) {
#pragma unroll
                    for (int t = 0; t < kTimes; ++t) {
                        const int m = first + t * kGap;
                        const long long at = (long long)(m < a.M ? m : a.M - 1) * e.ldr + n;
                        if (whole)
                            load_row<8>(e.residual, y_type, at, 8, r[t]);
                        else
                            load_row<8>(e.residual, y_type, at, c, r[t]);
                    }
                }
            }
            float v[kTimes][8], u[kGated ? kTimes : 1][8];
#pragma unroll
            for (int t = 0; t < kTimes; ++t) {
                const float* const at = sums + (from + t * kGap) * kPitch + col;
                __builtin_memcpy(v[t], __builtin_assume_aligned(at, 16), 32);
                if constexpr (kGated)
                    __builtin_memcpy(u[t], __builtin_assume_aligned(at + kCols, 16), 32);
            }
            if (part) {
                // the workgroup's own BM x BN floats, whole also at the edges
                float* to = e.part + (long long)(b - a.whole) * BM * BN +
                            (wm * MT + 32 * i + from) * BN + wn * kCols + col;
#pragma unroll
                for (int t = 0; t < kTimes; ++t, to += kGap * BN) {
                    store_row<8>(to, kF32, 0, 8, v[t]);
                    if constexpr (kGated) store_row<8>(to, kF32, BN / 2, 8, u[t]);
                }
                continue;
            }
            if constexpr (!kPlain) {
#pragma unroll
                for (int t = 0; t < kTimes; ++t) {
                    const int m = first + t * kGap;
                    constexpr bool kScaled = kIn == kE4M3;
                    const float s = kScaled ? e.x_scale[m < a.M ? m : a.M - 1] : 1.0f;
                    kv.template apply<kScaled>(s, v[t]);
                    if constexpr (kGated) ku.template apply<kScaled>(s, u[t]);
                }
                if (e.z) {
                    store(e.z, type16, e.ldz, n, v);
                    if constexpr (kGated) store(e.z, type16, e.ldz, e.N + n, u);
                }
                activate<8 * kTimes>(e.act, reinterpret_cast<float(&)[8 * kTimes]>(v));
                if constexpr (kGated) {
#pragma unroll
                    for (int t = 0; t < kTimes; ++t)
#pragma unroll
                        for (int x = 0; x < 8; ++x) v[t][x] *= u[t][x];
                } else if (e.residual) {
#pragma unroll
                    for (int t = 0; t < kTimes; ++t)
#pragma unroll
                        for (int x = 0; x < 8; ++x) v[t][x] += r[t][x];
                }
            }
            if (y_type == kF32)
                store(e.y, kF32, e.ldy, n, v);
            else
                store(e.y, type16, e.ldy, n, v);
        }
        asm volatile("" ::: "memory");
    }
}

template <int BM, int BN, int kSlots>
constexpr int kLdsBytes = kSlots * (BM + BN) * 128;
// (the 256 x 256 tile's sums take 256 registers a lane)
template <int BM>
constexpr int kWavesPerSimd = BM == 256 ? 1 : 2;

template <int kIn, int BM, int BN, int kSlots, bool kPT, bool kQT, bool kGated, bool kDma>
__global__ __launch_bounds__(256, kWavesPerSimd<BM>) void product_kernel(Product a) {
    __shared__ __align__(1024) char lds[kLdsBytes<BM, BN, kSlots>];
    product_tile<kIn, BM, BN, kSlots, kPT, kQT, kGated, kDma>(a, blockIdx.x, lds);
}

// Both gradients of a product in one launch, so that one's tiles fill the CUs
// that the other's leave idle.  The product whose workgroups take longer goes
// first, for a long one started last would keep the launch waiting; before it
// the parts of the other's last tiles, where only those are split.
// Last come the workgroups that sum the bias's gradient.  4805 x 1280 x 5120 with
// its sums: 122 us, 1030 TFLOP/s; 16389 x 1024 x 8192: 440 to 460, 1200 to 1250.
struct Gradients {
    Product input, weight;
    bool weight_first;
    ColumnSum sums;
};

// Workgroups of a launch.
inline long long groups_of(const Product& a) {
    return a.whole + ((long long)a.tiles_m * a.tiles_n - a.whole) * a.splits;
}
inline long long groups_of(const Gradients& g) {
    return groups_of(g.input) + groups_of(g.weight) + (g.sums.out ? (g.sums.cols + 31) / 32 : 0);
}

__device__ __forceinline__ int rest_of(const Product& a) {
    return (a.tiles_m * a.tiles_n - a.whole) * a.splits;
}

template <int kIn, int BM, int BN, int kSlots>
__global__ __launch_bounds__(256, kWavesPerSimd<BM>) void gradients_kernel(Gradients g) {
    __shared__ __align__(1024) char lds[kLdsBytes<BM, BN, kSlots>];
    const Product& first = g.weight_first ? g.weight : g.input;
    const Product& second = g.weight_first ? g.input : g.weight;
    const int parts = second.whole > 0 ? rest_of(second) : 0;
    const int longer = first.whole + rest_of(first);
    const int tiles = longer + second.whole + rest_of(second);
    int b = blockIdx.x;
    if (b >= tiles) {
        column_sum<8>(g.sums, b - tiles, reinterpret_cast<float(*)[32]>(lds));
        return;
    }
    bool weight = !g.weight_first;
    if (b < parts) {
        b += second.whole;
    } else if (b < parts + longer) {
        b -= parts;
        weight = g.weight_first;
    } else {
        b -= parts + longer;
    }
    if (weight)
        product_tile<kIn, BM, BN, kSlots, true, true, false, true>(g.weight, b, lds);
    else
        product_tile<kIn, BM, BN, kSlots, false, true, false, true>(g.input, b, lds);
}

}  // namespace bvml_ffn
