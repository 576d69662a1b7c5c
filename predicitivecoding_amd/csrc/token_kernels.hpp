// token_kernels.hpp -- gfx950 kernels of the token operators: the two ends of a
// model over a vocabulary of V tokens.
//
//   embedding      out_i = s E[t_i];  dE[v] = s sum_{i: t_i = v} dout_i
//   token losses   z = s H W^T, l_i = log sum_v exp z_iv, for hidden states H
//                  [N x D] and an output matrix W [V x D]:
//     cross entropy  loss_i = w_i (l_i - z_{i, y_i})
//     distillation   loss_i = w_i T^2 sum_j p_ij (log p_ij - log q_{i, id_ij}),
//                    q = softmax(z / T), p the teacher's over its own slots
//   and of sum_i loss_i:  G = w (q - p) (times s, or s T), dH = G W, dW = G^T H.
//
// The logits are in memory only as far as a call may keep them (TokArgs::z).  They are 2 N V D operations, as dH and
// dW each are, against (N + V) D values in and out: products, run on the phase
// kernels' tiles (pc_kernels.hpp) with epilogues of their own.
//   LSE    every tile's part of each row's maximum and sum of exponentials (and
//          the targets' logits), 8 bytes a row and tile; row_loss_kernel joins
//          them.
//   GRAD   for a piece of the vocabulary, the logits again and G by the rows'
//          sums, in the operand type: what the next two products read.
//   DH     G's piece times W's, added up over the pieces in fp32.  Its sweeps are
//          long and its tiles few, so K goes in ranges, each with a sum of its
//          own that scatter_rows_kernel joins.
//   DW     G's piece transposed times H: the piece's rows of dW, final.
// DH and DW read the same piece and go out in one launch: DH's few long sweeps
// first, DW's many short ones into the CUs that those leave.
// Every product's operands are read where they lie: G and H as they are for DH
// and DW, in K rows.
//
// Rows that are left out (no label, no weight, no teacher's slot) are packed
// away first: gather_rows_kernel copies the live rows together, in order, and
// counts them on the device; the products run over that many rows, so a row
// left out costs nothing and whatever its hidden state holds (an infinity, a
// NaN) reaches no sum.
#pragma once
#include "pc_kernels.hpp"

namespace pcd {

// 16 and 8 bytes at any address of whole elements: one access each (gfx950 takes
// global accesses of any alignment), slower across a line's end, and a third of
// the time of element by element.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef const __attribute__((address_space(1))) u32x4_any gu32x4c_any;
typedef const __attribute__((address_space(1))) u32x2_any gu32x2c_any;
typedef __attribute__((address_space(1))) u32x4_any gu32x4_any;
typedef __attribute__((address_space(1))) u32x2_any gu32x2_any;

// Device-side facts of a call: how many rows are live, the same in whole K
// stages, and what the gradients by the logits are multiplied by (the largest
// weight's inverse, in f16 times a power of two) with its inverse.
struct TokCtl {
    int live, padded;
    float gscale, inv_gscale;
    int dh_rows;     // rows of DH: the live ones, or all of a stacked call's (see grad_rows_kernel)
    int dh_ranges;   // ranges of its K (see dh_ranges)
};

// Vocabulary ids a bucket of the teacher's slots covers: the columns of one wave
// on the tiles of 128 and more columns.
constexpr int kTokBucket = 64;

// Kept logits of bf16 calls are codes of 16 bits: how far a logit lies below the
// largest of its row's 32 columns, in steps of 1 / kTokCode of base 2, up to 64
// (a probability below 2^-64 of a neighbour's is held as 0).
// Half a step is 3.4e-4 of a probability (2e-4 in the root mean square) beside
// the 2^-8 (1.7e-3) that rounding G to bf16 costs it; half the traffic of fp32
// and twice the columns in the same room.  Targets' columns, where q - p may cancel,
// take their logits from `taken`, whole.  f16 gradients would show it (their
// rounding costs 2e-4), fp32 ones all the more, so those keep fp32 logits.
constexpr float kTokCode = 1024.f;

struct TokArgs {
    const TokCtl* ctl;
    const int* map;              // the caller's row of each live row
    // targets, by the caller's rows
    const int* labels;           // cross entropy: the label (null: distillation)
    const uint16_t* starts;      // distillation: [row x (buckets + 1)] first slot of each bucket of ids
    const int* ids;              // [row x top] ids, increasing
    const float* probs;          // [row x top]
    int top, buckets;
    float scale2;                // s log2(e) (over T): a logit's factor in base 2
    const float* row_weight;     // by the caller's rows (nullable: 1)
    float2* part;                // LSE: [live row x slots] (maximum, sum), base 2
    int slots;
    float* z;                    // LSE: the logits themselves, base 2, of the first z_cols ids (null: none)
    uint16_t* zq;                // ... or as codes (see kTokCode)
    float* ztop;                 // [live row x z_cols / 32] the largest of each 32
    int z_cols;                  // whole tiles, but for the vocabulary's end
    float* taken;                // LSE: [row x top] the targets' logits, base 2
    float* lse2;                 // [live row] log2 of the row's sum
    float* loss;                 // by the caller's rows
    const float* plogp;          // distillation: sum p ln p of each of the caller's rows
    float factor;                // of every loss: T^2
    int id0;                     // vocabulary id of this product's first column (LSE, GRAD)
    int out_m, out_n;            // DW: rows and columns that are stored; GRAD: columns of the piece in memory
    // DH: from K stage tail_stage on, W's rows come from its last rows' copy, tail_delta bytes on
    int tail_stage;
    long long tail_delta;
    // LSE, GRAD: column tile last_tn reads W's last rows from their copy (null: in place)
    const void* b_last;
    int last_tn;
    int unit0;                   // LSE, GRAD: the launch's first work unit (see kGridUnits)
};

// Workgroups of one launch at most: HIP takes fewer than 2^32 threads in a grid,
// and a workgroup has up to 512.  Whole rounds over the XCDs.
constexpr int kGridUnits = 1 << 22;

__device__ __forceinline__ int tok_rows(const TokArgs* t, int epi) {
    return __builtin_amdgcn_readfirstlane(
        gld(epi == EPI_TOK_GRAD ? &t->ctl->padded : epi == EPI_TOK_DH ? &t->ctl->dh_rows : &t->ctl->live));
}
__device__ __forceinline__ int tok_depth(const TokArgs* t) {
    return __builtin_amdgcn_readfirstlane(gld(&t->ctl->padded));
}
__device__ __forceinline__ int tok_ranges(const TokArgs* t) {
    return __builtin_amdgcn_readfirstlane(gld(&t->ctl->dh_ranges));
}
__device__ __forceinline__ void tok_last_columns(const TokArgs* t, Problem& P, int tn) {
    if (t->b_last != nullptr && tn == t->last_tn) P.B = t->b_last;
}
__device__ __forceinline__ size_t tok_advance(const TokArgs* t, int kk, size_t step) {
    return (size_t)kk * step + (kk >= t->tail_stage ? (size_t)t->tail_delta : 0);
}

// Row-contiguous stores of NBJ 32 x 32 result blocks side by side, staged in the
// wave's region (see flush_block): whole 128-byte row segments for two 16-bit
// blocks.  Rows at or past m and columns at or past n are not written.
template <int OPB, int NBJ>
__device__ __forceinline__ void tok_flush(const char* st, void* out, size_t ld, int row0, int col0, int m, int n) {
    constexpr int LPR = NBJ * 32 * OPB / 16, UE = 16 / OPB;   // lanes a row, elements a lane
    const int lane = threadIdx.x & 63;
    static_for<0, 32 * LPR / 64>([&](auto Pc) PCD_INLINE {
        const int rr = lane / LPR + (64 / LPR) * decltype(Pc)::value, cc = (lane % LPR) * UE;
        const u32x4 w = *(const u32x4*)(st + rr * kStageRowBytes + (lane % LPR) * 16);
        char* dst = (char*)out + ((size_t)(row0 + rr) * ld + col0 + cc) * OPB;
        if (row0 + rr < m) {
            if (col0 + cc + UE <= n) {
                *(gu32x4_any*)dst = w;   // (non-temporal: the same time, for DW of 1 GB and logits of 1 GB)
            } else {
                static_for<0, UE>([&](auto K) PCD_INLINE {
                    constexpr int k = decltype(K)::value;
                    if (col0 + cc + k < n) {
                        if constexpr (OPB == 4) gst((float*)dst + k, __uint_as_float(w[k]));
                        else gst((uint16_t*)dst + k, (uint16_t)(w[k / 2] >> (16 * (k % 2))));
                    }
                });
            }
        }
    });
}
template <typename OP>
__device__ __forceinline__ void tok_stage(char* st, int jj, int g, f32x4 v) {
    const int lane = threadIdx.x & 63, lr = lane & 31, half = lane >> 5;
    char* at = st + lr * kStageRowBytes + (32 * jj + 8 * g + 4 * half) * OpTraits<OP>::bytes;
    if constexpr (OpTraits<OP>::bytes == 4) *(f32x4*)at = v;
    else *(u32x2*)at = OpTraits<OP>::pack4(v);
}

// The epilogues, on blocks held transposed (lane: row lr of block row i, register
// 4g + k of block (i, j): column 32 j + 8 g + 4 half + k of the wave's).
//
// A row's targets are few and rarely among a tile's columns.  The lane that holds
// one finds its register by comparing the index with every register's (no
// register is indexed by a variable), in a branch that a wave takes only if one
// of its lanes has a target.
template <typename OP, int BM, int BN, int EPI, typename C>
__device__ __forceinline__ void tok_epilogue(const Problem& P, const PhaseArgs& args, const TokArgs* t,
                                             f32x16 (&acc)[C::FM][C::FN], char* smem, int row0, int col0, int tm, int tn,
                                             int wm, int wn, int live) {
    constexpr int OPB = OpTraits<OP>::bytes, NBJ = OPB == 2 && C::FN >= 2 ? 2 : 1;
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    char* stage = smem + wave * kStageWaveBytes;
    __syncthreads();   // every wave is done reading the stage ring
    if constexpr (EPI == EPI_TOK_DW) {
        const float alpha = args.alpha * gld(&t->ctl->inv_gscale);
        static_for<0, C::FM>([&](auto I) PCD_INLINE {
            static_for<0, C::FN>([&](auto J) PCD_INLINE {
                constexpr int i = decltype(I)::value, j = decltype(J)::value;
                static_for<0, 4>([&](auto G) PCD_INLINE {
                    constexpr int g = decltype(G)::value;
                    f32x4 v;
                    static_for<0, 4>([&](auto K) PCD_INLINE { v[decltype(K)::value] = alpha * acc[i][j][4 * g + decltype(K)::value]; });
                    tok_stage<OP>(stage, j % NBJ, g, v);
                });
                if constexpr (j % NBJ == NBJ - 1)
                    tok_flush<OPB, NBJ>(stage, P.m, P.ldo, row0 + wm * C::WTM + i * 32,
                                        col0 + wn * C::WTN + (j - j % NBJ) * 32, t->out_m, t->out_n);
                __builtin_amdgcn_sched_barrier(0);
            });
        });
    } else {
        const int count = EPI == EPI_TOK_LSE ? live : __builtin_amdgcn_readfirstlane(gld(&t->ctl->live));
        const int lo = t->id0 + col0 + wn * C::WTN;   // vocabulary id of the wave's first column
        const int ncols = P.N - (col0 + wn * C::WTN);   // its columns in the vocabulary
        const bool xent = t->labels != nullptr;
        // What each row needs, asked for all at once.
        int orig[C::FM], first[C::FM], end[C::FM], id[C::FM];
        float prob[C::FM], fac[C::FM], lse2[C::FM];
        static_for<0, C::FM>([&](auto I) PCD_INLINE {
            constexpr int i = decltype(I)::value;
            const int row = row0 + wm * C::WTM + i * 32 + lr;
            orig[i] = row < count ? gld(t->map + row) : -1;
            if constexpr (EPI == EPI_TOK_GRAD) lse2[i] = row < count ? gld(t->lse2 + row) : 0.f;
        });
        const float gscale = EPI == EPI_TOK_GRAD ? gld(&t->ctl->gscale) : 1.f;
        static_for<0, C::FM>([&](auto I) PCD_INLINE {
            constexpr int i = decltype(I)::value;
            first[i] = end[i] = 0;
            fac[i] = 0.f;
            if (orig[i] >= 0) {
                if constexpr (EPI == EPI_TOK_GRAD)
                    fac[i] = t->row_weight != nullptr ? gscale * gld(t->row_weight + orig[i]) : gscale;
                if (xent) {
                    id[i] = gld(t->labels + orig[i]);
                    end[i] = id[i] >= lo && id[i] - lo < C::WTN;
                } else {
                    const gu16* at = (const gu16*)(t->starts + (size_t)orig[i] * (t->buckets + 1) + lo / kTokBucket);
                    if (ncols > 0) first[i] = at[0], end[i] = at[1];
                }
            }
        });
        if (!xent) {
            static_for<0, C::FM>([&](auto I) PCD_INLINE {
                constexpr int i = decltype(I)::value;
                if (first[i] < end[i]) {
                    id[i] = gld(t->ids + (size_t)orig[i] * t->top + first[i]);
                    if constexpr (EPI == EPI_TOK_GRAD) prob[i] = gld(t->probs + (size_t)orig[i] * t->top + first[i]);
                }
            });
        }
        // f(register index or -1, slot, probability) for the targets of block row
        // i among this lane's columns, and once for the whole wave per round.
        auto targets = [&](auto I, auto&& f) PCD_INLINE {
            constexpr int i = decltype(I)::value;
            for (int s = first[i]; __any(s < end[i]); ++s) {
                int v = id[i];
                float p = xent ? 1.f : prob[i];
                const bool has = s < end[i];
                if (s > first[i] && has) {
                    v = gld(t->ids + (size_t)orig[i] * t->top + s);
                    if constexpr (EPI == EPI_TOK_GRAD) p = gld(t->probs + (size_t)orig[i] * t->top + s);
                }
                const int c = v - lo;
                const bool mine = has && c >= 0 && c < C::WTN && ((c >> 2) & 1) == half;
                f(mine ? (c >> 5) * 16 + ((c >> 3) & 3) * 4 + (c & 3) : -1, s, p);
            }
        };
        const float scale2 = t->scale2;
        if constexpr (EPI == EPI_TOK_LSE) {
            float2* red = (float2*)(smem + C::NWAVES * kStageWaveBytes);   // [wave column][tile row]
            const bool keep = t->z != nullptr && col0 < t->z_cols;
            const bool code = std::is_same<OP, bf16_t>::value && t->zq != nullptr && col0 < t->z_cols;
            static_for<0, C::FM>([&](auto I) PCD_INLINE {
                constexpr int i = decltype(I)::value;
                float m = -__builtin_inff();
                static_for<0, C::FN>([&](auto J) PCD_INLINE {
                    static_for<0, 16>([&](auto R) PCD_INLINE {
                        constexpr int j = decltype(J)::value, r = decltype(R)::value;
                        acc[i][j][r] *= scale2;
                        if (ncols < C::WTN && j * 32 + 8 * (r >> 2) + 4 * half + (r & 3) >= ncols) acc[i][j][r] = -__builtin_inff();
                        m = fmaxf(m, acc[i][j][r]);
                    });
                });
                targets(I, [&](int at, int slot, float) PCD_INLINE {
                    float z = 0.f;
                    static_for<0, C::FN * 16>([&](auto X) PCD_INLINE {
                        constexpr int x = decltype(X)::value;
                        z = at == x ? acc[i][x / 16][x % 16] : z;
                    });
                    if (at >= 0) gst(t->taken + (size_t)orig[i] * t->top + slot, z);
                });
                if (keep) {
                    static_for<0, C::FN>([&](auto J) PCD_INLINE {
                        constexpr int j = decltype(J)::value;
                        static_for<0, 4>([&](auto G) PCD_INLINE {
                            constexpr int g = decltype(G)::value;
                            f32x4 v;
                            static_for<0, 4>([&](auto K) PCD_INLINE { v[decltype(K)::value] = acc[i][j][4 * g + decltype(K)::value]; });
                            tok_stage<float>(stage, 0, g, v);
                        });
                        tok_flush<4, 1>(stage, t->z, t->z_cols, row0 + wm * C::WTM + i * 32, col0 + wn * C::WTN + j * 32, live,
                                        t->z_cols);
                    });
                }
                if constexpr (std::is_same<OP, bf16_t>::value) {
                    if (code) {
                        const int row = row0 + wm * C::WTM + i * 32 + lr, at = (col0 + wn * C::WTN) / 32;
                        static_for<0, C::FN>([&](auto J) PCD_INLINE {
                            constexpr int j = decltype(J)::value;
                            float top = acc[i][j][0];
                            static_for<1, 16>([&](auto R) PCD_INLINE { top = fmaxf(top, acc[i][j][decltype(R)::value]); });
                            top = fmaxf(top, __shfl_xor(top, 32));
                            if (half == 0 && row < live && at + j < t->z_cols / 32) gst(t->ztop + (size_t)row * (t->z_cols / 32) + at + j, top);
                            const float from = __builtin_fmaf(top == -__builtin_inff() ? 0.f : top, kTokCode, 0.5f);
                            static_for<0, 4>([&](auto G) PCD_INLINE {
                                constexpr int g = decltype(G)::value;
                                uint32_t c[4];
                                static_for<0, 4>([&](auto K) PCD_INLINE {
                                    constexpr int k = decltype(K)::value;
                                    c[k] = (uint32_t)fminf(__builtin_fmaf(acc[i][j][4 * g + k], -kTokCode, from), 65535.f);
                                });
                                *(u32x2*)(stage + lr * kStageRowBytes + (32 * (j % NBJ) + 8 * g + 4 * half) * 2) =
                                    u32x2{c[0] | c[1] << 16, c[2] | c[3] << 16};
                            });
                            if constexpr (j % NBJ == NBJ - 1)
                                tok_flush<2, NBJ>(stage, t->zq, t->z_cols, row0 + wm * C::WTM + i * 32,
                                                  col0 + wn * C::WTN + (j - j % NBJ) * 32, live, t->z_cols);
                        });
                    }
                }
                m = fmaxf(m, __shfl_xor(m, 32));
                const float base = m == -__builtin_inff() ? 0.f : m;   // a row of nothing but -inf here: its sum is 0
                float s = 0.f;
                static_for<0, C::FN>([&](auto J) PCD_INLINE {
                    static_for<0, 16>([&](auto R) PCD_INLINE {
                        s += __builtin_amdgcn_exp2f(acc[i][decltype(J)::value][decltype(R)::value] - base);
                    });
                });
                s += __shfl_xor(s, 32);
                if (half == 0) red[wn * BM + wm * C::WTM + i * 32 + lr] = float2{m, s};
            });
            __syncthreads();
            for (int r = tid; r < BM; r += C::NT) {
                if (row0 + r >= count) continue;
                float m = red[r].x, s = red[r].y;
                static_for<1, C::WN>([&](auto W) PCD_INLINE {
                    const float2 o = red[decltype(W)::value * BM + r];
                    const float top = fmaxf(m, o.x), base = top == -__builtin_inff() ? 0.f : top;
                    s = s * __builtin_amdgcn_exp2f(m - base) + o.y * __builtin_amdgcn_exp2f(o.x - base);
                    m = top;
                });
                t->part[(size_t)(row0 + r) * t->slots + tn] = float2{m, s};
            }
        } else {   // EPI_TOK_GRAD
            static_for<0, C::FM>([&](auto I) PCD_INLINE {
                constexpr int i = decltype(I)::value;
                const bool rok = orig[i] >= 0;
                static_for<0, C::FN>([&](auto J) PCD_INLINE {
                    static_for<0, 16>([&](auto R) PCD_INLINE {
                        constexpr int j = decltype(J)::value, r = decltype(R)::value;
                        float q = fac[i] * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], scale2, -lse2[i]));
                        if (ncols < C::WTN && j * 32 + 8 * (r >> 2) + 4 * half + (r & 3) >= ncols) q = 0.f;
                        acc[i][j][r] = rok ? q : 0.f;   // rows past the live ones hold nothing
                    });
                });
                targets(I, [&](int at, int, float p) PCD_INLINE {
                    const float d = fac[i] * p;
                    static_for<0, C::FN * 16>([&](auto X) PCD_INLINE {
                        constexpr int x = decltype(X)::value;
                        acc[i][x / 16][x % 16] -= at == x ? d : 0.f;
                    });
                });
                static_for<0, C::FN>([&](auto J) PCD_INLINE {
                    constexpr int j = decltype(J)::value;
                    static_for<0, 4>([&](auto G) PCD_INLINE {
                        constexpr int g = decltype(G)::value;
                        f32x4 v;
                        static_for<0, 4>([&](auto K) PCD_INLINE { v[decltype(K)::value] = acc[i][j][4 * g + decltype(K)::value]; });
                        tok_stage<OP>(stage, j % NBJ, g, v);
                    });
                    if constexpr (j % NBJ == NBJ - 1)
                        tok_flush<OPB, NBJ>(stage, P.dout, P.ldo, row0 + wm * C::WTM + i * 32,
                                            col0 + wn * C::WTN + (j - j % NBJ) * 32, live, t->out_n);
                });
                __builtin_amdgcn_sched_barrier(0);
            });
        }
    }
}

// The product's Problem leads the kernel's arguments: phase_unit reads it from
// the kernarg segment.
template <typename OP, int BM, int BN, int EPI>
__global__ void __launch_bounds__((TileCfg<BM, BN, OpTraits<OP>::bytes>::NT), (TileCfg<BM, BN, OpTraits<OP>::bytes>::OCC))
tok_kernel(const Problem p, const PhaseArgs args, const TokArgs tok) {
    __shared__ __attribute__((aligned(16))) char smem[phase_smem_bytes<OP, BM, BN>()];
    phase_unit<OP, BM, BN, EPI>((KProblem*)__builtin_amdgcn_kernarg_segment_ptr(), 1, args, tok.unit0 + blockIdx.x, gridDim.x,
                                smem, &tok);
}

// DH on the first dh_grid workgroups and DW on the rest (either may have none).
// 2048 x 50257 x 2048 bf16 (1229 rows live): DH 276 us and DW 290 as launches of
// their own, 40 tiles in 6 ranges and 1576 tiles in 6.2 rounds.
struct TokPair {
    Problem dh, dw;   // first: read from the kernarg segment
    PhaseArgs dh_args, dw_args;
    TokArgs dh_tok, dw_tok;
    int dh_grid;      // a multiple of the XCDs
};
template <typename OP, int BM, int BN>
__global__ void __launch_bounds__((TileCfg<BM, BN, OpTraits<OP>::bytes>::NT), (TileCfg<BM, BN, OpTraits<OP>::bytes>::OCC))
tok_pair_kernel(const TokPair p) {
    __shared__ __attribute__((aligned(16))) char smem[phase_smem_bytes<OP, BM, BN>()];
    KProblem* problems = (KProblem*)__builtin_amdgcn_kernarg_segment_ptr();
    if ((int)blockIdx.x < p.dh_grid)
        phase_unit<OP, BM, BN, EPI_TOK_DH>(problems, 1, p.dh_args, blockIdx.x, p.dh_grid, smem, &p.dh_tok);
    else
        phase_unit<OP, BM, BN, EPI_TOK_DW>(problems + 1, 1, p.dw_args, blockIdx.x - p.dh_grid, gridDim.x - p.dh_grid, smem,
                                           &p.dw_tok);
}

// What `tiles` tiles of DH, sweeps of k in r ranges, take in elements of K a CU
// sweeps: whole rounds over the CUs, a range costing its start and end (`ends`),
// and 16 for the sum it writes and scatter_rows_kernel reads.
__host__ __device__ inline float ranges_cost(int tiles, int k, int ends, int r, int cus) {
    return (float)((tiles * r + cus - 1) / cus) * ((float)k / r + ends) + 16.f * r;
}

}  // namespace pcd
