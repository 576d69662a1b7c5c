// token_aux.hpp -- the token losses' kernels that are not products (packing of
// the live rows, the teacher's slots, the rows' losses, few rows' forms), and the
// loads, stores and block sums that the embedding's kernels share with them.
// Included by the host translation unit only.
#pragma once
#include "token_kernels.hpp"

namespace pcd {

// ------------------------------------------------------------- block sums

// Sum (or maximum) of one value per thread over 256 threads, in a fixed order;
// every thread gets it.  `red`: 4 words of LDS, free again after the next barrier.
template <typename T, typename F> __device__ __forceinline__ T block_join(T v, T* red, F&& join) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = join(v, __shfl_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return join(join(red[0], red[1]), join(red[2], red[3]));
}

__device__ __forceinline__ void round_to(float& o, float x) { o = x; }
__device__ __forceinline__ void round_to(bf16_t& o, float x) { o.v = to_bf16(x); }
__device__ __forceinline__ void round_to(f16_t& o, float x) { o.v = to_f16(x); }

// ---------------------------------------------------------- units of a row

// Elements e .. e + N - 1 (8, or 4) of a row as fp32 and back; elements at or
// past n (the same for the whole wave) read as zero and are not written.
//
// A load is in two parts, so that a lane can have several on their way: Unit's
// has no branch (a lane whose unit the row's end breaks takes the last whole one),
// and `get` moves that down and converts.  With one branch for whole units and one
// that gathers a broken one's elements, each load was waited for in its branch
// (embedding gradients of 14458 x 277 bf16, vocabulary 1472: 79 us, 50 so; 512 x 320
// fp32, vocabulary 108059: 39 and 35; 16384 x 4096 bf16, vocabulary 131072: 246 and 240).
template <int N, typename T> struct Unit {
    static constexpr int OPB = OpTraits<T>::bytes, WORDS = N * OPB / 4, PER = 4 / OPB;   // elements of a word
    static_assert(N == 8 || N == 4, "units of 8 or 4 elements");
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T* row, int e, int n) {
        if (n < N) {
#pragma unroll
            for (int k = 0; k < WORDS; ++k) w[k] = 0u;
            for (int k = 0; k < N && e + k < n; ++k) {
                const float x = OpTraits<T>::load(row, e + k);
                put(k, x);
            }
            return;
        }
        const int at = min(e, n - N);
        if constexpr (WORDS == 2) {
            const u32x2 x = *(gu32x2c_any*)((const uint16_t*)row + at);
            w[0] = x[0], w[1] = x[1];
        } else {
#pragma unroll
            for (int q = 0; q < WORDS / 4; ++q) {
                const u32x4 x = *((gu32x4c_any*)((const char*)row + (size_t)at * OPB) + q);
#pragma unroll
                for (int k = 0; k < 4; ++k) w[4 * q + k] = x[k];
            }
        }
    }
    __device__ __forceinline__ void get(int e, int n, float (&v)[N]) const {
        const int down = n < N ? 0 : min(e - min(e, n - N), N);
        uint32_t x[WORDS];
#pragma unroll
        for (int k = 0; k < WORDS; ++k) x[k] = w[k];
        if (__any(down)) {
#pragma unroll
            for (int d = N; d >= PER; d /= 2)   // d elements down, or not
#pragma unroll
                for (int k = 0; k < WORDS; ++k) x[k] = down & d ? (k + d / PER < WORDS ? x[k + d / PER] : 0u) : x[k];
            if constexpr (PER == 2)
#pragma unroll
                for (int k = 0; k < WORDS; ++k) x[k] = down & 1 ? x[k] >> 16 | (k + 1 < WORDS ? x[k + 1] << 16 : 0u) : x[k];
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if constexpr (OPB == 4) {
                v[k] = __uint_as_float(x[k]);
            } else {
                const uint16_t h = (uint16_t)(x[k / 2] >> (16 * (k % 2)));
                v[k] = OpTraits<T>::load(&h, 0);
            }
        }
    }

private:
    // element k of a row shorter than a unit
    __device__ __forceinline__ void put(int k, float x) {
        T o;
        round_to(o, x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (j != k) continue;
            if constexpr (OPB == 4) w[j] = __float_as_uint(o);
            else w[j / 2] |= (uint32_t)o.v << (16 * (j % 2));
        }
    }
};
template <int N, typename T> __device__ __forceinline__ void load_n(const T* row, int e, int n, float (&v)[N]) {
    Unit<N, T> u;
    u.load(row, e, n);
    u.get(e, n, v);
}
template <int N, typename T> __device__ __forceinline__ void store_n(T* row, int e, int n, const float (&v)[N]) {
    if (e + N <= n) {
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
            const f32x4 x = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            if constexpr (OpTraits<T>::bytes == 4) {
                *(gu32x4_any*)((float*)row + e + 4 * q) = __builtin_bit_cast(u32x4, x);
            } else if constexpr (N == 8) {
                if (q == 0) {
                    const u32x2 a = OpTraits<T>::pack4(x), b = OpTraits<T>::pack4(f32x4{v[N - 4], v[N - 3], v[N - 2], v[N - 1]});
                    *(gu32x4_any*)((uint16_t*)row + e) = u32x4{a[0], a[1], b[0], b[1]};
                }
            } else {
                *(gu32x2_any*)((uint16_t*)row + e) = OpTraits<T>::pack4(x);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (e + k < n) OpTraits<T>::store(row, e + k, v[k]);
    }
}
template <typename T> __device__ __forceinline__ void load8(const T* row, int e, int n, float (&v)[8]) { load_n<8>(row, e, n, v); }
template <typename T> __device__ __forceinline__ void store8(T* row, int e, int n, const float (&v)[8]) { store_n<8>(row, e, n, v); }


// ---------------------------------------------------------------- live rows

// Ranges of DH's K for `rows` rows of it (us of a call by ranges, DH alone, 37 x
// 5003 x 256 fp32: 6 48.3, 12 40.1, 24 36.5, 32 37.3; 16 x 32000 x 2048 bf16: 4
// 84.8, 8 65.7, 16 70.2), the best alone whether DW is beside it: with fewer,
// longer ones, DW filling the rest, 1024 x 32000 x 2048 took 511 us for 487.  At
// most two rounds of them: the sums then take at most 2 `cus` tiles.  Each lane of a wave weighs one.
struct RangeArgs {
    int tile, tiles_n, k, ends, most, cus;   // DH's tile, column tiles, K, what a range's ends are worth of K, the most ranges
};
__device__ __forceinline__ int dh_ranges(const RangeArgs& a, int rows) {
    const int r = (threadIdx.x & 63) + 1, tiles = max(1, (rows + a.tile - 1) / a.tile) * a.tiles_n;
    float cost = __builtin_inff();
    if (r == 1 || (r <= a.most && (long)tiles * r <= 2 * a.cus))
        cost = ranges_cost(tiles, a.k, a.ends, r, a.cus);
    float least = cost;
#pragma unroll
    for (int d = 32; d; d >>= 1) least = fminf(least, __shfl_xor(least, d));
    return __ffsll((unsigned long long)__ballot(cost == least));
}

// Rows of a loss: what says which are live, and where the packed ones go.
struct RowArgs {
    const int* marks;          // live where 0 <= mark < limit
    const float* row_weight;   // ... and the weight is not 0 (nullable)
    int rows, limit;
    int* chunk;                // many rows: live ones in each kRowChunk, and the chunk's largest |weight| (null: few)
    int f16;                   // gradients carry a power of two
    TokCtl* ctl;
    int* map;                  // caller's row of each live row
    int* rank;                 // live row of each caller's row, -1 where it is left out
    float* loss;               // rows left out get 0 (a mark past the limit and a weight: NaN)
    int stack;                 // few rows: the second copy of each lies this many rows on (0: there is none)
    RangeArgs dh;
    u32x4* clear;              // counters of the products' split K, cleared on the way (nullable)
    int clear_units;
};
constexpr int kRowChunk = 1024;
constexpr int kFewRows = 8192;   // up to these every workgroup counts the live rows itself

__device__ __forceinline__ bool row_live(const RowArgs& a, int i) {
    const int m = gld(a.marks + i);
    return m >= 0 && m < a.limit && (a.row_weight == nullptr || gld(a.row_weight + i) != 0.f);
}
__device__ __forceinline__ float row_size(const RowArgs& a, int i) {
    return a.row_weight != nullptr ? fabsf(gld(a.row_weight + i)) : 1.f;
}

__device__ __forceinline__ float row_left_out(const RowArgs& a, int i) {
    const bool past = gld(a.marks + i) >= a.limit && (a.row_weight == nullptr || gld(a.row_weight + i) != 0.f);
    return past ? __builtin_nanf("") : 0.f;
}

// Gradients by the logits are held as multiples of the largest weight, so that
// rows of that weight (all of them, mostly) have targets of whole 1s: as w (q - 1)
// every one of them would round by the same part of itself (1 / 8028 in bf16 by
// 1.6e-3, which is then off the whole of dH and dW).  In f16 times 2^13:
// probabilities down to 2^-27 of it keep their bits.
__device__ __forceinline__ float grad_scale(float most, int f16) {
    const float range = f16 ? 8192.f : 1.f;
    return most > 0.f && most <= 3.402823466e38f ? fminf(range / most, 8.5e37f) : range;
}

__global__ void __launch_bounds__(256) count_rows_kernel(const RowArgs a) {
    __shared__ int ired[4];
    __shared__ float fred[4];
    int n = 0;
    float most = 0.f;
    for (int i = blockIdx.x * kRowChunk + threadIdx.x; i < min(a.rows, (int)(blockIdx.x + 1) * kRowChunk); i += 256)
        if (row_live(a, i)) {
            ++n;
            most = fmaxf(most, row_size(a, i));
        }
    n = block_join(n, ired, [](int x, int y) { return x + y; });
    most = block_join(most, fred, [](float x, float y) { return fmaxf(x, y); });
    if (threadIdx.x == 0) {
        a.chunk[2 * blockIdx.x] = n;
        a.chunk[2 * blockIdx.x + 1] = __float_as_int(most);
    }
}

// Rows r0 .. of a matrix [rows x cols], `lds` elements apart, into `out_rows` rows
// `ldd` apart, zero past the rows and the columns: the output matrix's last rows
// (and all of it, where its rows cannot be read in place).
struct CopyArgs {
    const void* src;
    long long lds, ldd;
    int r0, rows, cols, out_rows;
    void* dst;
};
template <typename OP>
__device__ __forceinline__ void copy_rows(const CopyArgs& a, size_t from, size_t step) {
    const int units = (int)((a.ldd + 7) / 8);
    for (size_t q = from; q < (size_t)a.out_rows * units; q += step) {
        const int r = (int)(q / units), e = (int)(q % units) * 8;
        float v[8] = {};
        if (a.r0 + r < a.rows) load8((const OP*)a.src + (size_t)(a.r0 + r) * a.lds, e, a.cols, v);
        store8((OP*)a.dst + (size_t)r * a.ldd, e, (int)a.ldd, v);
    }
}
template <typename OP> __global__ void __launch_bounds__(256) copy_rows_kernel(const CopyArgs a) {
    copy_rows<OP>(a, (size_t)blockIdx.x * 256 + threadIdx.x, (size_t)gridDim.x * 256);
}

// Packs the live rows of `hidden` (rows `ldh` apart) together in the operand
// type, `pitch` elements apart, zero from `dim` on; then rows of zeros up to
// whole K stages (at least one), which the products in K rows read.  A wave takes
// kGatherCols columns (blockIdx.y) of one of the caller's rows.  Up to kFewRows
// rows every workgroup counts for itself what is live before its rows: one
// launch, 8192 marks are 32 KB out of L2.  Workgroups past the rows' `row_blocks`
// copy the output matrix's last rows.
//
// A few rows (`stack`) go in twice, `stack` rows apart, for gradients in two
// parts: see grad_rows_kernel.
constexpr int kGatherCols = 2048;
template <typename OP, typename SRC>
__global__ void __launch_bounds__(256) gather_rows_kernel(const RowArgs a, const SRC* __restrict__ hidden, long long ldh,
                                                          int dim, OP* __restrict__ out, int pitch, int row_blocks,
                                                          const CopyArgs last) {
    if ((int)blockIdx.x >= row_blocks) {
        copy_rows<OP>(last, ((size_t)(blockIdx.x - row_blocks) * gridDim.y + blockIdx.y) * 256 + threadIdx.x,
                      (size_t)(gridDim.x - row_blocks) * gridDim.y * 256);
        return;
    }
    __shared__ float fred[4];
    const int q0 = blockIdx.x * 4, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int i = q0 + wave, e0 = blockIdx.y * kGatherCols + lane * 8;
    // the row's values, asked for before anything is counted
    constexpr int STEPS = kGatherCols / 512;
    Unit<8, SRC> u[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) u[k].load(hidden + (size_t)min(i, a.rows - 1) * ldh, e0 + k * 512, dim);
    const bool mine_live = i < a.rows && row_live(a, i);
    int before = 0, total = 0;
    float most = 0.f;
    if (a.chunk == nullptr) {
        for (int q = threadIdx.x; q < a.rows; q += 256)
            if (row_live(a, q)) {
                ++total;
                before += q < q0;
                if (blockIdx.x == 0) most = fmaxf(most, row_size(a, q));
            }
    } else {
        const int mine = q0 / kRowChunk, chunks = (a.rows + kRowChunk - 1) / kRowChunk;
        for (int c = threadIdx.x; c < chunks; c += 256) {
            const int n = gld(a.chunk + 2 * c);
            total += n;
            before += c < mine ? n : 0;
            most = fmaxf(most, __int_as_float(gld(a.chunk + 2 * c + 1)));
        }
        for (int q = mine * kRowChunk + threadIdx.x; q < min(q0, a.rows); q += 256) before += row_live(a, q);
    }
    __shared__ int lives[4];
    if (lane == 0) lives[wave] = mine_live;
    __shared__ int2 pair[4];
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        total += __shfl_xor(total, d);
        before += __shfl_xor(before, d);
    }
    if (lane == 0) pair[wave] = int2{total, before};
    __syncthreads();
    total = pair[0].x + pair[1].x + pair[2].x + pair[3].x;
    before = pair[0].y + pair[1].y + pair[2].y + pair[3].y;
    const int padded = a.stack ? 2 * a.stack : max(64, (total + 63) / 64 * 64);
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        for (int k = threadIdx.x; k < a.clear_units; k += 256) a.clear[k] = u32x4{0u, 0u, 0u, 0u};
        most = block_join(most, fred, [](float x, float y) { return fmaxf(x, y); });
        const int rows = a.stack ? padded : total;
        const int ranges = dh_ranges(a.dh, rows);
        if (threadIdx.x == 0) {
            const float g = grad_scale(most, a.f16);
            a.ctl->live = total;
            a.ctl->padded = padded;
            a.ctl->gscale = g;
            a.ctl->inv_gscale = 1.f / g;
            a.ctl->dh_rows = rows;
            a.ctl->dh_ranges = ranges;
        }
    }
    // rows of this workgroup, in order
    int rank = before;
    for (int w = 0; w < wave; ++w) rank += lives[w];
    if (i < a.rows && lane == 0 && blockIdx.y == 0) {
        a.rank[i] = mine_live ? rank : -1;
        if (mine_live) a.map[rank] = i;
        else a.loss[i] = row_left_out(a, i);
    }
    if (mine_live) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
            if (e0 + k * 512 < pitch) {
                float v[8];
                u[k].get(e0 + k * 512, dim, v);
                store8(out + (size_t)rank * pitch, e0 + k * 512, pitch, v);
                if (a.stack) store8(out + (size_t)(rank + a.stack) * pitch, e0 + k * 512, pitch, v);
            }
    }
    // row total + i is one of the zeros (stacked: its second copy too)
    const int z = total + i;
    if (z < (a.stack ? a.stack : padded)) {
        const float zero[8] = {};
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
            if (e0 + k * 512 < pitch) {
                store8(out + (size_t)z * pitch, e0 + k * 512, pitch, zero);
                if (a.stack) store8(out + (size_t)(z + a.stack) * pitch, e0 + k * 512, pitch, zero);
            }
    }
}

// ----------------------------------------------------------- teacher's slots

constexpr int kMaxTop = 1024;

// Row of a workgroup in a grid of one for each row (row_grid; kGridUnits).
__device__ __forceinline__ int grid_row() { return (int)(blockIdx.y * gridDim.x + blockIdx.x); }
inline dim3 row_grid(int rows) { return dim3(std::min(rows, kGridUnits), (rows + kGridUnits - 1) / kGridUnits); }

// One row's slots: sorted by id (a slot's place is the number of smaller ids and
// of equal ones before it), probabilities softmax(t / T) over the slots that
// are there, those of equal ids summed into the first; where each bucket of 64
// ids begins; sum p ln p; and whether the row has a slot at all.
template <typename TT>
__global__ void __launch_bounds__(256) teacher_kernel(const int* __restrict__ ids, const TT* __restrict__ logits, int rows, int top,
                                                      int vocab, float inv_t, int buckets, int* __restrict__ out_ids,
                                                      float* __restrict__ out_probs, uint16_t* __restrict__ starts,
                                                      float* __restrict__ plogp, int* __restrict__ marks) {
    __shared__ int raw_id[kMaxTop], id[kMaxTop];
    __shared__ float raw_t[kMaxTop], t[kMaxTop];
    __shared__ float fred[4];
    __shared__ int ired[4];
    const size_t row = grid_row();
    if (row >= (size_t)rows) return;
    const int none = 0x7FFFFFFF;
    float m = -__builtin_inff();
    int past = 0;
    for (int j = threadIdx.x; j < top; j += 256) {
        int v = gld(ids + row * top + j);
        const float x = OpTraits<TT>::load(logits, row * top + j);
        past |= v >= vocab && x != -__builtin_inff();
        const bool there = v >= 0 && v < vocab && x != -__builtin_inff();
        raw_id[j] = there ? v : none;
        raw_t[j] = there ? x : -__builtin_inff();
        if (there) m = fmaxf(m, x);
    }
    m = block_join(m, fred, [](float x, float y) { return fmaxf(x, y); });   // also: every slot is in LDS
    past = block_join(past, ired, [](int x, int y) { return x | y; });
    for (int j = threadIdx.x; j < top; j += 256) {
        int place = 0;
        const int v = raw_id[j];
        for (int k = 0; k < top; ++k) place += raw_id[k] < v || (raw_id[k] == v && k < j);
        id[place] = v;
        t[place] = v == none ? 0.f : expf((raw_t[j] - m) * inv_t);   // (a logit over T may overflow, this only to 0)
    }
    __syncthreads();
    float sum = 0.f;
    for (int j = threadIdx.x; j < top; j += 256) sum += t[j];
    sum = block_join(sum, fred, [](float x, float y) { return x + y; });
    float h = 0.f;
    for (int j = threadIdx.x; j < top; j += 256) {
        const int v = id[j];
        float p = 0.f;
        if (v != none && (j == 0 || id[j - 1] != v)) {
            for (int k = j; k < top && id[k] == v; ++k) p += t[k];
            p /= sum;
        }
        out_ids[row * top + j] = v;
        out_probs[row * top + j] = p;
        if (p != 0.f) h += p * logf(p);
    }
    h = block_join(h, fred, [](float x, float y) { return x + y; });
    for (int b = threadIdx.x; b <= buckets; b += 256) {
        int lo = 0, hi = top;   // the first slot at or past the bucket's first id
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (id[mid] < b * kTokBucket) lo = mid + 1;
            else hi = mid;
        }
        starts[row * (buckets + 1) + b] = (uint16_t)lo;
    }
    if (threadIdx.x == 0) {
        plogp[row] = h;
        marks[row] = past ? none : id[0] != none ? 0 : -1;
    }
}

// -------------------------------------------------------------- row losses

__device__ __forceinline__ void join_sums(float& m, float& s, float om, float os) {
    const float top = fmaxf(m, om), base = top == -__builtin_inff() ? 0.f : top;
    s = s * __builtin_amdgcn_exp2f(m - base) + os * __builtin_amdgcn_exp2f(om - base);
    m = top;
}
// One of `width` threads' share of a row's sums, eight of them loaded at once
// (one after the other they were all of row_loss_kernel's time).
__device__ __forceinline__ float2 row_share(const TokArgs& t, int r, int at, int width) {
    const auto* part = (const __attribute__((address_space(1))) u32x2*)(t.part + (size_t)r * t.slots);
    float m = -__builtin_inff(), s = 0.f;
    for (int k = at; k < t.slots; k += 8 * width) {
        float x[8], y[8], top = m;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const u32x2 p = part[min(k + j * width, t.slots - 1)];
            x[j] = k + j * width < t.slots ? __uint_as_float(p[0]) : -__builtin_inff();
            y[j] = __uint_as_float(p[1]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
        const float base = top == -__builtin_inff() ? 0.f : top;
        s *= __builtin_amdgcn_exp2f(m - base);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += y[j] * __builtin_amdgcn_exp2f(x[j] - base);
        m = top;
    }
    return float2{m, s};
}
// log2 of a row's sum of exponentials from the 256 threads' shares; every thread of
// the workgroup gets it.
__device__ __forceinline__ float join_shares(float2 mine, float2* red) {
#pragma unroll
    for (int d = 32; d; d >>= 1) join_sums(mine.x, mine.y, __shfl_xor(mine.x, d), __shfl_xor(mine.y, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mine;
    __syncthreads();
    mine = red[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) join_sums(mine.x, mine.y, red[w].x, red[w].y);
    return (mine.x == -__builtin_inff() ? 0.f : mine.x) + log2f(mine.y);
}
// What a row's loss needs besides: asked for before the sums are joined.
struct RowTarget {
    float got, w, plogp;   // this thread's targets' logits by their probabilities; the row's weight, sum p ln p
};
__device__ __forceinline__ RowTarget row_target(const TokArgs& t, int r, int orig) {
    RowTarget x = {0.f, t.row_weight != nullptr ? gld(t.row_weight + orig) : 1.f, t.plogp != nullptr ? gld(t.plogp + orig) : 0.f};
    const float* z = t.z + (size_t)r * t.z_cols;   // where LSE's epilogue did not take the targets' out
    if (t.labels != nullptr) {
        x.got = t.taken != nullptr ? gld(t.taken + orig) : gld(z + gld(t.labels + orig));
    } else {
        for (int j = threadIdx.x; j < t.top; j += 256) {
            const size_t at = (size_t)orig * t.top + j;
            const float p = gld(t.probs + at);
            if (p != 0.f) x.got += p * (t.taken != nullptr ? gld(t.taken + at) : gld(z + gld(t.ids + at)));
        }
    }
    return x;
}
// The row's loss.
__device__ __forceinline__ void close_row(const TokArgs& t, int orig, float l2, RowTarget x, float* fred) {
    if (t.labels == nullptr) x.got = block_join(x.got, fred, [](float x, float y) { return x + y; });
    if (threadIdx.x == 0) t.loss[orig] = x.w * t.factor * (x.plogp + 0.6931471805599453f * (l2 - x.got));
}
__global__ void __launch_bounds__(256) row_loss_kernel(const TokArgs t, int rows) {
    __shared__ float fred[4];
    __shared__ float2 red[4];
    const int r = min(grid_row(), rows - 1), live = gld(&t.ctl->live), orig = gld(t.map + r);   // (past the live rows: whatever is there)
    const float2 mine = row_share(t, r, threadIdx.x, 256);
    if (grid_row() >= live) return;
    const RowTarget x = row_target(t, r, orig);
    const float l2 = join_shares(mine, red);
    if (threadIdx.x == 0) t.lse2[r] = l2;
    close_row(t, orig, l2, x, fred);
}

// c + the products of one 32-bit word of two operand vectors: an fp32 pair, or two
// pairs of a 16-bit type (exact products, summed in fp32; one instruction where
// unpacking both would take five, and the vector units then hold the stream up).
template <typename OP> __device__ __forceinline__ float dot_word(uint32_t a, uint32_t b, float c) {
    if constexpr (OpTraits<OP>::bytes == 4) {
        return __builtin_fmaf(__uint_as_float(a), __uint_as_float(b), c);
    } else if constexpr (std::is_same<OP, bf16_t>::value) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a), __builtin_bit_cast(bf16x2, b), c, false);
    } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, a), __builtin_bit_cast(f16x2, b), c, false);
    }
}

// One to kFewTok rows (kFewTok16 of a 16-bit type): what gather_rows_kernel and LSE do, in one launch that
// streams W.  A product of so few rows is W's read and nothing else; a wave takes
// four of W's rows at a time, whole, 16 bytes a lane, against the hidden states
// in LDS.  The 4 NR sums over its lanes halve as they go (each lane keeps half of
// what it holds and gives the other half away: 7, 10, 17 and 32 exchanges with 1,
// 2, 4 and 8 rows, for 24 NR),
// and a lane keeps the running sum of its own logits.  Every workgroup finds the
// live ones of the few rows by itself.  All logits are kept, 4 bytes to a row of
// W.  `nt`: W is larger than the caches, so its lines are not kept in them.
// `ranges`: of few_grads_kernel.
// With 8 rows the vector units' products are what 16-bit types wait for, and the
// matrix tiles take half the time where W's rows are whole (us, loss / both
// gradients, so and on the tiles: 8 x 32768 x 4096 bf16 81 / 229 and 69 / 203, 5 x
// 18688 x 1661 36 / 118 and 47 / 97, 4 x 48508 x 576 f16 23 / 77 and 31 / 85; 6 x
// 91008 x 2048 fp32 146 / 495 and 260 / 750).
constexpr int kFewTok = 8, kFewTok16 = 4, kFewLds = 64 * 1024;
template <typename OP, typename SRC, int NR>
__global__ void __launch_bounds__(256) few_rows_kernel(const RowArgs a, const TokArgs t, const SRC* __restrict__ hidden,
                                                       long long ldh, int dim, int pitch, const OP* __restrict__ W,
                                                       long long ldw, int vocab, int nt, int ranges) {
    constexpr int OPB = OpTraits<OP>::bytes, UE = 16 / OPB, G = 4;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float2 red[4][NR];
    // [live row][pitch], then [live row][UE]: the row's last UE, of which only
    // those past the last whole unit count (the others are zeros here)
    OP* h = (OP*)smem;
    OP* tails = h + NR * pitch;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // This wave's steps: groups of G rows of W, each `sweep` steps of 64 units; the
    // next FLY steps' loads are always on their way, the first ones before
    // anything else is looked at.  (Calls of 1 / 4 rows, 32768 x 4096 bf16, cold:
    // 56 / 64 us; G = 2 with 8 on their way 56 / 64, 4 with 4 55 / 69, 8 with 2
    // 68 / 83.  268 MB in the kernel's 49 us are 5.5 TB/s; reads of 3 GB reach 6.8.)
    constexpr int FLY = 2;
    const int sweep = (dim + 64 * UE - 1) / (64 * UE), stride = gridDim.x * 4 * G, first = (blockIdx.x * 4 + wave) * G;
    const int steps = first < vocab ? ((vocab - first + stride - 1) / stride) * sweep : 0;
    u32x4 w[FLY][G];
    int next_v = first, next_e = 0;   // the next step to load
    auto load = [&](u32x4 (&to)[G]) PCD_INLINE {
        const int e = min(next_e * (64 * UE) + lane * UE, dim - UE);   // past the row's end: multiplied by zeros
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const auto* at = (gu32x4c_any*)(W + (size_t)min(next_v + j, vocab - 1) * ldw + e);
            to[j] = nt ? __builtin_nontemporal_load(at) : *at;
        }
        if (++next_e == sweep) next_e = 0, next_v += stride;
    };
#pragma unroll
    for (int k = 0; k < FLY; ++k)
        if (k < steps) load(w[k]);
    const bool mine = lane < a.rows && row_live(a, lane);   // every row at once, a lane each
    const uint64_t lives = __ballot(mine);
    const int live = __popcll(lives);
    if (blockIdx.x == 0 && wave == 0 && lane < a.rows) {
        const int r = __popcll(lives & ((1ull << lane) - 1));
        a.rank[lane] = mine ? r : -1;
        if (mine) a.map[r] = lane;
        else a.loss[lane] = row_left_out(a, lane);
    }
    int orig[NR];
    uint64_t rest = lives;
#pragma unroll
    for (int r = 0; r < NR; ++r, rest &= rest - 1) orig[r] = __ffsll((unsigned long long)rest) - 1;   // -1: none
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.ctl = TokCtl{live, live, 1.f, 1.f, live, ranges};
#pragma unroll
    for (int r = 0; r < NR; ++r)
        for (int e = threadIdx.x * 8; e < pitch; e += 2048) {
            float v[8] = {};
            if (orig[r] >= 0) load8(hidden + (size_t)orig[r] * ldh, e, dim, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                round_to(h[r * pitch + e + k], v[k]);
                const int tail = e + k - (dim - UE);
                if (tail >= 0 && tail < UE) round_to(tails[r * UE + tail], e + k >= dim / UE * UE ? v[k] : 0.f);
            }
        }
    __syncthreads();
    // logits
    constexpr int N = G * NR, SPAN = 64 / N;   // SPAN lanes hold sum i = G r + j: lanes SPAN i ..
    const int row = lane / SPAN / G, j0 = lane / SPAN % G;
    float m = -__builtin_inff(), s = 0.f;
    float acc[G][NR] = {};
    int v0 = first, step = 0;
    auto multiply = [&](const u32x4 (&wv)[G]) PCD_INLINE {
        const int e = step * (64 * UE) + lane * UE;
        u32x4 x[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r)
            x[r] = e < dim ? *(const u32x4*)(e + UE <= dim ? h + r * pitch + e : tails + r * UE) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
                for (int j = 0; j < G; ++j) acc[j][r] = dot_word<OP>(wv[j][k], x[r][k], acc[j][r]);
    };
    auto finish = [&]() PCD_INLINE {   // the group's logits
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = acc[i % G][i / G], acc[i % G][i / G] = 0.f;
        static_for<0, 6>([&](auto Sc) PCD_INLINE {
            constexpr int d = 32 >> decltype(Sc)::value, half = N >> (decltype(Sc)::value + 1);
            if constexpr (half == 0) {
                x[0] += __shfl_xor(x[0], d);
            } else {
                const bool up = lane & d;
                static_for<0, half>([&](auto I) PCD_INLINE {
                    constexpr int i = decltype(I)::value;
                    x[i] = (up ? x[i + half] : x[i]) + __shfl_xor(up ? x[i] : x[i + half], d);
                });
            }
        });
        const int v = v0 + j0;
        const float z = v < vocab ? x[0] * t.scale2 : -__builtin_inff();
        const float top = fmaxf(m, z), base = top == -__builtin_inff() ? 0.f : top;
        s = s * __builtin_amdgcn_exp2f(m - base) + __builtin_amdgcn_exp2f(z - base);
        m = top;
        if (lane % SPAN == 0 && row < live && v < vocab) gst(t.z + (size_t)row * t.z_cols + v, z);
    };
    for (int i = 0; i < steps; i += FLY) {
        static_for<0, FLY>([&](auto Kc) PCD_INLINE {
            constexpr int k = decltype(Kc)::value;
            if (i + k < steps) {
                multiply(w[k]);
                if (i + k + FLY < steps) load(w[k]);
                if (++step == sweep) {
                    finish();
                    step = 0;
                    v0 += stride;
                }
            }
        });
    }
#pragma unroll
    for (int d = SPAN; d < SPAN * G; d *= 2) join_sums(m, s, __shfl_xor(m, d), __shfl_xor(s, d));
    if (lane % (SPAN * G) == 0) red[wave][row] = float2{m, s};
    __syncthreads();
    if ((int)threadIdx.x < live) {
        const int r = threadIdx.x;
        float top = red[0][r].x, sum = red[0][r].y;
        for (int w = 1; w < 4; ++w) join_sums(top, sum, red[w][r].x, red[w][r].y);
        t.part[(size_t)r * t.slots + blockIdx.x] = float2{top, sum};
    }
}

// Both gradients of those few rows in one more stream of W: G = w (q - p) of 64
// ids at a time from the kept logits, a lane each, in fp32; then id after id
// dH += G W and dW = G H on 16 bytes a lane, H's columns and dH's sums in
// registers.  A workgroup takes a range of the ids; its four waves stand side by
// side on the row (`across` of them, the next four on blockIdx.y), so that dW goes
// out in runs as long as they can be, and on narrow rows take `step` ids in turn.
// Each range's dH is a slab that scatter_rows_kernel sums.  Bound by W's read and
// dW's write (1 x 32768 x 4096 bf16: 537 MB in 99 us, 5.4 TB/s; 6 x 91008 x 2048
// fp32: 1.5 GB in 326, 4.6).  Of a row's last, broken unit the lane takes the row's
// last whole one instead: what two lanes then write is the same.  Every workgroup
// joins the rows' sums for itself; the first ones close a loss each.
struct FewArgs {
    const void* hidden;
    long long ldh;
    int dim, vocab, pitch, across, step, span;   // span: ids of a range, whole turns of its waves
    const void* W;
    long long ldw;
    float* slabs;   // [range][live row][pitch]; null: no dH
    void* dw;       // null: no dW
    long long lddw;
    float alpha;
    int nt;
};
template <typename OP, typename SRC, int NR>
__global__ void __launch_bounds__(256) few_grads_kernel(const FewArgs a, const TokArgs t) {
    constexpr int OPB = OpTraits<OP>::bytes, UE = 16 / OPB, FLY = 4;
    __shared__ float lse[NR], sums[4][64 * UE + UE], fred[4];
    const int ways = 4 / a.across;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, live = gld(&t.ctl->live);
    const int side = wave % a.across, turn = wave / a.across;
    const int col0 = (blockIdx.y * 4 + side) * 64 * UE, e = col0 + lane * UE, at = min(e, a.dim - UE);
    const bool on = e < a.dim;
    float h[NR][UE], sum[NR][UE] = {}, f[NR];
    int orig[NR], label[NR];
    {   // every row at once, a lane each
        const bool there = lane < live;
        const int o = there ? gld(t.map + lane) : 0;
        const float w = !there ? 0.f : t.row_weight != nullptr ? gld(t.row_weight + o) : 1.f;
        const int l = there && t.labels != nullptr ? gld(t.labels + o) : -1;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            orig[r] = r < live ? __builtin_amdgcn_readlane(o, r) : -1;
            f[r] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), r));
            label[r] = __builtin_amdgcn_readlane(l, r);
        }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) load_n<UE>((const SRC*)a.hidden + (size_t)max(orig[r], 0) * a.ldh, at, a.dim, h[r]);
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int k = 0; k < UE; ++k) {
            OP o;
            round_to(o, h[r][k]);
            h[r][k] = orig[r] >= 0 ? a.alpha * OpTraits<OP>::load(&o, 0) : 0.f;
        }
    for (int r = wave; r < live; r += 4) {
        float2 all = row_share(t, r, lane, 64);
#pragma unroll
        for (int d = 32; d; d >>= 1) join_sums(all.x, all.y, __shfl_xor(all.x, d), __shfl_xor(all.y, d));
        if (lane == 0) lse[r] = (all.x == -__builtin_inff() ? 0.f : all.x) + log2f(all.y);
    }
    __syncthreads();
    if (blockIdx.y == 0)
        for (int r = blockIdx.x; r < live; r += gridDim.x) {
            const int o = gld(t.map + r);
            close_row(t, o, lse[r], row_target(t, r, o), fred);
        }
    const int end = turn < ways ? min(a.vocab, (int)(blockIdx.x + 1) * a.span) : 0;
    for (int v0 = blockIdx.x * a.span + turn * a.step; v0 < end; v0 += ways * a.step) {
        u32x4 w[2][FLY];
        auto load = [&](u32x4 (&to)[FLY], int k0) PCD_INLINE {
#pragma unroll
            for (int j = 0; j < FLY; ++j) {
                const auto* from = (gu32x4c_any*)((const OP*)a.W + (size_t)min(v0 + k0 + j, a.vocab - 1) * a.ldw + at);
                to[j] = a.nt ? __builtin_nontemporal_load(from) : *from;
            }
        };
        const int v = v0 + lane;
        float g[NR];
        int slot[NR], last[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {   // of the last live row where there is none
            g[r] = gld(t.z + (size_t)max(min(r, live - 1), 0) * t.z_cols + min(v, a.vocab - 1));
            slot[r] = last[r] = 0;
            if (t.labels == nullptr) {
                const gu16* b = (const gu16*)(t.starts + (size_t)max(orig[r], 0) * (t.buckets + 1) + v0 / kTokBucket);
                slot[r] = b[0], last[r] = b[1];
            }
        }
        if (a.slabs != nullptr) load(w[0], 0), load(w[1], FLY);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            g[r] = r < live && v < a.vocab ? __builtin_amdgcn_exp2f(g[r] - lse[r]) : 0.f;
            if (v == label[r]) g[r] -= 1.f;
            if (r < live)
                for (int s = slot[r]; s < last[r]; ++s) {
                    const size_t i = (size_t)orig[r] * t.top + s;
                    const float p = gld(t.probs + i);
                    if (p != 0.f && v == gld(t.ids + i)) g[r] -= p;
                }
            g[r] *= f[r];
        }
        for (int k0 = 0; k0 < a.step; k0 += 2 * FLY) {
            static_for<0, 2>([&](auto B) PCD_INLINE {
                constexpr int b = decltype(B)::value;
#pragma unroll
                for (int j = 0; j < FLY; ++j) {
                    const int k = k0 + b * FLY + j;
                    float u[UE], o[UE] = {};
#pragma unroll
                    for (int i = 0; i < UE; ++i) {
                        const uint32_t word = w[b][j][i * OPB / 4];
                        if constexpr (OPB == 4) u[i] = __uint_as_float(word);
                        else if constexpr (std::is_same<OP, bf16_t>::value) u[i] = __uint_as_float(i % 2 ? word & 0xFFFF0000u : word << 16);
                        else u[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(word >> (16 * (i % 2))));
                    }
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const float gr = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g[r]), k));
                        if (a.slabs != nullptr) {
#pragma unroll
                            for (int i = 0; i < UE; ++i) sum[r][i] = __builtin_fmaf(gr, u[i], sum[r][i]);
                        }
#pragma unroll
                        for (int i = 0; i < UE; ++i) o[i] = __builtin_fmaf(gr, h[r][i], o[i]);
                    }
                    if (a.dw != nullptr && on && v0 + k < a.vocab) {
                        u32x4 out;
                        if constexpr (OPB == 4) {
                            out = __builtin_bit_cast(u32x4, f32x4{o[0], o[1], o[2], o[3]});
                        } else {
                            const u32x2 lo = OpTraits<OP>::pack4(f32x4{o[0], o[1], o[2], o[3]});
                            const u32x2 hi = OpTraits<OP>::pack4(f32x4{o[UE - 4], o[UE - 3], o[UE - 2], o[UE - 1]});
                            out = u32x4{lo[0], lo[1], hi[0], hi[1]};
                        }
                        *(gu32x4_any*)((OP*)a.dw + (size_t)(v0 + k) * a.lddw + at) = out;
                    }
                }
                if (a.slabs != nullptr && k0 + 2 * FLY < a.step) load(w[b], k0 + (2 + b) * FLY);
            });
        }
    }
    if (a.slabs == nullptr) return;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        if (r >= live) break;
        __syncthreads();
        if (on)
#pragma unroll
            for (int i = 0; i < UE; ++i) sums[wave][at - col0 + UE + i] = sum[r][i];
        __syncthreads();
        if (turn == 0)
            for (int c = lane; c < 64 * UE && col0 + c < a.dim; c += 64) {
                float v = 0.f;
                for (int k = 0; k < ways; ++k) v += sums[side + k * a.across][c + UE];
                a.slabs[((size_t)blockIdx.x * live + r) * a.pitch + col0 + c] = v;
            }
    }
}

// G's piece from logits that LSE kept: the counterpart of the GRAD product.  A
// workgroup takes kGradCols columns of a row (blockIdx.y), in LDS while the
// targets are taken off; rows past the live ones, up to whole K stages, are
// zeros.  `close`: it joins the rows' sums and closes their losses too, each
// workgroup for itself (a launch less where there are few).
//
// A few rows (`stack`) go out in two parts, the value in the operand type and
// what that left of it, `stack` rows on: DH adds its results' two halves up, DW
// has the hidden states twice.  The products of so few rows are bound by
// reading W whatever their rows, and a gradient of one or two large elements
// would else be off by what those round (bf16 up to 4e-3; the mean over
// hundreds of rows is 1.7e-3 and less).
constexpr int kGradCols = 2048;
template <typename OP>
__global__ void __launch_bounds__(256) grad_rows_kernel(const TokArgs t, OP* __restrict__ out, int ldo, int n, int n64,
                                                        int close, int stack) {
    __shared__ float v[kGradCols];
    __shared__ float fred[4];
    __shared__ float2 red[4];
    const int r = blockIdx.y, c0 = blockIdx.x * kGradCols, cols = min(kGradCols, n64 - c0);
    if (r >= gld(&t.ctl->padded)) return;
    OP* row = out + (size_t)r * ldo + c0;
    const int e = threadIdx.x * 8;
    if (r >= gld(&t.ctl->live)) {
        const float zero[8] = {};
        if (e < cols) store8(row, e, cols, zero);
        if (e < cols && stack) store8(row + (size_t)stack * ldo, e, cols, zero);
        return;
    }
    float q[8] = {};
    if (e < cols) {   // z_cols and id0 are whole 64s
        const size_t at = (size_t)r * t.z_cols + t.id0 + c0 + e;
        if (std::is_same<OP, bf16_t>::value && t.zq != nullptr) {
            const u32x4 w = *(const __attribute__((address_space(1))) u32x4*)(t.zq + at);
            const float top = gld(t.ztop + at / 32);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t c = w[k / 2] >> (16 * (k % 2)) & 0xFFFF;
                q[k] = c == 65535 ? -__builtin_inff() : __builtin_fmaf((float)c, -1.f / kTokCode, top);
            }
        } else {
            const f32x4 a = gld4(t.z + at), b = gld4(t.z + at + 4);
#pragma unroll
            for (int k = 0; k < 8; ++k) q[k] = k < 4 ? a[k] : b[k - 4];
        }
    }
    const int orig = gld(t.map + r);
    const float f = gld(&t.ctl->gscale) * (t.row_weight != nullptr ? gld(t.row_weight + orig) : 1.f);
    float l2;
    if (close) {
        const float2 mine = row_share(t, r, threadIdx.x, 256);
        RowTarget x;
        if (blockIdx.x == 0) x = row_target(t, r, orig);
        l2 = join_shares(mine, red);
        if (blockIdx.x == 0) close_row(t, orig, l2, x, fred);
    } else {
        l2 = gld(t.lse2 + r);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = c0 + e + k < n ? f * __builtin_amdgcn_exp2f(q[k] - l2) : 0.f;
    int first = 0, end = 0, id = 0;
    if (t.labels != nullptr) {
        id = gld(t.labels + orig) - t.id0 - c0;
        end = id >= 0 && id < cols;
    } else {
        const gu16* at = (const gu16*)(t.starts + (size_t)orig * (t.buckets + 1) + (t.id0 + c0) / kTokBucket);
        first = at[0], end = at[(cols + kTokBucket - 1) / kTokBucket];
    }
    if (first < end) {   // the same for the whole workgroup
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (e < cols) v[e + k] = q[k];
        __syncthreads();
        for (int s = first + threadIdx.x; s < end; s += 256) {
            float p = 1.f;
            const size_t slot = (size_t)orig * t.top + s;
            if (t.labels == nullptr) {
                id = gld(t.ids + slot) - t.id0 - c0;
                p = gld(t.probs + slot);
            }
            if (p != 0.f) {   // ids are distinct but for slots of probability 0
                if (std::is_same<OP, bf16_t>::value && t.zq != nullptr)
                    v[id] = f * (__builtin_amdgcn_exp2f(gld(t.taken + slot) - l2) - p);   // q - p cancels: not of a code
                else
                    v[id] -= f * p;
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (e < cols) q[k] = v[e + k];
    }
    if (e < cols) {
        store8(row, e, cols, q);
        if (stack) {
            OP hi[8];
            float lo[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) round_to(hi[k], q[k]);
#pragma unroll
            for (int k = 0; k < 8; ++k) lo[k] = q[k] - OpTraits<OP>::load(hi, k);
            store8(row + (size_t)stack * ldo, e, cols, lo);
        }
    }
}

// DW of a few rows: K = 64 KH (all of `padded`) in one go.  Its time is the
// output's, so a wave keeps H's fragments of its 128 columns in registers and
// walks down the vocabulary, 64 ids (a tile of G, [K x 64] in LDS, shared by four
// waves, the next one on its way) after another: the stores never stop for a tile's
// start.  On the product's tiles every 128 KB of output waited for a new tile's
// operands (16 x 32000 x 2048 bf16: 38 us for 131 MB).
constexpr int kSlimCols = 512, kSlimIds = 64, kSlimRing = 2;
template <int KH> constexpr int slim_smem() {   // the ring and the stores' regions; at first a wave's H, 16 KB at a time
    constexpr int run = kSlimRing * KH * 64 * kSlimIds * 2 + 4 * kStageWaveBytes, start = 4 * 64 * 128 * 2;
    return run > start ? run : start;
}
template <typename OP, int KH>
__global__ void __launch_bounds__(256, 2) slim_dw_kernel(const TokCtl* ctl, const OP* __restrict__ G, int ldg,
                                                         const OP* __restrict__ H, int pitch, int ids, int ids64, int dim,
                                                         float alpha, OP* __restrict__ out, long long ldo) {
    __shared__ __attribute__((aligned(16))) char smem[slim_smem<KH>()];
    constexpr int KC = 4 * KH, TILE = KH * 64 * kSlimIds * 2;   // chunks of 16, bytes of a tile of G
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    const int col0 = blockIdx.y * kSlimCols + wave * 128;
    alpha *= gld(&ctl->inv_gscale);
    // H's fragments: 64 rows of K at a time through the wave's 16 KB, laid out for tr_fragment<128>
    u32x4 b[KC][4];
    static_for<0, KH>([&](auto Hc) PCD_INLINE {
        constexpr int half = decltype(Hc)::value;
#pragma unroll
        for (int q = 0; q < 16; ++q) {   // 4 rows of 256 bytes a load
            const int k = q * 4 + lane / 16, unit = (lane % 16) ^ kn_swz<128>(k);
            const OP* src = H + (size_t)(half * 64 + k) * pitch + min(col0 + unit * 8, pitch - 8);
            lds_dma16(src, lds0 + wave * 16384 + q * 1024);
        }
        wait_vmcnt<0>();
        static_for<0, 4>([&](auto Cc) PCD_INLINE {
            static_for<0, 4>([&](auto J) PCD_INLINE {
                b[half * 4 + decltype(Cc)::value][decltype(J)::value] =
                    tr_fragment<128>(smem + wave * 16384, decltype(Cc)::value, decltype(J)::value * 32);
            });
        });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before the next half lands there
    });
    __syncthreads();
    const int tiles = ids64 / kSlimIds, step = gridDim.x;
    char* stage = smem + kSlimRing * TILE + wave * kStageWaveBytes;
    // tile `t` into slot `slot`: 8 rows of 128 bytes a load, this wave's share of them
    auto issue = [&](int t, int slot) PCD_INLINE {
#pragma unroll
        for (int q = 0; q < 2 * KH; ++q) {
            const int row = (wave * 2 * KH + q) * 8 + lane / 8, unit = (lane % 8) ^ kn_swz<64>(row);
            lds_dma16(G + (size_t)row * ldg + t * kSlimIds + unit * 8, lds0 + slot * TILE + (wave * 2 * KH + q) * 1024);
        }
    };
    int t = blockIdx.x, slot = 0;
    if (t < tiles) issue(t, 0);
    for (; t < tiles; t += step) {
        // One tile ahead.  Stores share the counter with the loads, so the wait is
        // for both; the next tile's loads are on their way meanwhile.
        wait_vmcnt<0>();
        __syncthreads();   // the tile is there, and the other slot no longer read
        const int next = slot ^ 1;
        if (t + step < tiles) issue(t + step, next);
        static_for<0, 2>([&](auto Vc) PCD_INLINE {
            constexpr int vb = decltype(Vc)::value;
            f32x16 acc[4] = {};
            static_for<0, KC>([&](auto Cc) PCD_INLINE {
                constexpr int c = decltype(Cc)::value;
                const u32x4 a = tr_fragment<64>(smem + slot * TILE, c, vb * 32);
                static_for<0, 4>([&](auto J) PCD_INLINE { mfma_chunk<OP>(acc[decltype(J)::value], b[c][decltype(J)::value], a); });
            });
            static_for<0, 4>([&](auto J) PCD_INLINE {
                constexpr int j = decltype(J)::value;
                static_for<0, 4>([&](auto Gc) PCD_INLINE {
                    constexpr int g = decltype(Gc)::value;
                    f32x4 v;
                    static_for<0, 4>([&](auto K) PCD_INLINE { v[decltype(K)::value] = alpha * acc[j][4 * g + decltype(K)::value]; });
                    tok_stage<OP>(stage, j % 2, g, v);
                });
                if constexpr (j % 2 == 1)
                    tok_flush<2, 2>(stage, out, (size_t)ldo, t * kSlimIds + vb * 32, col0 + (j - 1) * 32, ids, dim);
            });
        });
        slot = next;
    }
}

// dH of the live rows, summed over the ranges of K (and a stacked row's two
// parts), back to the caller's rows, zero in those left out (all of them without
// `rank`).  A wave takes 512 columns of a row.  WAYS 32, where that leaves the
// card idle: a workgroup 64 columns of a row, eight lanes a range, so that up to
// 256 ranges are on their way at once (calls of 32 x 10000 x 784 f16 45.7 us with WAYS 1,
// 40.6 with 32; 64 of them 47 / 43; 37 x 5003 x 256 fp32 39 / 37).
template <typename TD, int WAYS>
__global__ void __launch_bounds__(256) scatter_rows_kernel(const float* __restrict__ src, int pitch, const TokCtl* ctl,
                                                           const int* __restrict__ rank, int rows, int dim, float alpha,
                                                           TD* __restrict__ dst, long long ldd, int stack) {
    constexpr int LANES = WAYS == 1 ? 64 : 8, COLS = 8 * LANES;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int ranges = 1;
    size_t range = 0;
    if (ctl != nullptr) {
        alpha *= gld(&ctl->inv_gscale);
        ranges = gld(&ctl->dh_ranges);
        range = (size_t)gld(&ctl->dh_rows) * pitch;
    }
    const int chunks = (dim + COLS - 1) / COLS, from = WAYS == 1 ? 0 : threadIdx.x / LANES;
    const size_t tasks = (size_t)rows * chunks, first = WAYS == 1 ? (size_t)blockIdx.x * 4 + wave : blockIdx.x;
    for (size_t task = first; task < tasks; task += (size_t)gridDim.x * (WAYS == 1 ? 4 : 1)) {
        const size_t i = task / chunks;
        const int e = (int)(task - i * chunks) * COLS + lane % LANES * 8, r = rank != nullptr ? gld(rank + i) : -1;
        float v[8] = {};
        for (int half = 0; r >= 0 && half <= (stack > 0); ++half) {
            const float* at = src + (size_t)(r + half * stack) * pitch;
            for (int n = 0; n < ranges; n += 8 * WAYS) {   // the same for the whole wave
                f32x4 o[8][2];   // whole units: the pitch is
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (n + j * WAYS < ranges) {
                        const float* p = at + (size_t)min(n + from + j * WAYS, ranges - 1) * range + min(e, pitch - 8);
                        o[j][0] = gld4(p), o[j][1] = gld4(p + 4);
                    }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (n + j * WAYS < ranges)
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] += n + from + j * WAYS < ranges ? o[j][k / 4][k % 4] : 0.f;
            }
        }
        if constexpr (WAYS > 1) {
            __shared__ float others[4][COLS];
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int d = LANES; d < 64; d *= 2) v[k] += __shfl_xor(v[k], d);
            __syncthreads();
            if (lane < LANES)
#pragma unroll
                for (int k = 0; k < 8; ++k) others[wave][lane * 8 + k] = v[k];
            __syncthreads();
            if (threadIdx.x >= LANES) continue;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[k] = (others[0][lane * 8 + k] + others[1][lane * 8 + k]) + (others[2][lane * 8 + k] + others[3][lane * 8 + k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= alpha;
        store8(dst + i * ldd, e, dim, v);
    }
}

}  // namespace pcd
