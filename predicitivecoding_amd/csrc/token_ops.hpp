// token_ops.hpp -- the token operators' entry points: the host side of the
// embedding and of the losses over a vocabulary.  Part of the host translation
// unit (pcdevice.hip).
#pragma once
#include "token_embed.hpp"
#include "token_launch.hpp"

namespace {

// One block of the pool, cut into pieces of whole 256 bytes.
struct Arena {
    size_t size = 0;
    char* base = nullptr;
    size_t add(size_t bytes) {
        const size_t at = size;
        size += round_up(std::max<size_t>(bytes, 1), 256);
        return at;
    }
    template <typename T = void> T* at(size_t off) const { return (T*)(base + off); }
};

bool whole_words(const void* p, long long ld, int bytes) { return (uintptr_t)p % 4 == 0 && ld * bytes % 4 == 0; }

int device_cus(int* cus) {
    int dev = 0;
    HIP_TRY(hipGetDevice(&dev));
    HIP_TRY(hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev));
    return PCD_SUCCESS;
}

// f(a null pointer of dtype's element type)
template <typename F> int with_type(int dtype, F&& f) {
    switch (dtype) {
    case PCD_F32: return f((float*)nullptr);
    case PCD_BF16: return f((bf16_t*)nullptr);
    default: return f((f16_t*)nullptr);
    }
}
// ... for two types of which one is fp32 or both are the same
template <typename F> int with_types(int a, int b, F&& f) {
    return with_type(a, [&](auto* pa) {
        if (a == b) return f(pa, pa);
        if (b == PCD_F32) return f(pa, (float*)nullptr);
        return with_type(b, [&](auto* pb) { return f((float*)nullptr, pb); });
    });
}
bool known_type(int dtype) { return dtype == PCD_F32 || dtype == PCD_BF16 || dtype == PCD_F16; }
bool types_fit(int a, int b) { return known_type(a) && known_type(b) && (a == b || a == PCD_F32 || b == PCD_F32); }

unsigned blocks_for(size_t n, size_t per, size_t most) { return (unsigned)std::max<size_t>(1, std::min(most, (n + per - 1) / per)); }

// A C entry's body: no C++ exception leaves it.
template <typename F> int guarded(const char* name, F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return fail(PCD_OUT_OF_MEMORY, "%s: out of host memory", name);
    } catch (...) {
        return fail(PCD_UNKNOWN, "%s: unexpected exception", name);
    }
}

// ------------------------------------------------------------ token losses

template <typename OP>
int launch_token_op(int t, int epi, const Problem& p, const PhaseArgs& a, const TokArgs& k, int grid, hipStream_t s) {
    if constexpr (!std::is_same<OP, float>::value)
        if (t == 256) return from_hip(launch_token_tile<OP, 256, 256>(epi, p, a, k, grid, s), "tok_kernel launch");
    if (t == 128) return from_hip(launch_token_tile<OP, 128, 128>(epi, p, a, k, grid, s), "tok_kernel launch");
    return from_hip(launch_token_tile<OP, 64, 64>(epi, p, a, k, grid, s), "tok_kernel launch");
}

// What the products of one call share.
struct TokCall {
    int dtype, cus;
    hipStream_t s;
    SplitScratch split;
};

// Tiles.  A tile's time is its area times its sweep, k elements and a start and
// end worth some more, at the tile's rate.  Measured, all in us: 16-bit 128 x 128
// and 64 x 64 tiles multiply at 0.6 and 0.3 of the 256 x 256 tile's rate
// (2048 x 50257 x 2048 LSE 256 / 128 / 64: 404 / 500 / 692), fp32 64 x 64 tiles at
// 0.6 of the 128 x 128 tile's (1024 x 16000 x 1024: 207 against 299); starts and
// ends are worth 1000, 400 and 128 elements of k (LSE 256 x 32000 x 2048: 68 / 65 /
// 85, 64 x 10000 x 784: 34 / 26 / 20), DW's 400 at least, whose tiles end in
// stores to memory (16 x 32000 x 2048: 38 / 39 / 73).  In K rows the 16-bit 128 x
// 128 tile's reads cost it a sixth (DH 300 x 50257 x 1024: 256 152, 128 165).
int tile_ends(int t, bool dw = false) { return t == 256 ? 1000 : t == 128 || dw ? 400 : 128; }
double tile_rate(int dtype, int t, bool k_rows = false) {
    if (dtype == PCD_F32) return t == 64 ? 0.6 : 1.0;
    return t == 64 ? 0.3 : t == 256 ? 1.0 : k_rows ? 0.5 : 0.6;
}
long tile_count(long m, long n, int t) { return ((m + t - 1) / t) * ((n + t - 1) / t); }
// The tile with the least time, by a cost of the tile in elements of k.
template <typename F> int best_tile(int dtype, bool k_rows, F&& cost) {
    int best = 64;
    double least = 0;
    for (int t : {64, 128, 256}) {
        if (t == 256 && dtype == PCD_F32) continue;
        const double v = cost(t) * t * t / tile_rate(dtype, t, k_rows);
        if (t == 64 || v < least) best = t, least = v;
    }
    return best;
}
// LSE's and GRAD's: whole rounds of tiles over the CUs.
int logits_tile(const TokCall& c, long m, long n, long k) {
    return best_tile(c.dtype, false, [&](int t) {
        return (double)((tile_count(m, n, t) + c.cus - 1) / c.cus) * (k + tile_ends(t));
    });
}
// DH's [m x n] over k and, if dw_m, DW's [dw_m x n] over dw_k in one launch with
// it: what they sweep a CU in the mean, and some of a last tile.
int pair_tile(const TokCall& c, long m, long n, int k, int most, long dw_m, int dw_k) {
    return best_tile(c.dtype, true, [&](int t) {
        const int dh = m ? (int)tile_count(m, n, t) : 0, dw = (int)tile_count(dw_m, n, t);
        int ranges = 1;
        float alone = ranges_cost(dh, k, tile_ends(t), 1, c.cus);
        for (int r = 2; r <= most && (long)dh * r <= 2 * c.cus; ++r) {
            const float v = ranges_cost(dh, k, tile_ends(t), r, c.cus);
            if (v < alone) alone = v, ranges = r;
        }
        const int split = dw && t <= 128 && 2 * dw <= c.cus ? std::min(kMaxSplit, c.cus / dw) : 1;   // of DW's K
        const double unit = (double)dw_k / split + tile_ends(t, true);
        return dw ? ((double)dh * (k + ranges * tile_ends(t)) + dw * split * unit) / c.cus + 0.4 * unit : (double)alone;
    });
}

// A product's tile grid, its split of K where the tiles fill too few CUs (but
// DH's, whose ranges have sums of their own), and K stagger.
void lay_tiles(const TokCall& c, int t, Problem& p, PhaseArgs& a, bool may_split) {
    p.tiles_m = (p.M + t - 1) / t;
    p.tiles_n = (p.N + t - 1) / t;
    p.tiles = p.tiles_m * p.tiles_n;
    a.k_stagger = c.dtype == PCD_F32 ? 0 : auto_k_stagger(p.K / stage_k(c.dtype, Tile{t, t}));
    if (!may_split || p.tiles * 2 > c.cus) return;
    std::vector<ProblemSet> sets(1);
    std::memset(&sets[0], 0, sizeof(ProblemSet));
    sets[0].n = 1;
    sets[0].p[0] = p;
    assign_split(c.cus, 1, c.dtype, Tile{t, t}, c.split, sets, kSplitMinStages);
    p = sets[0].p[0];
}
int grid_of(size_t units) { return (int)((units + kXcds - 1) / kXcds * kXcds); }

// LSE or GRAD.
int logits_product(const TokCall& c, int epi, int t, Problem p, PhaseArgs a, const TokArgs& k) {
    lay_tiles(c, t, p, a, true);
    return with_type(c.dtype, [&](auto* op) {
        const int grid = grid_of(p.tiles);
        TokArgs kk = k;
        for (kk.unit0 = 0; kk.unit0 < grid; kk.unit0 += kGridUnits) {
            const int st = launch_token_op<std::remove_pointer_t<decltype(op)>>(t, epi, p, a, kk, std::min(grid - kk.unit0, kGridUnits), c.s);
            if (st) return st;
        }
        return (int)PCD_SUCCESS;
    });
}

template <typename OP> int launch_pair_op(int t, const TokPair& p, int grid, hipStream_t s) {
    if constexpr (!std::is_same<OP, float>::value)
        if (t == 256) return from_hip(launch_token_pair<OP, 256, 256>(p, grid, s), "tok_pair_kernel launch");
    if (t == 128) return from_hip(launch_token_pair<OP, 128, 128>(p, grid, s), "tok_pair_kernel launch");
    return from_hip(launch_token_pair<OP, 64, 64>(p, grid, s), "tok_pair_kernel launch");
}

// Bytes of gradient that a piece of the vocabulary may take: enough columns for
// long sweeps of DH, few enough that the piece is still in the 256 MB cache
// when DH and DW read it.
constexpr size_t kTokPieceBytes = (size_t)256 << 20;

// Bytes of logits that a call may keep between its two passes over the
// vocabulary (pcd_token_keep_logits); the columns past them are multiplied again.
std::atomic<size_t> g_keep_logits{(size_t)1 << 30};

// Rows whose 16-bit gradients by the logits are held in two parts: twice that
// many rows still fit the tiles that read W at memory speed.
constexpr int kTokStackRows = 64;

// Few rows' DW takes slim_dw_kernel, whose workgroups want 512 columns, from
// kSlimLeast of them on, but beside DH only from kSlimBytes of output on: below,
// what one launch for both saves is more.  Calls with both gradients of 8 to 64 rows,
// bf16, 512 to 4096 columns, on the tiles and slim: outputs of 128 to 384 MB 0.97 to
// 1.13 (1.04 in the mean of up to 32 rows, 1.06 of more), 64 and 96 MB 0.93 to 1.06
// (1.03 and 0.99), 16 and 32 MB 0.87 to 1.02 (0.99 and 0.91).  d_weight alone, us slim
// and not: 16 x 32000 x 2048 bf16 77 / 86, 40 x 50257 x 1024 79 / 89, 64 x 10000 x 784
// 32 / 35.
constexpr int kSlimLeast = 384;
constexpr size_t kSlimBytes = (size_t)112 << 20;

constexpr float kLog2E = 1.4426950408889634f;

struct Teacher {
    const int* ids;
    const void* logits;
    int dtype, top;
    float temperature;
};

// How a loss goes about its call: which kernels, their tiles, and what stays in scratch.
struct LossPlan {
    bool grads, few, in_place, last_copy, coded, slim, close;
    int ob, unit, pitch;                 // bytes of an element, elements of a load, the packed hidden states' row
    int few_nr, few_blocks, few_across, few_step, few_span, few_ranges, few_y;
    int stack;                           // rows apart of the two parts of G (0: one part)
    size_t rows_pad;                     // rows of G and of the packed hidden states
    long long wld;                       // row pitch of W, or of its copy
    int v0, buckets, top, t_lse, slots;
    int width;                           // of the vocabulary's pieces
    int z_cols;                          // columns whose logits are kept
    int dh_rows, dh_k, dh_most, dw_ids, t;
    size_t dh_units;
};
LossPlan plan_loss(const TokCall& c, const void* weight, long long ldw, int rows, int dim, int vocab, int top, bool d_hidden,
                   bool d_weight, size_t keep) {
    LossPlan p;
    std::memset(&p, 0, sizeof p);
    const int ob = p.ob = op_bytes(c.dtype), unit = p.unit = 16 / ob, pitch = p.pitch = (int)round_up(dim, kFeatPad);
    const int v64 = (int)round_up(vocab, 64);
    p.grads = d_hidden || d_weight;
    // A few rows stream W (few_rows_kernel, few_grads_kernel), if the hidden states
    // fit beside each other in LDS and the limit lets their logits be kept.
    p.few_nr = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
    p.few = rows <= (ob == 4 ? kFewTok : kFewTok16) && dim >= unit && p.few_nr * pitch * ob <= kFewLds && (size_t)rows * 4 * v64 <= keep;
    // Up to kTokStackRows rows of a 16-bit type: gradients in two parts (grad_rows_kernel).
    // Their logits are kept whole, which a low limit forbids.
    p.stack = !p.few && p.grads && ob == 2 && rows <= kTokStackRows && round_up(rows, 32) * 8 * v64 <= keep ? (int)round_up(rows, 32) : 0;
    p.rows_pad = p.stack ? 2 * p.stack : round_up(rows, 64);
    // W is read in place where its rows are whole 32-bit words, which the tiles'
    // loads take, and what a K sweep reads past a row's end is the next row
    // (multiplied by zeros); else a padded copy is.
    p.in_place = whole_words(weight, ldw, ob) && (dim % kFeatPad == 0 || (ldw == dim && dim >= kFeatPad));
    p.wld = p.in_place ? ldw : pitch;
    // The last rows' copy: where a sweep would read past the matrix's end.
    p.v0 = (vocab - 1) / 256 * 256;
    p.last_copy = p.in_place && !p.few && (dim % kFeatPad != 0 || (d_hidden && vocab % 64 != 0));
    p.buckets = (vocab + kTokBucket - 1) / kTokBucket;
    p.top = top;

    p.t_lse = logits_tile(c, rows, vocab, dim);
    p.few_blocks = std::max(1, std::min(4 * c.cus, (vocab + 15) / 16));
    // few_grads_kernel: as many workgroups as the CUs hold at once (four of one or two
    // rows, two of more: calls of 2 x 16832 x 1536 fp32 with four and two a CU 75 / 87 us,
    // 1 x 32768 x 4096 bf16 169 / 176, 4 x 32768 x 4096 199 / 187), over the columns
    // first, and shorter turns of the waves rather than fewer.
    const int few_cols = (dim + 64 * unit - 1) / (64 * unit);
    p.few_across = std::min(4, few_cols);
    p.few_y = (few_cols + 3) / 4;
    const int few_ways = 4 / p.few_across, few_want = ((p.few_nr <= 2 ? 4 : 2) * c.cus + p.few_y - 1) / p.few_y;
    const int few_ids = vocab / (few_ways * few_want);
    p.few_step = few_ids >= 64 ? 64 : few_ids >= 32 ? 32 : 16;   // whole parts of a bucket
    p.few_span = (int)round_up((vocab + few_want - 1) / few_want, few_ways * p.few_step);
    p.few_ranges = (vocab + p.few_span - 1) / p.few_span;
    p.slots = p.few ? p.few_blocks : (vocab + p.t_lse - 1) / p.t_lse;
    // pieces of the vocabulary, of like width
    p.width = (int)std::max<size_t>(256, std::min<size_t>(round_up(vocab, 256), kTokPieceBytes / (p.rows_pad * ob) / 256 * 256));
    const int pieces = (vocab + p.width - 1) / p.width;
    p.width = (int)round_up((vocab + pieces - 1) / pieces, 256);
    p.coded = c.dtype == PCD_BF16 && !p.few && !p.stack;   // kept logits: 17 bits each, or 32
    // All columns where they fit the limit (a stacked call's do), else whole pieces.
    const size_t fit = keep / (p.rows_pad * (p.coded ? 17 : 32) / 8);
    p.z_cols = p.few || (p.grads && fit >= (size_t)v64) ? v64 : p.grads ? (int)(fit / p.width * p.width) : 0;
    // Few rows with every logit kept: grad_rows_kernel closes the losses.
    p.close = p.grads && !p.few && p.z_cols >= vocab && pieces == 1 && p.rows_pad * ((vocab + kGradCols - 1) / kGradCols) <= (size_t)8 * c.cus;
    // Few rows, all of rows_pad always padded: DW in a kernel of its own (slim_dw_kernel).
    p.slim = d_weight && !p.few && ob == 2 && (p.stack || p.rows_pad == 64) && dim >= kSlimLeast &&
             (!d_hidden || (size_t)vocab * dim * ob >= kSlimBytes);
    p.dh_rows = !d_hidden || p.few ? 0 : p.stack ? (int)p.rows_pad : rows;
    p.dw_ids = d_weight && !p.slim && !p.few ? std::min(p.width, vocab) : 0;
    p.dh_k = std::min(p.width, vocab);                                     // K of a piece
    const int dh_least = vocab - (vocab - 1) / p.width * p.width;   // ... and of the last
    p.dh_most = std::max(1, std::min(64, dh_least / 128));
    p.t = pair_tile(c, p.dh_rows, dim, p.dh_k, p.dh_most, p.dw_ids, (int)p.rows_pad);
    p.dh_units = d_hidden && !p.few ? std::max<size_t>(tile_count(p.dh_rows, dim, p.t), p.dh_most > 1 ? 2 * c.cus : 0) : 0;
    return p;
}

// Both losses (`teacher` null: cross entropy).
int token_loss(int dtype, const void* hidden, int hidden_dtype, long long ldh, const void* weight, long long ldw,
               const int* labels, const Teacher* teacher, const float* row_weight, int rows, int dim, int vocab, float scale,
               float* loss, void* d_hidden, long long ld_dh, void* d_weight, long long ld_dw, hipStream_t s) {
    if (rows == 0) {
        if (!d_weight) return PCD_SUCCESS;
        return with_type(dtype, [&](auto* td) {   // a sum over no rows
            using TD = std::remove_pointer_t<decltype(td)>;
            hipLaunchKernelGGL((scatter_rows_kernel<TD, 1>), dim3(blocks_for((size_t)vocab * ((dim + 511) / 512), 4, 1 << 20)), dim3(256), 0, s,
                               (const float*)nullptr, 0, (const TokCtl*)nullptr, (const int*)nullptr, vocab, dim, 0.f,
                               (TD*)d_weight, ld_dw, 0);
            return from_hip(hipGetLastError(), "scatter_rows_kernel launch");
        });
    }
    TokCall c{dtype, 0, s, {}};
    if (int st = device_cus(&c.cus)) return st;
    const LossPlan plan = plan_loss(c, weight, ldw, rows, dim, vocab, teacher ? teacher->top : 1, d_hidden, d_weight,
                                    g_keep_logits.load(std::memory_order_relaxed));
    const bool grads = plan.grads, few = plan.few, in_place = plan.in_place, last_copy = plan.last_copy, coded = plan.coded;
    const bool slim = plan.slim, close = plan.close;
    const int ob = plan.ob, unit = plan.unit, pitch = plan.pitch, stack = plan.stack, v0 = plan.v0, buckets = plan.buckets;
    const int top = plan.top, slots = plan.slots, width = plan.width, z_cols = plan.z_cols, dh_rows = plan.dh_rows, t = plan.t;
    const int few_nr = plan.few_nr, few_blocks = plan.few_blocks, few_ranges = plan.few_ranges, few_y = plan.few_y;
    const size_t rows_pad = plan.rows_pad, dh_units = plan.dh_units;
    const long long wld = plan.wld;

    Arena m;
    const size_t o_ctl = m.add(sizeof(TokCtl)), o_map = m.add((size_t)rows * 4), o_rank = m.add((size_t)rows * 4);
    const size_t o_chunk = m.add((size_t)((rows + kRowChunk - 1) / kRowChunk) * 8);
    const size_t o_h = few ? 0 : m.add(rows_pad * pitch * ob + 256);
    const size_t o_w = in_place ? (last_copy ? m.add((size_t)257 * ldw * ob + 256) : 0)
                                : !few ? m.add((round_up(vocab, 64) + 1) * (size_t)pitch * ob) : 0;
    const size_t o_part = m.add((size_t)rows * slots * 8), o_taken = m.add((size_t)rows * top * 4);
    const size_t o_lse = m.add((size_t)rows * 4);
    const size_t o_z = z_cols ? m.add((few ? rows : rows_pad) * z_cols * (coded ? 2 : 4)) : 0;
    const size_t o_ztop = z_cols && coded ? m.add(rows_pad * (z_cols / 32) * 4) : 0;
    const size_t o_g = grads && !few ? m.add(rows_pad * width * ob) : 0;
    // `ranges` sums of [live x pitch], at most dh_units tiles in all (pitch: whole 64s, at most the column tiles)
    const size_t o_dh = d_hidden ? m.add(few ? (size_t)few_ranges * rows * pitch * 4 : dh_units * t * t * 4) : 0;
    size_t o_ids = 0, o_probs = 0, o_starts = 0, o_plogp = 0, o_marks = 0;
    if (teacher) {
        o_ids = m.add((size_t)rows * top * 4);
        o_probs = m.add((size_t)rows * top * 4);
        o_starts = m.add((size_t)rows * (buckets + 1) * 2);
        o_plogp = m.add((size_t)rows * 4);
        o_marks = m.add((size_t)rows * 4);
    }
    const size_t part_bytes = (size_t)c.cus * 128 * 128 * 4, count_bytes = split_count_bytes(c.cus);
    const size_t o_split = m.add(part_bytes + count_bytes);
    void* block = nullptr;
    if (int st = scratch_alloc(&block, m.size, s)) return st;
    m.base = (char*)block;

    auto run = [&]() -> int {
        c.split.part = m.at<float>(o_split);
        c.split.count = (int*)m.at<char>(o_split + part_bytes);
        c.split.budget = c.cus;
        TokArgs k;
        std::memset(&k, 0, sizeof k);
        k.ctl = m.at<TokCtl>(o_ctl);
        k.map = m.at<int>(o_map);
        k.labels = labels;
        k.top = top;
        k.buckets = buckets;
        k.row_weight = row_weight;
        k.part = m.at<float2>(o_part);
        k.slots = slots;
        k.taken = m.at<float>(o_taken);
        k.lse2 = m.at<float>(o_lse);
        const float inv_t = teacher ? 1.f / teacher->temperature : 1.f;
        k.scale2 = scale * inv_t * kLog2E;
        k.tail_stage = 0x7FFFFFFF;
        k.loss = loss;
        k.factor = 1.f;
        if (teacher) {
            k.labels = nullptr;
            k.ids = m.at<int>(o_ids);
            k.probs = m.at<float>(o_probs);
            k.starts = m.at<uint16_t>(o_starts);
            k.plogp = m.at<float>(o_plogp);
            k.factor = teacher->temperature * teacher->temperature;
            with_type(teacher->dtype, [&](auto* tt) {
                using TT = std::remove_pointer_t<decltype(tt)>;
                hipLaunchKernelGGL(teacher_kernel<TT>, row_grid(rows), dim3(256), 0, s, teacher->ids, (const TT*)teacher->logits,
                                   rows, top, vocab, inv_t, buckets, m.at<int>(o_ids), m.at<float>(o_probs),
                                   m.at<uint16_t>(o_starts), m.at<float>(o_plogp), m.at<int>(o_marks));
                return 0;
            });
            if (int st = from_hip(hipGetLastError(), "teacher_kernel launch")) return st;
        }
        RowArgs ra;
        std::memset(&ra, 0, sizeof ra);
        ra.marks = teacher ? m.at<int>(o_marks) : labels;
        ra.row_weight = row_weight;
        ra.rows = rows;
        ra.limit = teacher ? 1 : vocab;
        ra.chunk = rows > kFewRows ? m.at<int>(o_chunk) : nullptr;
        ra.f16 = dtype == PCD_F16;
        ra.ctl = m.at<TokCtl>(o_ctl);
        ra.map = m.at<int>(o_map);
        ra.rank = m.at<int>(o_rank);
        ra.loss = loss;
        ra.dh = RangeArgs{t, (dim + t - 1) / t, plan.dh_k, tile_ends(t), plan.dh_most, c.cus};
        ra.stack = stack;
        ra.clear = (u32x4*)c.split.count;
        ra.clear_units = (int)(count_bytes / 16);
        if (ra.chunk) {
            hipLaunchKernelGGL(count_rows_kernel, dim3((rows + kRowChunk - 1) / kRowChunk), dim3(256), 0, s, ra);
            if (int st = from_hip(hipGetLastError(), "count_rows_kernel launch")) return st;
        }
        const char* W = (const char*)weight;
        const char* last = nullptr;   // where row 0 would lie in front of the last rows' copy
        CopyArgs cp;
        std::memset(&cp, 0, sizeof cp);
        if ((!in_place && !few) || last_copy) {
            cp.src = weight;
            cp.lds = ldw;
            cp.ldd = wld;
            cp.r0 = in_place ? v0 : 0;
            cp.rows = vocab;
            cp.cols = dim;
            cp.out_rows = in_place ? 257 : (int)round_up(vocab, 64) + 1;
            cp.dst = m.at<char>(o_w);
            if (in_place) last = m.at<char>(o_w) - (ptrdiff_t)v0 * wld * ob;
            else W = m.at<char>(o_w);
        }
        if (z_cols) {
            if (coded) {
                k.zq = m.at<uint16_t>(o_z);
                k.ztop = m.at<float>(o_ztop);
            } else {
                k.z = m.at<float>(o_z);
            }
            k.z_cols = z_cols;
        }
        if (few) k.taken = nullptr;   // its logits are there
        const float alpha = scale * (teacher ? teacher->temperature : 1.f);
        const int nt = (size_t)vocab * dim * ob > kTokPieceBytes;
        const FewArgs fa{hidden, ldh, dim, vocab, pitch, plan.few_across, plan.few_step, plan.few_span, weight, ldw, d_hidden ? m.at<float>(o_dh) : nullptr,
                         d_weight, ld_dw, alpha, nt};
        const int row_blocks = (int)((stack ? (size_t)stack : rows_pad) / 4);
        const dim3 grid(row_blocks + (last_copy ? 32 : 0), (pitch + kGatherCols - 1) / kGatherCols);
        with_types(dtype, hidden_dtype, [&](auto* op, auto* src) {
            using OP = std::remove_pointer_t<decltype(op)>;
            using SRC = std::remove_pointer_t<decltype(src)>;
            if constexpr (std::is_same<OP, SRC>::value || std::is_same<SRC, float>::value) {   // the operand type or fp32
                auto launch_few = [&](auto N) {
                    constexpr int NR = decltype(N)::value;
                    hipLaunchKernelGGL((few_rows_kernel<OP, SRC, NR>), dim3(few_blocks), dim3(256), NR * (pitch * ob + 16), s, ra, k,
                                       (const SRC*)hidden, ldh, dim, pitch, (const OP*)weight, ldw, vocab, nt, few_ranges);
                    if (grads) hipLaunchKernelGGL((few_grads_kernel<OP, SRC, NR>), dim3(few_ranges, few_y), dim3(256), 0, s, fa, k);
                };
                if (!few)
                    hipLaunchKernelGGL((gather_rows_kernel<OP, SRC>), grid, dim3(256), 0, s, ra, (const SRC*)hidden, ldh, dim,
                                       m.at<OP>(o_h), pitch, row_blocks, cp);
                else if (few_nr == 1) launch_few(std::integral_constant<int, 1>{});
                else if (few_nr == 2) launch_few(std::integral_constant<int, 2>{});
                else if (few_nr == 4) launch_few(std::integral_constant<int, 4>{});
                else if constexpr (std::is_same<OP, float>::value) launch_few(std::integral_constant<int, kFewTok>{});
            }
            return 0;
        });
        if (int st = from_hip(hipGetLastError(), "gather_rows_kernel launch")) return st;
        if (!in_place && !few) {
            with_type(dtype, [&](auto* op) {
                using OP = std::remove_pointer_t<decltype(op)>;
                hipLaunchKernelGGL(copy_rows_kernel<OP>, dim3(blocks_for((size_t)cp.out_rows * (wld / 8), 256, 8192)), dim3(256),
                                   0, s, cp);
                return 0;
            });
            if (int st = from_hip(hipGetLastError(), "copy_rows_kernel launch")) return st;
        }
        PhaseArgs a;
        std::memset(&a, 0, sizeof a);
        a.alpha = 1.f;

        // a product of the live rows with vocabulary rows [id0, id0 + n) of W
        auto logits = [&](int epi, int t, int id0, int n, void* out, int ldo) {
            Problem p;
            std::memset(&p, 0, sizeof p);
            p.A = m.at(o_h);
            p.lda = pitch;
            p.B = W + (size_t)id0 * wld * ob;
            p.ldb = (int)wld;
            p.M = rows;
            p.N = n;
            p.K = (int)round_up(dim, stage_k(dtype, Tile{t, t}));
            p.dout = out;
            p.ldo = ldo;
            TokArgs kk = k;
            kk.id0 = id0;
            kk.out_n = (int)round_up(n, 64);
            if (last && dim % kFeatPad != 0 && id0 + n == vocab) {
                kk.last_tn = (n - 1) / t;
                kk.b_last = last + (size_t)id0 * wld * ob;
            }
            return logits_product(c, epi, t, p, a, kk);
        };
        if (!few)
            if (int st = logits(EPI_TOK_LSE, plan.t_lse, 0, vocab, nullptr, 0)) return st;
        if (!close && !(few && grads)) {
            hipLaunchKernelGGL(row_loss_kernel, row_grid(rows), dim3(256), 0, s, k, rows);
            if (int st = from_hip(hipGetLastError(), "row_loss_kernel launch")) return st;
        }
        if (!grads) return PCD_SUCCESS;

        for (int id0 = 0; id0 < vocab && !few; id0 += width) {
            const int n = std::min(width, vocab - id0), n64 = (int)round_up(n, 64);
            if (id0 + n64 <= z_cols) {
                TokArgs kk = k;
                kk.id0 = id0;
                const dim3 grid((n64 + kGradCols - 1) / kGradCols, (unsigned)(stack ? stack : rows_pad));
                with_type(dtype, [&](auto* op) {
                    using OP = std::remove_pointer_t<decltype(op)>;
                    hipLaunchKernelGGL(grad_rows_kernel<OP>, grid, dim3(256), 0, s, kk, m.at<OP>(o_g), width, n, n64,
                                       (int)close, stack);
                    return 0;
                });
                if (int st = from_hip(hipGetLastError(), "grad_rows_kernel launch")) return st;
            } else if (int st = logits(EPI_TOK_GRAD, logits_tile(c, rows, n, dim), id0, n, m.at(o_g), width)) {
                return st;
            }
            TokPair pair;
            std::memset(&pair, 0, sizeof pair);
            pair.dh_args = pair.dw_args = a;
            int grid = 0;
            if (d_hidden) {
                Problem& p = pair.dh;
                p.A = m.at(o_g);
                p.lda = width;
                p.B = W + (size_t)id0 * wld * ob;
                p.ldb = (int)wld;
                p.M = dh_rows;
                p.N = in_place ? (int)round_up(dim, unit) : pitch;   // whole loads
                p.K = n64;
                p.m = m.at<float>(o_dh);
                p.ldo = pitch;
                pair.dh_tok = k;
                if (in_place && id0 + n == vocab && (n64 != n || dim % unit != 0)) {
                    // the matrix ends in a broken stage, or in the middle of a load
                    pair.dh_tok.tail_stage = (dim % unit != 0 ? n - 1 : n) / stage_k(dtype, Tile{t, t});
                    pair.dh_tok.tail_delta = last - W;
                }
                pair.dh_args.beta = id0 ? 1.f : 0.f;
                lay_tiles(c, t, p, pair.dh_args, false);
                grid = pair.dh_grid = grid_of(dh_units);
            }
            if (d_weight && !slim) {
                Problem& p = pair.dw;
                p.A = m.at(o_g);
                p.lda = width;
                p.B = m.at(o_h);
                p.ldb = pitch;
                p.M = n64;
                p.N = pitch;
                p.K = (int)rows_pad;
                p.m = (float*)((char*)d_weight + (size_t)id0 * ld_dw * ob);
                p.ldo = (int)ld_dw;
                pair.dw_tok = k;
                pair.dw_tok.out_m = n;
                pair.dw_tok.out_n = dim;
                pair.dw_args.alpha = alpha;
                lay_tiles(c, t, p, pair.dw_args, true);
                grid += grid_of(p.tiles);
            }
            if (grid) {
                const int st = with_type(dtype, [&](auto* op) {
                    return launch_pair_op<std::remove_pointer_t<decltype(op)>>(t, pair, grid, s);
                });
                if (st) return st;
            }
            if (slim) {
                // a workgroup a share of the piece's ids and 512 columns, two a CU
                const int groups = (dim + kSlimCols - 1) / kSlimCols;
                const dim3 shares(std::max(1, std::min(n64 / kSlimIds, (2 * c.cus + groups - 1) / groups)), groups);
                with_type(dtype, [&](auto* op) {
                    using OP = std::remove_pointer_t<decltype(op)>;
                    if constexpr (!std::is_same<OP, float>::value) {
                        auto launch = [&](auto K) {
                            hipLaunchKernelGGL((slim_dw_kernel<OP, decltype(K)::value>), shares, dim3(256), 0, s, k.ctl,
                                               m.at<OP>(o_g), width, m.at<OP>(o_h), pitch, n, n64, dim, alpha,
                                               (OP*)d_weight + (size_t)id0 * ld_dw, ld_dw);
                        };
                        if (rows_pad <= 64) launch(std::integral_constant<int, 1>{});
                        else launch(std::integral_constant<int, 2>{});
                    }
                    return 0;
                });
                if (int st = from_hip(hipGetLastError(), "slim_dw_kernel launch")) return st;
            }
        }
        if (d_hidden) {
            with_type(hidden_dtype, [&](auto* td) {
                using TD = std::remove_pointer_t<decltype(td)>;
                const size_t tasks = (size_t)rows * ((dim + 511) / 512);
                auto launch = [&](auto kernel, unsigned blocks) {
                    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, s, m.at<float>(o_dh), pitch, m.at<TokCtl>(o_ctl),
                                       m.at<int>(o_rank), rows, dim, alpha, (TD*)d_hidden, ld_dh, stack);
                };
                if (tasks <= (size_t)c.cus) launch(scatter_rows_kernel<TD, 32>, (unsigned)((size_t)rows * ((dim + 63) / 64)));
                else launch(scatter_rows_kernel<TD, 1>, blocks_for(tasks, 4, 1 << 20));
                return 0;
            });
            if (int st = from_hip(hipGetLastError(), "scatter_rows_kernel launch")) return st;
        }
        return PCD_SUCCESS;
    };
    const int st = run();
    const int st2 = scratch_free(block, s);
    return st ? st : st2;
}

// Most logits of a call: 2^27 tiles of 64 x 64, which the deal of tiles over the XCDs counts in eighths of an int.
constexpr long long kMostLogits = 1ll << 39;

// The checks both losses make.
int check_loss(const char* name, int dtype, const void* hidden, int hidden_dtype, long long* ldh, const void* weight,
               long long* ldw, int rows, int dim, int vocab, float scale, float temperature, const float* loss, long long* ld_dh,
               long long* ld_dw) {
    if (!types_fit(dtype, hidden_dtype) || (dtype == PCD_F32 && hidden_dtype != PCD_F32))
        return fail(PCD_INVALID_VALUE, "%s: types %d and %d (hidden states have the weight's type or are fp32)", name, dtype,
                    hidden_dtype);
    if (!weight || (rows > 0 && (!hidden || !loss))) return fail(PCD_INVALID_VALUE, "%s: null pointer", name);
    if (rows < 0 || dim < 1 || vocab < 1 || rows > (1 << 24) || dim > (1 << 20) || vocab > (1 << 24))
        return fail(PCD_INVALID_VALUE, "%s: bad shape: %d rows, dimension %d, vocabulary %d", name, rows, dim, vocab);
    if ((long long)rows * vocab > kMostLogits)
        return fail(PCD_INVALID_VALUE, "%s: %d rows of a vocabulary of %d are more than 2^39 logits", name, rows, vocab);
    for (long long* ld : {ldh, ldw, ld_dh, ld_dw}) {
        if (*ld == 0) *ld = dim;
        if (*ld < dim || *ld > (1 << 30))
            return fail(PCD_INVALID_VALUE, "%s: rows of %d elements are %lld apart", name, dim, *ld);
    }
    // the factors of the logits in base 2, of their gradients and of the losses
    if (!std::isfinite(scale * (1.f / temperature) * kLog2E) || !std::isfinite(scale * temperature))
        return fail(PCD_INVALID_VALUE, "%s: a scale of %g at a temperature of %g is not finite in fp32", name, scale, temperature);
    if (!std::isnormal(temperature * temperature))
        return fail(PCD_INVALID_VALUE, "%s: the square of a temperature of %g is not a normal fp32 number", name, temperature);
    return PCD_SUCCESS;
}

// Most elements of an embedding's row: units and a wave's columns past its end are still an int.
constexpr int kMostDim = 1 << 30;

}  // namespace

int pcd_token_xent(int dtype, const void* hidden, int hidden_dtype, long long ld_hidden, const void* weight,
                   long long ld_weight, const int* labels, const float* row_weight, int rows, int dim, int vocab, float scale,
                   float* loss, void* d_hidden, long long ld_dhidden, void* d_weight, long long ld_dweight, void* stream) {
    if (int st = check_loss("pcd_token_xent", dtype, hidden, hidden_dtype, &ld_hidden, weight, &ld_weight, rows, dim, vocab,
                            scale, 1.f, loss, &ld_dhidden, &ld_dweight))
        return st;
    if (rows > 0 && !labels) return fail(PCD_INVALID_VALUE, "pcd_token_xent: null labels");
    return guarded("pcd_token_xent", [&] {
        return token_loss(dtype, hidden, hidden_dtype, ld_hidden, weight, ld_weight, labels, nullptr, row_weight, rows, dim,
                          vocab, scale, loss, d_hidden, ld_dhidden, d_weight, ld_dweight, (hipStream_t)stream);
    });
}

int pcd_token_distill(int dtype, const void* hidden, int hidden_dtype, long long ld_hidden, const void* weight,
                      long long ld_weight, const int* teacher_ids, const void* teacher_logits, int teacher_dtype, int top,
                      const float* row_weight, int rows, int dim, int vocab, float scale, float temperature, float* loss,
                      void* d_hidden, long long ld_dhidden, void* d_weight, long long ld_dweight, void* stream) {
    if (!std::isfinite(temperature) || !(temperature > 0.f) || !std::isfinite(1.f / temperature))
        return fail(PCD_INVALID_VALUE, "pcd_token_distill: the temperature is not a positive number with a finite inverse");
    if (int st = check_loss("pcd_token_distill", dtype, hidden, hidden_dtype, &ld_hidden, weight, &ld_weight, rows, dim,
                            vocab, scale, temperature, loss, &ld_dhidden, &ld_dweight))
        return st;
    if (rows > 0 && (!teacher_ids || !teacher_logits)) return fail(PCD_INVALID_VALUE, "pcd_token_distill: null teacher");
    if (!known_type(teacher_dtype)) return fail(PCD_INVALID_VALUE, "pcd_token_distill: unknown teacher type %d", teacher_dtype);
    if (top < 1 || top > kMaxTop)
        return fail(PCD_INVALID_VALUE, "pcd_token_distill: %d slots a row (1 to %d)", top, kMaxTop);
    const Teacher t{teacher_ids, teacher_logits, teacher_dtype, top, temperature};
    return guarded("pcd_token_distill", [&] {
        return token_loss(dtype, hidden, hidden_dtype, ld_hidden, weight, ld_weight, nullptr, &t, row_weight, rows, dim,
                          vocab, scale, loss, d_hidden, ld_dhidden, d_weight, ld_dweight, (hipStream_t)stream);
    });
}

int pcd_token_keep_logits(size_t bytes) {
    g_keep_logits.store(bytes, std::memory_order_relaxed);
    return PCD_SUCCESS;
}

int pcd_token_embed(int dtype, const void* table, long long ld_table, const int* tokens, int count, int vocab, int dim,
                    float scale, void* out, int out_dtype, long long ld_out, void* stream) {
    if (!types_fit(dtype, out_dtype))
        return fail(PCD_INVALID_VALUE, "pcd_token_embed: types %d and %d", dtype, out_dtype);
    if (count < 0 || vocab < 1 || dim < 1 || dim > kMostDim)
        return fail(PCD_INVALID_VALUE, "pcd_token_embed: bad shape: %d tokens, vocabulary %d, dimension %d", count, vocab, dim);
    if (!table || (count > 0 && (!tokens || !out))) return fail(PCD_INVALID_VALUE, "pcd_token_embed: null pointer");
    if (ld_table == 0) ld_table = dim;
    if (ld_out == 0) ld_out = dim;
    if (ld_table < dim || ld_out < dim)
        return fail(PCD_INVALID_VALUE, "pcd_token_embed: rows of %d elements are %lld and %lld apart", dim, ld_table, ld_out);
    if (count == 0) return PCD_SUCCESS;
    return with_types(dtype, out_dtype, [&](auto* ti, auto* to) {
        using TI = std::remove_pointer_t<decltype(ti)>;
        using TO = std::remove_pointer_t<decltype(to)>;
        const size_t units = (size_t)count * ((dim + embed_unit<TI, TO>() - 1) / embed_unit<TI, TO>());
        hipLaunchKernelGGL((embed_kernel<TI, TO>), dim3(blocks_for(units, 1024, 1 << 20)), dim3(256), 0, (hipStream_t)stream,
                           (const TI*)table, ld_table, tokens, count, vocab, dim, scale, (TO*)out, ld_out);
        return from_hip(hipGetLastError(), "embed_kernel launch");
    });
}

int pcd_token_embed_grad(int dtype, void* d_table, long long ld_table, const int* tokens, int count, int vocab, int dim,
                         float scale, int accumulate, const void* d_out, int out_dtype, long long ld_out, void* stream) {
    hipStream_t s = (hipStream_t)stream;
    if (!types_fit(dtype, out_dtype))
        return fail(PCD_INVALID_VALUE, "pcd_token_embed_grad: types %d and %d", dtype, out_dtype);
    if (count < 0 || count > (1 << 28) || vocab < 1 || vocab > (1 << 30) || dim < 1 || dim > kMostDim)
        return fail(PCD_INVALID_VALUE, "pcd_token_embed_grad: bad shape: %d tokens, vocabulary %d, dimension %d", count, vocab,
                    dim);
    if (!d_table || (count > 0 && (!tokens || !d_out))) return fail(PCD_INVALID_VALUE, "pcd_token_embed_grad: null pointer");
    if (ld_table == 0) ld_table = dim;
    if (ld_out == 0) ld_out = dim;
    if (ld_table < dim || ld_out < dim)
        return fail(PCD_INVALID_VALUE, "pcd_token_embed_grad: rows of %d elements are %lld and %lld apart", dim, ld_table,
                    ld_out);
    if (count == 0 && accumulate) return PCD_SUCCESS;
    return guarded("pcd_token_embed_grad", [&]() -> int {
        int cus = 0;
        if (int st = device_cus(&cus)) return st;
        const size_t shares = std::max<size_t>(1, clear_shares(op_bytes(dtype), vocab, dim));
        auto clear = [&]() {
            return with_type(dtype, [&](auto* to) {
                using TO = std::remove_pointer_t<decltype(to)>;
                hipLaunchKernelGGL(clear_kernel<TO>, dim3((unsigned)std::min<size_t>(shares, 1 << 20)), dim3(1024), 0, s, (TO*)d_table,
                                   ld_table, vocab, dim);
                return from_hip(hipGetLastError(), "clear_kernel launch");
            });
        };
        if (count == 0) return clear();
        const int tiles = (count + kSortTile - 1) / kSortTile;
        const int window = count <= kFewTokens ? kWindowFew : kWindow;
        const int windows = count > window ? (count + window - 1) / window : 0;   // none: no long tokens
        const bool small = count <= kSortSmall && vocab < 1 << (32 - kSortPosBits);
        const int pitch = (int)round_up(dim, 8);
        Arena m;
        size_t o_key[2], o_pos[2];
        for (int i = 0; i < (small ? 1 : 2); ++i) {
            o_key[i] = m.add((size_t)count * 4);
            o_pos[i] = m.add((size_t)count * 4);
        }
        const size_t o_counts = small ? 0 : m.add((size_t)tiles * 256 * 4), o_totals = small ? 0 : m.add(256 * 4);
        const size_t o_parts = windows ? m.add((size_t)2 * windows * pitch * 4) : 0;
        void* block = nullptr;
        if (int st = scratch_alloc(&block, m.size, s)) return st;
        m.base = (char*)block;
        auto run = [&]() -> int {
            const int *keys = nullptr, *pos = nullptr;
            if (small) {
                int width = 1, low = 0;   // bits of a key: the classes', and the rest dealt evenly over the passes
                while (vocab >> width) ++width;
                while (low < width - 1 && (2 << low) <= std::min(kSortClasses, count / 64)) ++low;
                const int rest = width - low, passes = (rest + kSortDigit - 1) / kSortDigit, bits = (rest + passes - 1) / passes;
                const unsigned others = accumulate ? 0 : (unsigned)std::min<size_t>(shares, 1 << 20);
                with_type(dtype, [&](auto* to) {
                    using TO = std::remove_pointer_t<decltype(to)>;
                    hipLaunchKernelGGL(sort_small_kernel<TO>, dim3((1u << low) + others), dim3(1024), 0, s, tokens, count, vocab, low, passes, bits,
                                       m.at<int>(o_key[0]), m.at<int>(o_pos[0]), (TO*)d_table, ld_table, dim);
                    return 0;
                });
                keys = m.at<int>(o_key[0]);
                pos = m.at<int>(o_pos[0]);
            } else {
                if (!accumulate)
                    if (int st = clear()) return st;
                keys = tokens;
                for (int shift = 0, to = 0; shift == 0 || (shift < 32 && vocab >> shift); shift += 8, to ^= 1) {
                    hipLaunchKernelGGL(sort_count_kernel, dim3(tiles), dim3(256), 0, s, keys, count, vocab, shift,
                                       m.at<int>(o_counts), tiles);
                    hipLaunchKernelGGL(sort_scan_kernel, dim3(256), dim3(256), 0, s, m.at<int>(o_counts), tiles,
                                       m.at<int>(o_totals));
                    hipLaunchKernelGGL(sort_move_kernel, dim3(tiles), dim3(256), 0, s, keys, pos, count, vocab, shift,
                                       m.at<int>(o_counts), tiles, m.at<int>(o_totals), m.at<int>(o_key[to]),
                                       m.at<int>(o_pos[to]));
                    keys = m.at<int>(o_key[to]);
                    pos = m.at<int>(o_pos[to]);
                }
            }
            if (int st = from_hip(hipGetLastError(), "the token sort's launches")) return st;
            return with_types(out_dtype, dtype, [&](auto* ti, auto* to_) {
                using TI = std::remove_pointer_t<decltype(ti)>;
                using TO = std::remove_pointer_t<decltype(to_)>;
                constexpr int N = embed_unit<TI, TO>();
                const size_t chunks = (dim + 64 * N - 1) / (64 * N);
                const int places = (size_t)count * chunks > 256 * (size_t)cus ? kEmbedPlaces : 1;
                const size_t tasks = ((size_t)windows + (count + places - 1) / places) * chunks;
                hipLaunchKernelGGL((embed_grad_kernel<TI, TO>), dim3(blocks_for(tasks, 4, 1 << 20)), dim3(256), 0, s,
                                   (const TI*)d_out, ld_out, keys, pos, count, vocab, dim, scale, accumulate,
                                   m.at<float>(o_parts), pitch, (TO*)d_table, ld_table, places, windows, window);
                if (windows)
                    hipLaunchKernelGGL((embed_long_kernel<TO, N>), dim3(blocks_for(windows * chunks, 4, 1 << 20)), dim3(256), 0,
                                       s, keys, count, vocab, dim, scale, accumulate, m.at<float>(o_parts), pitch,
                                       (TO*)d_table, ld_table, windows, window);
                return from_hip(hipGetLastError(), "embed_grad_kernel launch");
            });
        };
        const int st = run();
        const int st2 = scratch_free(block, s);
        return st ? st : st2;
    });
}
