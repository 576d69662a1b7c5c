// Host-only check of the token losses' plans: over shapes and limits of kept
// logits, every piece of the vocabulary takes its gradient by the logits from a
// kernel that writes all of its rows, and what is kept stays within the limit.
// Nothing here touches a GPU.
//   token_check SEED COUNT                  random shapes, limits drawn towards the ends of what a plan decides by
//   token_check DTYPE ROWS DIM VOCAB KEEP   one plan, both gradients
#include "../../predicitivecoding_amd/csrc/pcdevice.hip"

#include <cstdio>
#include <cstdlib>
#include <random>

static int check(int dtype, int rows, int dim, int vocab, long long ldw, bool d_hidden, bool d_weight, size_t keep, bool verbose,
                 int* stacked) {
    const TokCall c{dtype, 256, nullptr, {}};
    const LossPlan p = plan_loss(c, (const void*)4096, ldw, rows, dim, vocab, 1, d_hidden, d_weight, keep);
    *stacked += p.stack != 0;
    const char* what = nullptr;
    if (!p.few) {
        const size_t kept = p.rows_pad * p.z_cols * (p.coded ? 17 : 32) / 8;
        if (kept > keep) what = "more kept than the limit";
        if (p.z_cols % 64 != 0 || p.z_cols > (int)round_up(vocab, 64)) what = "kept columns";
        if (p.stack && p.z_cols < vocab) what = "two parts without every logit";
        const size_t padded = p.stack ? 2 * p.stack : round_up(rows, 64);
        for (int id0 = 0; p.grads && id0 < vocab; id0 += p.width) {
            const int n = std::min(p.width, vocab - id0), n64 = (int)round_up(n, 64);
            if (id0 + n64 <= p.z_cols) continue;   // grad_rows_kernel
            // the second product: its tiles are laid over `rows`
            const int t = logits_tile(c, rows, n, dim);
            if ((size_t)tile_count(rows, t, t) * t < padded) what = "a second product of fewer rows than G has";
        }
    }
    if (what || verbose)
        std::printf("%s: dtype %d rows %d dim %d vocab %d keep %zu: stack %d kept %d of %d: %s\n", what ? "BAD" : "ok", dtype, rows,
                    dim, vocab, keep, p.stack, p.z_cols, vocab, what ? what : "");
    return what != nullptr;
}

int main(int argc, char** argv) {
    int bad = 0, stacked = 0;
    if (argc > 3) {
        const int dim = std::atoi(argv[3]);
        bad = check(std::atoi(argv[1]), std::atoi(argv[2]), dim, std::atoi(argv[4]), dim, true, true, std::strtoull(argv[5], nullptr, 10),
                    true, &stacked);
        return bad;
    }
    std::mt19937 rng((unsigned)std::atoi(argv[1]));
    auto uniform = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    auto log_uniform = [&](double lo, double hi) {
        return (int)std::exp(std::uniform_real_distribution<double>(std::log(lo), std::log(hi))(rng));
    };
    const int count = std::atoi(argv[2]);
    for (int i = 0; i < count; ++i) {
        const int dtype = uniform(0, 2), rows = uniform(0, 1) ? uniform(1, 70) : log_uniform(1, 1 << 20);
        const int dim = log_uniform(1, 8192), vocab = log_uniform(1, 1 << 21), grads = uniform(0, 3);
        // a limit about one that the plan's decisions turn on: the logits of some rows, whole or as codes, over whole 64s or 256s
        const size_t at = (size_t)(uniform(0, 1) ? round_up(rows, 64) : uniform(0, 1) ? round_up(rows, 32) : rows) *
                          round_up(vocab, uniform(0, 1) ? 64 : 256);
        const size_t limits[] = {0, at * 4, at * 8, at * 17 / 8, (size_t)log_uniform(1, 1e9), (size_t)1 << 30};
        const size_t keep = limits[uniform(0, 5)];
        for (int d = -1; d <= 1; ++d)
            bad += check(dtype, rows, dim, vocab, dim + (uniform(0, 3) ? 0 : uniform(1, 64)), grads & 1, grads & 2,
                         d < 0 && keep == 0 ? 0 : keep + d, false, &stacked);
    }
    std::printf("%d plans, %d with gradients in two parts, %d bad\n", 3 * count, stacked, bad);
    return bad ? 1 : 0;
}
