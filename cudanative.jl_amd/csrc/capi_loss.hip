// C ABI of the loss over a large vocabulary (declared in include/miwmma.h): checks of the arguments, the layout of the
// workspace and the sequence of launches.  Nothing here allocates or throws.
#include "api_checks.hpp"
#include "loss.hpp"

#include <algorithm>

namespace {

constexpr int64_t LEAST_PIECE = 8192, PIECE_ELEMENTS = 1 << 27;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t up_to(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

}  // namespace

namespace miw {

// By itself pieces of one size, of at most 2^27 probabilities (256 MiB), which the last-level cache partly holds for the two products that read them, or of 8192 columns
// where that is more, since the rows' gradients are read and written in Float32 once a piece.
int64_t loss_piece(int64_t tokens, int64_t vocabulary, int64_t piece)
{
    if (piece == 0) {
        piece = std::max(LEAST_PIECE, PIECE_ELEMENTS / std::max<int64_t>(tokens, 1) / 64 * 64);
        piece = ceil_div(vocabulary, ceil_div(vocabulary, piece));
    }
    return std::min(up_to(piece, 64), up_to(vocabulary, 64));
}

}  // namespace miw

namespace {

using miw::loss_params;

using miw::LOSS_SLICED, miw::LOSS_SLICES;

int check_sizes(const char *what, int64_t tokens, int64_t vocabulary, int64_t width)
{
    CHECK(check_extent(what, "tokens", tokens, 0, 1 << 26));
    CHECK(check_extent(what, "vocabulary", vocabulary, 1, EXTENT));
    return check_extent(what, "width", width, 1, EXTENT);
}

// The workspace, piece by piece; each starts on 256 bytes.
struct layout {
    char *base;
    size_t used = 0;
    template <class T>
    T *take(int64_t count)
    {
        T *at = (T *)(base + used);
        used += (size_t)up_to(count * (int64_t)sizeof(T), 256);
        return at;
    }
};
struct scores_space {
    float *goals, *stats;
};
scores_space take_scores(layout &l, int64_t tokens, int64_t vocabulary)
{
    scores_space s{};
    s.goals = l.take<float>(2 * tokens);
    s.stats = l.take<float>(2 * miw::loss_stats(tokens, vocabulary));
    return s;
}
struct gradient_space {
    miw::loss_rows rows;
    float *partial;
    char *copy, *probabilities;
};
gradient_space take_gradient(layout &l, int64_t tokens, int64_t vocabulary, int64_t width, int64_t piece)
{
    gradient_space s{};
    s.rows.place = l.take<int>(tokens);
    s.rows.list = l.take<int>(tokens);
    s.rows.goal = l.take<int>(tokens);
    s.rows.offsets = l.take<int>(2);
    s.rows.lse = l.take<float>(tokens);
    s.rows.share = l.take<float>(tokens);
    s.rows.scale = l.take<float>(2);
    s.rows.slice_offsets = l.take<int>(LOSS_SLICES + 1);
    s.rows.slice_rows = l.take<int>(std::min(LOSS_SLICES * tokens, LOSS_SLICED));
    s.partial = l.take<float>(std::max(tokens * width, std::min(LOSS_SLICES * tokens * width, LOSS_SLICED)));
    s.copy = l.take<char>(2 * tokens * width);
    const int64_t whole = tokens * up_to(vocabulary, 64);
    s.probabilities = l.take<char>(2 * std::min(whole, piece ? tokens * miw::loss_piece(tokens, vocabulary, piece) : std::max(LEAST_PIECE * tokens, PIECE_ELEMENTS)));
    return s;
}

size_t workspace_bytes_of(int64_t tokens, int64_t vocabulary, int64_t width, bool grad, int64_t piece)
{
    if (tokens == 0) return 0;
    layout scores{nullptr}, gradient{nullptr};
    take_scores(scores, tokens, vocabulary);
    if (grad) take_gradient(gradient, tokens, vocabulary, width, piece);
    return std::max(scores.used, gradient.used);  // (a gradient's workspace does for the scores before it)
}
int check_workspace(const char *what, int64_t tokens, int64_t vocabulary, int64_t width, bool grad, int64_t piece, const void *workspace, size_t bytes)
{
    const size_t need = workspace_bytes_of(tokens, vocabulary, width, grad, piece);
    CHECK(check_element(what, "workspace", workspace, 16));
    if (bytes < need) return api_fail(MIW_ERR_INVALID_VALUE, "%s: the workspace has %zu bytes, %zu are needed", what, bytes, need);
    return 0;
}

// Scores: hidden rows by the vocabulary's vectors from `first` on.  Rows are all tokens, whose targets goal has, until the caller says otherwise.
loss_params score_product(const int *goal, int64_t tokens, int64_t first, int64_t columns, int64_t width, int64_t ldx, int64_t ldw, const void *X, const void *W)
{
    loss_params p{};
    p.X = (const char *)W + 2 * first * ldw;
    p.Y = (const char *)X;
    p.groups = 1;
    p.rows = p.source_rows = (int)tokens;
    p.I = (int)columns;
    p.K = (int)width;
    p.ldx = 2 * ldw;
    p.ldy = 2 * ldx;
    p.x_k_major = 1;
    p.vector = aligned(X, 16) && aligned(W, 16) && ldx % 8 == 0 && ldw % 8 == 0 && width % 8 == 0;
    p.goal = goal;
    p.first = first;
    return p;
}

}  // namespace

extern "C" {

int miw_cross_entropy_workspace(int64_t tokens, int64_t vocabulary, int64_t width, int grad, int64_t piece, size_t *bytes)
{
    const char *what = "cross_entropy_workspace";
    if (!bytes) return api_fail(MIW_ERR_NULL_POINTER, "%s: null output pointer", what);
    CHECK(check_sizes(what, tokens, vocabulary, width));
    CHECK(check_extent(what, "piece", piece, 0, EXTENT));
    *bytes = workspace_bytes_of(tokens, vocabulary, width, grad != 0, piece);
    return 0;
}

int miw_cross_entropy(int dtype, int64_t tokens, int64_t vocabulary, int64_t width, int64_t ldx, int64_t ldw, const void *X, const void *W, const int *targets,
                      float *losses, float *lse, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *what = "cross_entropy";
    if (!half_type(dtype)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: unknown element type %d", what, dtype);
    CHECK(check_sizes(what, tokens, vocabulary, width));
    CHECK(check_pitch(what, "ldx", &ldx, width));
    CHECK(check_pitch(what, "ldw", &ldw, width));
    if (!tokens) return 0;
    CHECK(check_element(what, "X", X, 2));
    CHECK(check_element(what, "W", W, 2));
    CHECK(check_element(what, "targets", targets, 4));
    CHECK(check_element(what, "losses", losses, 4));
    CHECK(check_element(what, "lse", lse, 4));
    CHECK(check_workspace(what, tokens, vocabulary, width, false, 0, workspace, workspace_bytes));
    REQUIRE_INIT(what);
    hipStream_t s = (hipStream_t)stream;
    const int cus = miw::api_cu_count();
    layout l{(char *)workspace};
    const scores_space at = take_scores(l, tokens, vocabulary);
    // Every token has scores, whatever its target: lse is theirs.  All in one go, unless their statistics have no room; then the last run has tokens of the one before
    // again, since its kernel, and so its slices, go by the number of tokens.
    const int64_t run = miw::loss_run(score_product(targets, tokens, 0, vocabulary, width, ldx, ldw, X, W), cus);
    for (int64_t done = 0; done < tokens; done += run) {
        const int64_t first = std::min(done, tokens - run);
        loss_params p = score_product(targets + first, run, 0, vocabulary, width, ldx, ldw, (const char *)X + 2 * first * ldx, W);
        const miw::loss_slices slices = miw::loss_score_slices(p, cus);
        p.stats = at.stats;
        p.goals = at.goals;
        p.stat_rows = run;
        HIP_TRY(miw::launch_loss_scores(p, dtype, cus, s));
        HIP_TRY(miw::launch_loss_join({targets + first, at.stats, at.goals, losses + first, lse + first, (int)run, slices.count, slices.width, (long)run, (long)vocabulary}, s));
    }
    return 0;
}

int miw_cross_entropy_grad(int dtype, int dw_type, int accumulate, int64_t tokens, int64_t vocabulary, int64_t width, int64_t ldx, int64_t ldw, int64_t lddx,
                           int64_t lddw, int64_t piece, const void *X, const void *W, const int *targets, const float *lse, const float *dlosses, void *dX,
                           void *dW, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *what = "cross_entropy_grad";
    if (!half_type(dtype) || (dw_type != dtype && dw_type != MIW_F32)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: element types %d and %d", what, dtype, dw_type);
    CHECK(check_sizes(what, tokens, vocabulary, width));
    CHECK(check_pitch(what, "ldx", &ldx, width));
    CHECK(check_pitch(what, "ldw", &ldw, width));
    CHECK(check_pitch(what, "lddx", &lddx, width));
    CHECK(check_pitch(what, "lddw", &lddw, width));
    CHECK(check_extent(what, "piece", piece, 0, EXTENT));
    if (dW) CHECK(check_element(what, "dW", dW, type_size(dw_type)));
    if (tokens) {
        CHECK(check_element(what, "X", X, 2));
        CHECK(check_element(what, "W", W, 2));
        CHECK(check_element(what, "targets", targets, 4));
        CHECK(check_element(what, "lse", lse, 4));
        CHECK(check_element(what, "dlosses", dlosses, 4));
        if (dX) CHECK(check_element(what, "dX", dX, 2));
        CHECK(check_workspace(what, tokens, vocabulary, width, true, piece, workspace, workspace_bytes));
    }
    if ((!dX && !dW) || (!tokens && !dW)) return 0;
    REQUIRE_INIT(what);
    hipStream_t s = (hipStream_t)stream;
    const int cus = miw::api_cu_count();
    auto vectors_gradient = [&](loss_params p) { return dtype == MIW_F16 ? miw::launch_loss_vectors_gradient_f16(p, dw_type, cus, s) : miw::launch_loss_vectors_gradient_bf16(p, dw_type, cus, s); };
    if (!tokens) {  // dW is a sum of nothing
        if (accumulate) return 0;
        loss_params p{};
        p.groups = 1;
        p.I = (int)width;
        p.J = p.store_j = (int)vocabulary;
        p.D = dW;
        p.ldd = lddw;
        HIP_TRY(vectors_gradient(p));
        return 0;
    }
    layout l{(char *)workspace};
    const gradient_space at = take_gradient(l, tokens, vocabulary, width, piece);
    const int64_t columns = miw::loss_piece(tokens, vocabulary, piece), longest = std::min(columns, vocabulary);
    const miw::loss_cut cut = dX ? miw::cut_loss_rows(tokens, width, longest, cus) : miw::loss_cut{1, 0};
    const int64_t slice = up_to(ceil_div(longest, cut.slices), 64), slices = ceil_div(longest, slice);
    HIP_TRY(miw::launch_loss_look({at.rows, targets, lse, dlosses, (int)tokens, (int)slices, dtype == MIW_F16, (long)vocabulary}, s));
    const float *unscale = dtype == MIW_F16 ? at.rows.scale + 1 : nullptr;
    loss_params sum{};  // of the vectors' gradient, but for the piece
    sum.X = (const char *)X;
    sum.Y = at.probabilities;
    sum.offsets = at.rows.offsets;
    sum.gather = at.rows.list;
    sum.groups = 1;
    sum.rows = sum.source_rows = (int)tokens;
    sum.I = (int)width;
    sum.ldx = 2 * ldx;
    sum.ldy = 2 * columns;
    sum.ldd = lddw;
    sum.accumulate = accumulate != 0;
    sum.unscale = unscale;
    sum.vector = score_product(at.rows.goal, tokens, 0, vocabulary, width, ldx, ldw, X, W).vector;
    sum.d_vector = stores_vectors(dW, lddw, 0, type_size(dw_type), false);
    auto sum_of = [&](int64_t first, int64_t n) {
        loss_params q = sum;
        q.J = (int)up_to(n, 8);  // (rows of the workspace are that long)
        q.store_j = (int)n;
        q.D = (char *)dW + type_size(dw_type) * first * lddw;
        return q;
    };
    if (dW && miw::loss_sum_is_dense(sum_of(0, longest), cus)) {
        HIP_TRY(miw::launch_loss_copy({X, at.copy, at.rows.list, at.rows.offsets, (int)tokens, (long)width / 8, (long)ldx / 8}, s));
        sum.X = at.copy;
        sum.ldx = 2 * width;
        sum.gather = nullptr;
        sum.dense = 1;
    }
    for (int64_t first = 0; first < vocabulary; first += columns) {
        const int64_t n = std::min(columns, vocabulary - first);
        loss_params p = score_product(at.rows.goal, tokens, first, n, width, ldx, ldw, X, W);
        p.offsets = at.rows.offsets;
        p.gather = at.rows.list;
        p.lse = at.rows.lse;
        p.share = at.rows.share;
        p.D = at.probabilities;
        p.ldd = columns;
        HIP_TRY(miw::launch_loss_probabilities(p, dtype, cus, s));
        const bool vector = p.vector;
        if (dX) {
            loss_params q{};
            q.X = (const char *)W + 2 * first * ldw;
            q.Y = at.probabilities;
            q.groups = (int)ceil_div(n, slice);  // (the last piece may have fewer)
            q.offsets = slices > 1 ? at.rows.slice_offsets : at.rows.offsets;
            q.gather = slices > 1 ? at.rows.slice_rows : nullptr;
            q.rows = (int)(tokens * q.groups);
            q.source_rows = (int)tokens;
            q.I = (int)width;
            q.K = (int)n;
            q.slice = (int)slice;
            q.tile = cut.tile;
            q.ldx = 2 * ldw;
            q.ldy = 2 * columns;
            q.sx = 2 * slice * ldw;
            q.D = at.partial;
            q.ldd = width;
            q.accumulate = first > 0;
            q.vector = vector;
            q.d_vector = width % 4 == 0;
            HIP_TRY((dtype == MIW_F16 ? miw::launch_loss_rows_gradient_f16 : miw::launch_loss_rows_gradient_bf16)(q, cus, s));
        }
        if (dW) HIP_TRY(vectors_gradient(sum_of(first, n)));
    }
    if (dX)
        HIP_TRY(miw::launch_loss_dx({at.rows.place, at.rows.offsets, at.partial, unscale, dX, (int)tokens, (int)slices, (long)width, (long)lddx,
                                     aligned(dX, 16) && lddx % 8 == 0 && width % 8 == 0},
                                    dtype, s));
    return 0;
}

}  // extern "C"
