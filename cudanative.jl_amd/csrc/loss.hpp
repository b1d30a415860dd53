// Declarations of the loss over a large vocabulary and its C ABI layer.
#pragma once
#include "experts.hpp"

namespace miw {

// A product whose ends the loss has of its own (loss_ends.hpp).  Rows are all tokens in the scores, and those that count, in their order, in the gradient: row r is
// token list[r].
struct loss_params : grouped_params {
    const int *goal;        // target of each row
    float *stats;           // scores: largest score and sum of exponentials of each slice of columns and row, two values together
    float *goals;           // scores: of each row the target's, and its slice's sum without it
    long stat_rows;         // rows that a slice of stats has room for
    const float *lse;       // probabilities: of each row
    const float *share;     // probabilities: of each row, times the power of two that keeps Float16 in range
    const float *unscale;   // gradient to the vocabulary's vectors: that power's inverse, or null
    long first;             // first column's place in the vocabulary
    int slice, tile;        // gradient to the rows: columns of a group's sum; the kernel's tile
    int store_j;            // gradient to the vocabulary's vectors: rows of D
    int dense;              // gradient to the vocabulary's vectors: X's rows lie in their order
};

// What the gradient knows of the tokens once they have been looked at.  All arrays are in the workspace.
struct loss_rows {
    int *place;            // of each token: its row, or -1
    int *list, *goal;      // of each row: its token and target
    int *offsets;          // 0 and the number of rows
    float *lse, *share;    // of each row
    float *scale;          // the power of two that shares are multiplied by, and its inverse
    int *slice_offsets, *slice_rows;  // groups of the same rows, one for each slice of a sum
};
struct loss_look_params {
    loss_rows rows;
    const int *targets;
    const float *lse, *shares;
    int tokens, slices, scaled;
    long vocabulary;
};
hipError_t launch_loss_look(const loss_look_params &p, hipStream_t s);

// The rows that count, one behind the other (16-byte pieces; rows of X and of the copy are whole numbers of them).
struct loss_copy_params {
    const void *X;
    void *copy;
    const int *list, *offsets;
    int tokens;
    long pieces, ldx;  // of a row; from row to row of X
};
hipError_t launch_loss_copy(const loss_copy_params &p, hipStream_t s);

// Losses from the slices' statistics.
struct loss_join_params {
    const int *targets;
    const float *stats, *goals;
    float *losses, *lse;
    int tokens, slices, slice;  // columns of a slice
    long stat_rows, vocabulary;
};
hipError_t launch_loss_join(const loss_join_params &p, hipStream_t s);

// The rows' gradients: partial sums of all slices joined, at the tokens' places.
struct loss_dx_params {
    const int *place, *offsets;
    const float *partial, *unscale;
    void *dX;
    int tokens, slices;
    long width, lddx;
    int vector;
};
hipError_t launch_loss_dx(const loss_dx_params &p, int dtype, hipStream_t s);

// Columns of the vocabulary (a multiple of 64) that the gradient has probabilities of at a time, where the caller asks for `piece` or leaves it (0).
int64_t loss_piece(int64_t tokens, int64_t vocabulary, int64_t piece);

// Products.  The kernel that makes scores; columns of a slice of the statistics; slices there are.
struct loss_slices {
    int width, count;
};
// Slices of a piece of the vocabulary that the gradient to the rows is summed in, each in Float32 in the workspace, and the tile (grouped_tile_size) of its product.
constexpr int64_t LOSS_SLICES = 32, LOSS_SLICED = 1 << 24;  // the most of them, and of values in more than one
struct loss_cut {
    int slices, tile;
};
loss_cut cut_loss_rows(long tokens, long width, long columns, int cus);
grouped_choice choose_loss_rows(const grouped_params &p, int cus);
loss_slices loss_score_slices(const grouped_params &p, int cus);
// Statistics (slices times tokens) that the workspace has room for, and the tokens that scores are made of at a time, all in that room, of p.rows.
constexpr int64_t LOSS_STATS = 1 << 24, LOSS_RUN = 256;
long loss_stats(long tokens, long vocabulary);
long loss_run(grouped_params p, int cus);
bool loss_sum_is_dense(const grouped_params &p, int cus);  // the vectors' gradient, of the first and longest piece
hipError_t launch_loss_scores(const loss_params &p, int dtype, int cus, hipStream_t s);
hipError_t launch_loss_probabilities(const loss_params &p, int dtype, int cus, hipStream_t s);
hipError_t launch_loss_rows_gradient_f16(const loss_params &p, int cus, hipStream_t s);
hipError_t launch_loss_rows_gradient_bf16(const loss_params &p, int cus, hipStream_t s);
hipError_t launch_loss_vectors_gradient_f16(const loss_params &p, int d_type, int cus, hipStream_t s);
hipError_t launch_loss_vectors_gradient_bf16(const loss_params &p, int d_type, int cus, hipStream_t s);

}  // namespace miw
