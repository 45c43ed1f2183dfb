// w4.h - 4-bit weights with group scales, and tokens sorted by expert: what the kernels of w4_*.cu and
// expert_rows.cu share (internal to libglm53f_b200). Every launcher enqueues on the given stream.
//
// A matrix W[rows][cols]: codes of 4 bits, two to a byte (the even column in the low half), rows `pitch` bytes apart; a
// BF16 scale for each row and group of 32, 64 or 128 columns, rows `sp` scales apart. W[r][k] = (code - 8) * scale. What
// lies behind the last column or group of a row is never used.
#pragma once

#include "kernels.h"

namespace g5b {

struct W4Mat {
    const uint8_t  *codes;
    const uint16_t *scales;
    int rows, cols, group;      // group: 32, 64 or 128
    int pitch, sp;              // bytes of a row of codes (a multiple of 16), scales of a row (a multiple of 8)
    int groups;                 // scales of a row that count
    size_t codes_stride, scales_stride;     // between the matrices of a stack
};

// Activation rows as F16 terms: x 2^e = hi (+ mid), e of the row; `kp` columns a term, a multiple of 128, zero behind the
// last one, in each eight the order 0 4 1 5 2 6 3 7 (the order in which the nibbles of a word come out as pairs). A row
// with an infinity or NaN: zero terms and inv = NaN.
struct W4Terms {
    void  *terms;               // [row][term][kp] F16
    float *inv;                 // [row] 2^-e
    int n_terms, kp;
};
inline int w4_kp(int cols) { return (cols + 127) / 128 * 128; }

// rows: at most; n_rows (device, may be null): how many of them count; order (may be null): row i is x's row order[i] / topk
void w4_split(cudaStream_t st, const W4Terms &t, const void *x, int dt, size_t ldx, int rows, int cols, const int *n_rows, const int *order, int topk,
              bool early);

// Tiles of the experts' rows: slot s multiplies expert[s] with rows first[s] .. first[s] + count[s] of the sorted ones.
struct W4Slots {
    int *n, *expert, *first, *count;
    int max, rows;              // slots at most; rows of a tile at most
    // many_rows > 0: the sort chooses. Up to few_most picks of experts here make slots of `rows`; with more, slots of many_rows, and then
    // their number is n[1], that of the picks n[2], and n[0] is 0 (else n[1] and n[2] are).
    int many_rows, few_most;
};
enum { W4_DENSE = 0, W4_GATEUP = 1, W4_DOWN = 2 };
struct W4Job {
    int mode;
    W4Mat w, up;                // gate/up: w is the gate
    int count;                  // matrices of the stack
    int T;                      // rows of activations (experts: picks, at most)
    const void *x; int x_dt; size_t ldx;        // w4_few: the activations (dense, gate/up: the caller's; down: F32 rows of picks)
    const int *order; int topk;                 // w4_few, gate/up: the activation row of sorted row i is order[i] / topk
    const int *idx;             // w4_few: not sorted, every pick a slot of its own (32 at most; slots and order are not used then)
    bool early;                 // w4_few: may be scheduled while the kernel before it drains
    W4Terms terms;              // w4_many: the activations as terms, in the order of the rows
    W4Slots slots;
    void *y; size_t ldy; int y_dt;
    float limit;
};
// Rows that w4_few takes at a time, of a matrix of so many columns (0: none). Dense products of up to as many are its (past three
// or four rows the weights twice take 20.8 us for 12288 x 4096 in groups of 32, w4_many 17.6).
int  w4_few_rows(int cols);
inline bool w4_few_takes(int cols, int T) { return T <= w4_few_rows(cols); }
int  w4_few(cudaStream_t st, const W4Job &job);
int  w4_few_status(cudaStream_t st);
constexpr int W4_MANY_ROWS = 64;
size_t w4_many_part_floats(int rows, int cols, int T);                           // room for the sums of a dense product's parts
int  w4_many(cudaStream_t st, const W4Job &job, float *part);
int  w4_many_status(cudaStream_t st);

// ---- expert_rows.cu
int  expert_sort(cudaStream_t st, const int *idx, int T, int topk, int E, int *order, int *place, int *offsets, const W4Slots *slots);
void expert_gather(cudaStream_t st, const void *x, size_t row_bytes, size_t x_bytes, size_t out_bytes, const int *order, const int *offsets,
                   int n, int topk, int E, void *rows);
// place, or (E > 0) picks as they came: row p is pick p's, if its expert is one of E
void expert_combine(cudaStream_t st, const void *rows, int rows_dt, size_t ldr, const int *place, int E, const float *w, int T, int topk, int cols,
                    void *out, int out_dt, size_t ldo, bool early);

// ---- w4_convert.cu
void w4_quantize(cudaStream_t st, const W4Mat &w, const void *src, int dt, const float *scale, int br, int bc);
void w4_dequantize(cudaStream_t st, const W4Mat &w, void *out, int dt, size_t ldo);

}  // namespace g5b
