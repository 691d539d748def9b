/* hellm_b200.h -- C entry points of libhellm_b200.so: the HELLM::HEMMer call surface on one B200.
 *
 * The reference exposes this surface as the C++ class HELLM::HEMMer
 * (ciphertext/include/HELLM/HEMMer.hpp:33-438) over HETensor values (HETensor.hpp:46-86); it
 * has no C ABI.  The same class, with the reference's method names, is in this repository's
 * csrc/hellm/HEMMer.hpp for C++ callers; the functions below are that class for callers that
 * bind through C.  Each one names the HEMMer method (header line) and the schedule it runs
 * (ciphertext/src/MatrixUtils.cpp or HEMMer.cpp lines).
 *
 * Conventions
 *   - a tile tensor travels as a ciphertext handle plus (rows, cols, block_width), the
 *     TileTensorShape of the reference (HETensor.hpp:16-44);
 *   - inputs are borrowed for the call, outputs are new caller-owned handles (hb_ct_free);
 *   - every function returns 0 or a negative HB_E_* code (hemmer_b200.h); the reference throws
 *     std::invalid_argument for shape and level violations (MatrixUtils.cpp:27,36,680,1113,1322),
 *     reported here as HB_E_ARG with the same message through hb_hemmer_last_error();
 *   - all ciphertext handles may hold a batch: every function applies the schedule to all batch
 *     members with one set of launches.
 */
#ifndef HELLM_B200_H
#define HELLM_B200_H

#include "hemmer_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct hb_hemmer hb_hemmer;

/* HEMMer::HEMMer over an existing context with keys (HEMMer.cpp:93-209); masks are cached per object */
int hb_hemmer_create(hb_ctx *ctx, hb_hemmer **out);
void hb_hemmer_destroy(hb_hemmer *h);
/* message of the last failure raised above the primitive layer (thread-local) */
const char *hb_hemmer_last_error(void);
/* 0: the reference's rotation sequence, each shifted copy rotated from the previous one (default);
 * 1: every shifted copy is one rotation of the transformed operand, sharing its decomposition;
 * 2: as 1, and each wrapped copy (two rotations, two masks, add, rescale) is one hb_assemble_masked; the operands
 *    of singleCCMatMul are levelled down before sigma / tau; inside the transforms every masked sum is rescaled
 *    once (hb_sum_mul_pt_rescale) and the giant-step rotations share one ModDown (hb_rotate_sum).
 * All give the same slots and different ciphertext bits; no counterpart in the reference. */
int hb_hemmer_set_schedule(hb_hemmer *h, int mode);

/* HEMMer::genHEMMer (HEMMer.hpp:38-44; HEMMer.cpp:93-112): creates the context on `device`, generates the keys and
 * builds the HEMMer in one call; hb_hemmer_destroy then releases the context too.  hb_hemmer_context gives the
 * primitive-layer handle of either kind of HEMMer. */
int hb_hemmer_gen(int device, const hb_params *prm, hb_hemmer **out);
hb_ctx *hb_hemmer_context(const hb_hemmer *h);
/* HEMMer::getRank / getMaxRank (HEMMer.hpp:56-57): this process's GPU among the GPUs of the job (set by the launcher) */
int hb_hemmer_set_rank(hb_hemmer *h, int rank, int max_rank);
int hb_hemmer_get_rank(const hb_hemmer *h);
int hb_hemmer_get_max_rank(const hb_hemmer *h);
/* HEMMer::save (HEMMer.hpp:61; HEMMer.cpp:225-230): secret key and switching keys to files under keys_path */
int hb_hemmer_save(hb_hemmer *h, const char *keys_path);

/* HEMMer::encode / encode2 / encodeDiagonalToRow4 (HEMMer.hpp:65-86; HEMMer.cpp:232-275, 353-416): row-major rows x cols
 * matrices of doubles instead of torch::Tensor; level 0 means the encryption level, as in the reference.  encode2 lays
 * [d1 | d2] side by side (block width 2 * cols); encodeDiagonalToRow4 packs 1/2 (w1 - i w3) | 1/2 (w2 - i w4) with
 * column j rolled up by j rows. */
int hb_hemmer_encode(hb_hemmer *h, const double *data, int rows, int cols, int level, hb_pt **out);
int hb_hemmer_encode2(hb_hemmer *h, const double *d1, const double *d2, int rows, int cols, int level, hb_pt **out);
int hb_hemmer_encode_diagonal_to_row4(hb_hemmer *h, const double *w1, const double *w2, const double *w3, const double *w4, int rows, int cols,
                                      int level, hb_pt **out);
/* HEMMer::encrypt / encrypt2 (HEMMer.hpp:93-94; HEMMer.cpp:579-594); `nonce` selects the random streams (the reference
 * draws unseeded randomness) */
int hb_hemmer_encrypt(hb_hemmer *h, const double *data, int rows, int cols, uint64_t nonce, hb_ct **out);
int hb_hemmer_encrypt2(hb_hemmer *h, const double *d1, const double *d2, int rows, int cols, uint64_t nonce, hb_ct **out);
/* HEMMer::decrypt / decrypt2 (HEMMer.hpp:98-100; HEMMer.cpp:603-638): rows * cols doubles, or [2][rows][cols] */
int hb_hemmer_decrypt(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, double *out);
int hb_hemmer_decrypt2(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, double *out);
/* HEMMer::addInplace / hadamardMultInplace (HEMMer.hpp:102-115; HEMMer.cpp:683-713), returning a new handle */
int hb_hemmer_add(hb_hemmer *h, const hb_ct *a, const hb_ct *b, hb_ct **out);
int hb_hemmer_hadamard_mult(hb_hemmer *h, const hb_ct *a, const hb_ct *b, hb_ct **out);
int hb_hemmer_hadamard_mult_pt(hb_hemmer *h, const hb_ct *a, const hb_pt *p, hb_ct **out);
/* HEMMer::oneMatRotSumInplace (HEMMer.hpp:168; HEMMer.cpp:882-919) on two-tile ciphertexts */
int hb_hemmer_one_mat_rot_sum(hb_hemmer *h, const hb_ct *a, const hb_ct *b, hb_ct **out_a, hb_ct **out_b);
/* HEMMer::tr_oneMatRotSumInplace (HEMMer.cpp:921-962, HEAD_DIM = tile side): after an optional level-down to target_level + 1,
 * a holds the sum of every tile row on the left half of the row, b on the right half. */
int hb_hemmer_tr_one_mat_rot_sum(hb_hemmer *h, const hb_ct *a, const hb_ct *b, int target_level, hb_ct **out_a, hb_ct **out_b);

/* HEMMer::maskFirstColInplace (which = 0), maskLeftHalfInplace (1), maskRightHalfInplace (2) -- HEMMer.cpp:1251-1269 */
int hb_hemmer_mask_inplace(hb_hemmer *h, const hb_ct *a, int which, int rows, int cols, int width, hb_ct **out);
/* HEMMer::squareSum (HEMMer.cpp:2499-2510): rescale(relinearize(sum_i tensor(v[i], v[i]))) */
int hb_hemmer_square_sum(hb_hemmer *h, const hb_ct *const *v, int count, int rows, int cols, int width, hb_ct **out);
/* HEMMer::reduceRowSumWithScaledMask (HEMMer.cpp:2512-2530) on one rank; `mask` is encoded at the ciphertext's level */
int hb_hemmer_reduce_row_sum_with_scaled_mask(hb_hemmer *h, const hb_ct *a, const hb_pt *mask, int rows, int cols, int width, hb_ct **out);
/* The score assembly of the Gaussian-kernel attention in the reference's layer, TransformerBlock::attention2_bert_loraOpti
 * (TransformerBlock.cpp:2420-2482, for one query / key pair, up to the bootstrap): heads separated by maskRightLeft,
 * squared norms by square + oneMatRotSumInplace (+ transposeInplace on the key side), the products by complexPacking* +
 * packedMatMul + repackCC; out_j = |q_r|^2 + |k_c|^2 - 2 q_r . k_c for head position j of both tiles, at target_level. */
int hb_hemmer_gaussian_kernel_scores(hb_hemmer *h, const hb_ct *query, const hb_ct *key, int rows, int cols, int width, int target_level,
                                     hb_ct **out0, hb_ct **out1);
/* The rank-2 LoRA branch of a projection in the reference's layer, TransformerBlock::attention2_bert_loraOpti
 * (TransformerBlock.cpp:2199-2365) without the bootstraps around it: X A by slot-wise products with the rank vectors
 * spread over the token rows and a rotate-and-add across each row, then (X A) B the same way.  cur0..2: the three
 * [X_2i | X_2i+1] activation pairs; lora_wa / lora_wb: two-tile ciphertexts whose row 2i+j holds rank vector j for
 * pair i.  out0..2: the three output pairs. */
int hb_hemmer_lora_opti_forward(hb_hemmer *h, const hb_ct *cur0, const hb_ct *cur1, const hb_ct *cur2, const hb_ct *lora_wa, const hb_ct *lora_wb,
                                hb_ct **out0, hb_ct **out1, hb_ct **out2);

/* HEMMer::transposeInplace (HEMMer.hpp:129; HEMMer.cpp:1166-1172; MatrixUtils.cpp:671-739) */
int hb_hemmer_transpose(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int target_level, hb_ct **out);
/* MatrixTransformer::diagonalToColumn / diagonalToRow (MatrixUtils.cpp:776-848, 924-996) */
int hb_hemmer_sigma(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, hb_ct **out);
int hb_hemmer_tau(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, hb_ct **out);

/* HEMMer::singleCCMatMul (HEMMer.hpp:164-166; MatrixUtils.cpp:1307-1446) */
int hb_hemmer_matmul_cc(hb_hemmer *h, const hb_ct *a, int ra, int ca, int wa, const hb_ct *b, int rb, int cb, int wb,
                        int target_level, hb_ct **out);
/* the same product in two halves: the transforms (both results at target_level + 2), then the product loop.
 * Operands of different input levels can be transformed one by one and multiplied as one batch. */
int hb_hemmer_matmul_cc_prepare(hb_hemmer *h, const hb_ct *a, int ra, int ca, int wa, const hb_ct *b, int rb, int cb, int wb,
                                int target_level, hb_ct **sigma_a, hb_ct **tau_b);
int hb_hemmer_matmul_cc_core(hb_hemmer *h, const hb_ct *sigma_a, const hb_ct *tau_b, int rows, int inner, int cols, int width,
                             int target_level, hb_ct **out);
/* HEMMer::singleMatMul (HEMMer.hpp:160-162; MatrixUtils.cpp:1448-1570) */
int hb_hemmer_matmul_cp(hb_hemmer *h, const hb_ct *a, int ra, int ca, int wa, const hb_pt *b, int rb, int cb, int wb,
                        int target_level, hb_ct **out);
/* HEMMer::packedMatMul (HEMMer.cpp:833-838; MatrixUtils.cpp:1100-1216) */
int hb_hemmer_packed_matmul(hb_hemmer *h, const hb_ct *a, int ra, int ca, int wa, const hb_ct *b, int rb, int cb, int wb,
                            int target_level, hb_ct **out);

/* HEMMer::matMulPre (HEMMer.hpp:190-191; MatrixUtils.cpp:1572-1610): `out` is ONE handle whose batch holds the
 * shifted copies, copy k of input b at index k * batch(a) + b */
int hb_hemmer_matmul_pre(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int target_level, hb_ct **out);
/* HEMMer::matMulReUse (HEMMer.hpp:192-194; MatrixUtils.cpp:1612-1639; HEaaN matmul, HomEvaluator.hpp:595-601) */
int hb_hemmer_matmul_reuse(hb_hemmer *h, const hb_ct *pre, const hb_pt *w, int rows, int cols, int width, hb_ct **out);
/* sum over `bcount` inputs b0.. of matMulReUse(copies of input b, pts[b - b0]) in one pass; `pre` holds the copies
 * of `btotal` inputs.  The sum the reference takes with addInplace over K tiles (bert-matmul.cpp:268-287). */
int hb_hemmer_matmul_reuse_groups(hb_hemmer *h, const hb_ct *pre, int btotal, int b0, const hb_pt *const *pts, int bcount,
                                  int width, hb_ct **out);
/* the same for `tiles` weights (pts[t * bcount + b]) that meet the same copies: out[t], t < tiles */
int hb_hemmer_matmul_reuse_groups_tiles(hb_hemmer *h, const hb_ct *pre, int btotal, int b0, const hb_pt *const *pts, int bcount, int tiles,
                                        int width, hb_ct **out);
/* Products grouped by expert (hb_matmul_acc_grouped): position p takes input order[p] (NULL: p) and the weights of the expert whose run of
 * sizes[e] positions it lies in; copy k of K-group b of input i at batch position (k * inputs + i) * bcount + b of `pre`; member p * tiles + t of out. */
int hb_hemmer_matmul_reuse_grouped(hb_hemmer *h, const hb_ct *pre, int inputs, const int32_t *order, const int32_t *sizes, int experts,
                                   const hb_pt *const *pts, int bcount, int tiles, int width, hb_ct **out);
/* Tiles against tiles of another number: out[j][hd][i] = sum over r < inner of a[r][hd][i] * b[r][hd][j] for `heads` heads, members in that order, at
 * target_level; a needs target_level + 3 at least.  ra and cb divide ca, rounded up to a power of two, which is wb at most: tiles whose inner side is shorter
 * than their rows or columns are padded with zeros (HB_E_ARG otherwise).  The shifted copies of a tile are made once for all its pairs.  cross_scores: b = the transposed key
 * tiles, inner = 1 (schedule 2 transposes at target_level + 4, the others at the key's level).  No counterpart in the reference, whose sequences are one tile
 * long. */
int hb_hemmer_cross_matmul(hb_hemmer *h, const hb_ct *a, int ra, int ca, int wa, const hb_ct *b, int rb, int cb, int wb, int heads, int inner,
                           int target_level, hb_ct **out);
int hb_hemmer_cross_scores(hb_hemmer *h, const hb_ct *query, const hb_ct *key, int rows, int cols, int width, int heads, int target_level, hb_ct **out);
/* the same with key tiles of another number of rows.  A key tile that is not one of a pair (wk below rk + ck) has wk rows. */
int hb_hemmer_cross_scores_shaped(hb_hemmer *h, const hb_ct *query, int rq, int cq, int wq, const hb_ct *key, int rk, int ck, int wk, int heads, int target_level, hb_ct **out);
/* Encrypted vectors times a matrix in 4 bits (hb_matvec_q4), rescaled and summed over the rows.  x: ceil(rows / 4 d) members a vector (d: the tile two of
 * which fill a ciphertext), entry 4 d b + s of the vector in all columns of row s % d of member b: s < d left half, real part; s < 2 d right half, real
 * part; s < 3 d left half, imaginary part; then right half, imaginary part.  out: one member per vector and column tile, in every row
 * y / 2 = Re(left half) + Re(right half), one level below x. */
int hb_hemmer_matvec_q4(hb_hemmer *h, const hb_ct *x, const hb_qweight *w, hb_ct **out);
/* Layer norm and its gradients over rows that reach across `groups` column tiles (members [column tile][token tile], tiles whose rows fill the slots); `columns`
 * in all, the last tile may end early.  gamma, beta: `columns` doubles on the host, or NULL.  y = xhat gamma + beta with xhat = (x - mean) rstd; rstd is the polynomial of `degree`
 * (1 to 63) that stands for 1 / sqrt(variance + eps) on [lo, hi].  x needs 4 levels, those of the polynomial (hb_hemmer_polynomial), and one for gamma or a tile that
 * ends early.  hi - lo may be as wide as values are large: x is shrunk by a power of two on its way (at most to where the masks of the row sums keep 16 bits, else refused).
 * Outside [lo, hi] the polynomial soon grows beyond all bounds, and a slot beyond the modulus spoils all of them, so rows of padding (all zeros) have to be named: `tokens` has the
 * number of rows in front of them for every token tile (NULL: all rows), and they come out as beta.  Columns past the width have to be zero in x and dy and come out as zeros in y, dx,
 * dgamma and dbeta; in xhat they are not.  Rows of padding have to be zero in dy, or dbeta counts them.
 * The gradients need xhat at level 4 (5 where a tile ends early) and rstd at 1 (2); dy may be of another level than xhat, but is multiplied by gamma first, which takes one of its own.  So
 * in a ring of 12 levels forward passes of degrees up to 14 keep what they need (up to 6 where a tile ends early); with higher ones xhat ends too low, and the framework has no
 * bootstrapping to refresh it.  dgamma and dbeta have one member per column tile, summed over all rows and token tiles, in every row.  Plaintexts are encoded from the host at every call that has
 * gamma, beta or padding, which cannot be recorded then.  No counterparts in the reference's HEMMer: its LayerNorm class does the like with other polynomials. */
int hb_hemmer_layer_norm(hb_hemmer *h, const hb_ct *x, int rows, int cols, int width, int groups, int columns, const double *gamma, const double *beta, double eps, double lo, double hi, int degree,
                         const int32_t *tokens, hb_ct **y, hb_ct **xhat, hb_ct **rstd);
int hb_hemmer_layer_norm_backward(hb_hemmer *h, const hb_ct *dy, const hb_ct *xhat, const hb_ct *rstd, int rows, int cols, int width, int groups, int columns, const double *gamma, hb_ct **dx,
                                  hb_ct **dgamma, hb_ct **dbeta);
/* The square of the global norm of the gradients, over all slots of all members of all handles (imaginary parts have to be zero), in every slot, one level below the lowest of them; and all of
 * them times min(1, max_norm / norm): a polynomial of `degree` in the square of the norm, right up to norms of `bound` > max_norm, which a degree of 15 meets to 0.05 for bound = 4 max_norm.  3 levels and those of the
 * polynomial; outs receives a handle per gradient, norm_squared (may be NULL) the square.  Beyond `bound` the polynomial is no root and soon grows beyond all bounds: decrypted, norm_squared tells.
 * 2 / bound^2 is a whole number at the scale (2^42): from a bound of 2048 on the bound is widened to where it is one, by up to 1/16 at 10^6; larger ones are refused, as are
 * those below 2^-9, whose number has more than 62 bits. */
int hb_hemmer_grad_norm_squared(hb_hemmer *h, const hb_ct *const *grads, int count, hb_ct **out);
int hb_hemmer_clip_grad_norm(hb_hemmer *h, const hb_ct *const *grads, int count, double max_norm, double bound, int degree, hb_ct **outs, hb_ct **norm_squared);
/* Those count every slot: a gradient that holds its values several times, as dgamma and dbeta of hb_hemmer_layer_norm_backward do in every row, counts as many times.  With `periods`, a power of two
 * for every gradient (the block width for dgamma and dbeta, the number of slots for those that do not repeat), values count once; what is said to repeat has to.  NULL: none does. */
int hb_hemmer_grad_norm_squared_periodic(hb_hemmer *h, const hb_ct *const *grads, const int32_t *periods, int count, hb_ct **out);
int hb_hemmer_clip_grad_norm_periodic(hb_hemmer *h, const hb_ct *const *grads, const int32_t *periods, int count, double max_norm, double bound, int degree, hb_ct **outs, hb_ct **norm_squared);
/* Those polynomials: which = 0 for 1 / sqrt over [a, b], 1 for min(1, a / sqrt) over [0, b^2], as degree + 1 coefficients of T_j(u), u the place of the argument in [-1, 1].  depth (may be NULL):
 * levels of its evaluation.  Needs no device. */
int hb_hemmer_polynomial(int which, double a, double b, int degree, double *coefficients, int *depth);
/* HEMMer::matMulPreRev, matMulCCReUse (HEMMer.cpp:1114-1124; MatrixUtils.cpp:1641-1679) */
int hb_hemmer_matmul_pre_rev(hb_hemmer *h, const hb_ct *b, int rows, int cols, int width, int target_level, hb_ct **out);
int hb_hemmer_matmul_cc_reuse(hb_hemmer *h, const hb_ct *pre, const hb_ct *b, int rows, int cols, int width, hb_ct **out);
/* HEMMer::packedMatMulPre, PreRot, PreRev, CCReuse (HEMMer.cpp:840-864; MatrixUtils.cpp:1218-1305) */
int hb_hemmer_packed_matmul_pre(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int target_level, hb_ct **out);
int hb_hemmer_packed_matmul_pre_rot(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int target_level, hb_ct **out);
int hb_hemmer_packed_matmul_pre_rev(hb_hemmer *h, const hb_ct *b, int rows, int cols, int width, int target_level, hb_ct **out);
int hb_hemmer_packed_matmul_cc_reuse(hb_hemmer *h, const hb_ct *pre, const hb_ct *b, int rows, int cols, int width, hb_ct **out);

/* HEMMer::complexPackingInplace, complexPackingRowInplace, transposeComplexPackingInplace (HEMMer.cpp:764-817) */
int hb_hemmer_complex_packing(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, hb_ct **out);
int hb_hemmer_complex_packing_row(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, hb_ct **out);
int hb_hemmer_transpose_complex_packing(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int target_level, hb_ct **out);
/* HEMMer::splitInTwo (HEMMer.cpp:819-831) */
int hb_hemmer_split_in_two(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, hb_ct **out1, hb_ct **out2);
/* HEMMer::repackCC (HEMMer.cpp:964-969), complexPacking(ct, ct) (:980-986), complexPackingRev (:988-994),
 * repack_notBTS (:1025-1053) */
int hb_hemmer_repack_cc(hb_hemmer *h, const hb_ct *a, hb_ct **out);
int hb_hemmer_complex_packing2(hb_hemmer *h, const hb_ct *a, const hb_ct *b, hb_ct **out);
int hb_hemmer_complex_packing_rev(hb_hemmer *h, const hb_ct *a, const hb_ct *b, hb_ct **out);
int hb_hemmer_repack_not_bts(hb_hemmer *h, const hb_ct *a, const hb_ct *b, hb_ct **out);
/* HEMMer::repack_loraOpti (HEMMer.cpp:1055-1091): repack_notBTS followed by the split of real and imaginary part
 * that the reference otherwise gets from bootstrapExtended */
int hb_hemmer_repack_lora_opti(hb_hemmer *h, const hb_ct *a, const hb_ct *b, hb_ct **out);

/* LoRA low-rank family.  `low_dim` is the width of the thin factor, ModelArgs::LOW_DIM in the reference
 * (ModelArgs.hpp:67, a compile-time 2 there); `in_*_block` / `block` is the index of the low_dim-wide column
 * (row) block the thin factor occupies inside its tile.
 * HEMMer::matMulHighLow / matMulLowHigh / matMulLowLow (HEMMer.hpp:326-334; MatrixUtils.cpp:1681-1996) */
int hb_hemmer_matmul_high_low(hb_hemmer *h, const hb_ct *a, int ra, int ca, int wa, const hb_ct *b, int rb, int cb, int wb,
                              int in_col_block, int target_level, int low_dim, hb_ct **out);
int hb_hemmer_matmul_low_high(hb_hemmer *h, const hb_ct *a, int ra, int ca, int wa, const hb_ct *b, int rb, int cb, int wb,
                              int in_row_block, int target_level, int low_dim, hb_ct **out);
int hb_hemmer_matmul_low_low(hb_hemmer *h, const hb_ct *a, int ra, int ca, int wa, const hb_ct *b, int rb, int cb, int wb,
                             int in_col_block, int in_row_block, int target_level, int low_dim, hb_ct **out);
/* HEMMer::repackToOneCol / MultiCol / OneRow / MultiRow (HEMMer.hpp:336-343; HEMMer.cpp:2131-2290): fold the
 * partial sums the products above leave spread over the blocks into block `block` */
int hb_hemmer_repack_to_one_col(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int block, int low_dim, hb_ct **out);
int hb_hemmer_repack_to_multi_col(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int block, int low_dim, hb_ct **out);
int hb_hemmer_repack_to_one_row(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int block, int low_dim, hb_ct **out);
int hb_hemmer_repack_to_multi_row(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int block, int low_dim, hb_ct **out);
/* HEMMer::getLowColBlock / getLowRowBlock (HEMMer.hpp:345-346; HEMMer.cpp:2292-2332): keep one block of every tile */
int hb_hemmer_low_col_block(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int block, int low_dim, hb_ct **out);
int hb_hemmer_low_row_block(hb_hemmer *h, const hb_ct *a, int rows, int cols, int width, int block, int low_dim, hb_ct **out);

#ifdef __cplusplus
}
#endif
#endif /* HELLM_B200_H */
