/* helix_b200_kernels.h — kernel-level C ABI (plain device pointers + sizes, stream 0 unless given).
 * These are the individual sm_100a ops K1–K11 of SURVEY.md §2.3 that the engine composes; they are
 * exported so parity tests (and a host shim that wants a single op) can drive each kernel in
 * isolation.  All return a cudaError_t value (0 = ok) or -1 for an invalid argument; launches are
 * asynchronous on the legacy default stream and the caller synchronises.
 */
#ifndef HELIX_B200_KERNELS_H_
#define HELIX_B200_KERNELS_H_
#include <stddef.h>
#include <stdint.h>

#include "helix_b200.h"
#ifdef __cplusplus
extern "C" {
#endif

int hbk_init(void);
const char* hbk_last_error(void);

/* C[M,N] = A[M,K] . W[N,K]^T, bf16 in; epi = enum hb::Epi (0 none,1 bias,2 bias+gelu,3 resid,4 bias+resid,
 * 5 swiglu (W packed [128 gate|128 up] per 256 rows, C has N/2 columns), 6 fp32 out). block_n 0 = auto. */
int hbk_gemm(const void* A, int lda, const void* W, int ldw, void* C, int ldc, const void* R, int ldr, const void* bias,
             int M, int N, int K, int epi, int block_n);
/* tile that hbk_gemm with block_n 0 picks on `sms` SMs: columns | CTAs of 128 rows << 12 | groups of four epilogue warps << 16; no device is asked */
int hbk_gemm_tile(int M, int N, int K, int epi, int sms);
/* decode-step GEMM (M<=256): swap-AB + stream-K partial slabs summed in fixed order -> out fp32 [M,N] */
int hbk_gemm_skinny(const void* X, int ldx, const void* W, int ldw, float* out_f32, int ldo, int M, int N, int K);
/* the same GEMM with the fused tile finisher (last-arriving CTA of each output tile sums the slabs in slab order and
 * writes out[m, n]); launched `repeats` times back to back: the arrival counters must return to zero by themselves */
int hbk_gemm_skinny_finish(const void* X, int ldx, const void* W, int ldw, float* out_f32, int ldo, int M, int N, int K,
                           int repeats);
/* two such products of the same M rows in one launch, cut for `sms` SMs (0 = all): the bits that each has by itself */
int hbk_gemm_skinny_pair(const void* X, int ldx, const void* W, int ldw, float* out_f32, int ldo, int N, int K, const void* X2, int ldx2,
                         const void* W2, int ldw2, float* out2_f32, int ldo2, int N2, int K2, int M, int sms);
/* slabs of a 128-column tile at most where such a product is cut for `sms` SMs; no device is asked */
int hbk_gemm_skinny_slabs(int N, int K, int sms);
/* floats that an engine with this sm_budget (0 = none) sets aside for such slabs, for steps of up to 256 tokens of a layer-list decoder; -1: a
 * description that the engine refuses.  No device is asked */
int64_t hbk_stack_slab_floats(const hb_stack_desc* desc, const hb_layer_desc* layers, int sm_budget);
int hbk_gemm_naive(const void* A, int lda, const void* W, int ldw, void* C_f32, int ldc, int M, int N, int K);

int hbk_embed_gather(const int32_t* tokens, const void* table, void* x, int T, int H);
int hbk_bert_embed_ln(const int32_t* tokens, const int32_t* positions, const void* word, const void* pos,
                      const void* type0, const void* gamma, const void* beta, void* x, int T, int H, float eps);
int hbk_rmsnorm(const void* x, const void* w, void* out, const int32_t* row_index, int rows, int H, float eps);
int hbk_layernorm(const void* x, const void* gamma, const void* beta, void* out, int rows, int H, float eps);
int hbk_rope_kv_write(void* qkv, const int32_t* positions, const int32_t* slot_mapping, const float* inv_freq,
                      void* k_cache, void* v_cache, int T, int Hq, int Hkv, int D, int page_size);
/* QKV projection with RoPE + KV scatter in the GEMM epilogue (EPI_ROPE): qkv[T, (Hq+2Hkv)*D] = A[T,K] * W^T (+ bias), q / k heads
   rotated, k / v rows also written to the paged cache — must equal hbk_gemm followed by hbk_rope_kv_write bit for bit */
int hbk_gemm_qkv_rope(const void* A, int lda, const void* W, int ldw, void* qkv, const void* bias, const int32_t* positions,
                      const int32_t* slot_mapping, const float* inv_freq, void* k_cache, void* v_cache, int T, int K,
                      int Hq, int Hkv, int D, int page_size);
int hbk_sample(const float* logits, int ldl, const float* temperature, const uint64_t* seed, int32_t* out, int B, int V);
/* as hbk_sample, restricted per row to the top_k / top_p survivors (either pointer may be NULL) */
int hbk_sample_filtered(const float* logits, int ldl, const float* temperature, const uint64_t* seed, const int32_t* top_k,
                        const float* top_p, int32_t* out, int B, int V);
/* OpenAI presence / frequency penalties: logits[b, tok] -= val over row b's entries {int32 tok; float val}
 * [pen_off[b], pen_off[b+1]) (distinct tokens per row; val = presence + frequency * count, computed by the caller) */
int hbk_apply_penalties(float* logits, int ldl, const int32_t* pen_off, const void* pen_entries, int B, int V);
/* rows with width[b] > 0: out_ids/out_lp[b][0] = sampled[b] and its log-softmax; [1..width[b]) = the most likely tokens in
 * descending order (lowest id first on ties).  out_* are [B][max_width]. */
int hbk_logprob_topk(const float* logits, int ldl, int V, const int32_t* sampled, const int32_t* width, int32_t* out_ids,
                     float* out_lp, int B, int max_width);
/* The start of a stack with parallel sublayers: x = rms norm (gain off + w0) of scale * table[token] (+ the row of a token pair in `pairs`: buckets + 1 rows,
 * row (prev mul_prev + token mul_cur) % buckets, the last one where prev < 0; NULL: none), h1 / h2 = rms norms of x with gains w1 / w2 (w2 may be NULL),
 * fp32 and bf16 (any output of h1, h2 may be NULL).  f32: fp32 weights, else bf16.  parts: three launches instead of one, the same bits. */
int hbk_embed_step(const int32_t* tokens, const void* table, float scale, const void* pairs, const int32_t* prev, int buckets, int mul_prev,
                   int mul_cur, const void* w0, float off, const void* w1, const void* w2, int f32, float eps, float* x, float* h1, void* h1_b16,
                   float* h2, void* h2_b16, int T, int W, int parts);
int hbk_cls_pool_l2(const void* x, const int32_t* first_row, float* out, int B, int H);

int hbk_attn_prefill(const void* q, int ldq, const void* k, int ldk, const void* v, int ldv, void* out, int ldo,
                     const int32_t* cu_seqlens, int B, int T, int max_seqlen, int Hq, int Hkv, int D, int causal,
                     float scale);
/* chunked prefill: the cu_seqlens[b+1]-cu_seqlens[b] q rows of sequence b are the LAST positions of a kv_lens[b]-long
 * sequence whose K/V (this chunk's included) are in the paged pool plane [num_pages][Hkv][64][D] (page size 64). */
int hbk_attn_prefill_paged(const void* q, int ldq, const void* k_cache, const void* v_cache, const int32_t* page_table,
                           int max_pages, const int32_t* kv_lens, void* out, int ldo, const int32_t* cu_seqlens, int B,
                           int T, int max_q_len, int Hq, int Hkv, int D, int causal, float scale, int num_pages);
/* the same, causal, with what layers add to it: window > 0: a position sees that many, itself included; block_mask > 0: those of its own
 * block of so many positions; softcap > 0: scores pass softcap * tanh(s / softcap); unit_sink: one unit more in the denominator;
 * sink [Hq] bf16 (or NULL): exp(sink[h]) more; head_gate fp32 [T, ldg] (or NULL): head h's result times sigmoid(head_gate[t][h]). */
int hbk_attn_prefill_paged_with(const void* q, int ldq, const void* k_cache, const void* v_cache, const int32_t* page_table,
                                int max_pages, const int32_t* kv_lens, void* out, int ldo, const int32_t* cu_seqlens, int B,
                                int T, int max_q_len, int Hq, int Hkv, int D, float scale, int num_pages, int window,
                                int block_mask, float softcap, int unit_sink, const void* sink, const float* head_gate, int ldg);
/* how hbk_attn_prefill (paged 0) or hbk_attn_prefill_paged (1) cuts a launch of these sizes on `sms` SMs: query heads of a kv head that
 * share the rows of a tile, + 256 where the items are sorted by length.  Host arithmetic only; -1 for sizes that are refused. */
int hbk_attn_prefill_plan(int B, int T, int max_seqlen, int Hq, int Hkv, int paged, int sms);
int hbk_attn_naive(const void* q, int ldq, const void* k, int ldk, const void* v, int ldv, float* out_f32, int ldo,
                   const int32_t* cu_seqlens, int B, int T, int max_seqlen, int Hq, int Hkv, int D, int causal,
                   float scale);
int hbk_attn_decode(const void* q, int ldq, const void* k_cache, const void* v_cache, const int32_t* page_table,
                    int max_pages, const int32_t* ctx_lens, void* out, int ldo, float* workspace, int B, int Hq, int Hkv,
                    int D, int page_size, int num_splits, float scale, int num_pages);
size_t hbk_attn_decode_workspace_floats(int B, int Hq, int D, int num_splits);

/* ---- a step whose cache and weights are held in 4 bits.  32 neighbouring entries share a scale d and a code c in 0..15 stands for d (c - 8); with m the
 * entry of largest magnitude (the first of equals) d = m / -8 rounded, c = clamp(floor(x / d + 1/2) + 8, 0, 15), 8 where d = 0.  These calls take the
 * stream they run on (NULL: the legacy default stream), allocate nothing, never wait, and can be captured into a graph; a call's buffers must be on the
 * current device, and outputs overlap no input but where it is said.  Row strides count entries and are multiples of 8, rows of bf16 read in whole begin on 16 bytes.
 *
 * Page tables, slot maps and packed-row indices from lengths, in one launch.  Request b has ctx_lens[b] cached positions in the first ceil(ctx / 64) pages of
 * its row of page_table [B][max_pages].  new_lens[b] >= 0: it has that many more tokens in this step and takes the pages that they need from the top
 * of the stack free_pages[0 .. *free_count), in request order; new_lens[b] < 0: it has ended, its pages go on top of the stack first.
 * Out: the new entries of page_table; the stack and its height *free_left; cu_seqlens [B + 1], rows of the packed batch (capped at T); kv_lens [B] = ctx + new,
 * 0 for a request that has ended; positions [T] and slot_mapping [T] (page * 64 + place), 0 and -1 behind the last token.
 * A request that does not fit (more than max_pages pages, rows past T, or the first that finds too few pages and every later one that needs some) takes no page:
 * kv_lens[b] = ctx_lens[b] says so, and its rows have slot -1.  free_left may be free_count and kv_lens may be ctx_lens; nothing else may overlap.
 * free_pages has room for num_pages entries.  1 <= B <= 2048, T up to 2^30, page_size 64.  Lengths below 0 in ctx_lens count as 0. */
int hbk_page_tables(const int32_t* ctx_lens, const int32_t* new_lens, int B, int32_t* page_table, int max_pages, int32_t* free_pages,
                    const int32_t* free_count, int32_t* free_left, int num_pages, int32_t* cu_seqlens, int32_t* kv_lens, int32_t* positions,
                    int32_t* slot_mapping, int T, int page_size, void* stream);
/* A 4-bit cache plane (one of K, one of V): [num_pages][Hkv][block], block = 64 rows of D / 2 bytes of codes, then 64 rows of D / 32 bf16 scales (D 64 or 128).
 * K codes: position p's row at p D / 2; word j (4 bytes) of its quarter t (D / 8 bytes) holds entries 32 j + 8 t + i, i = 0..7, even i in nibble i / 2, odd i in
 * nibble 4 + i / 2.  V codes: positions 2 n and 2 n + 1 share the D bytes at n D; chunk g (D / 8 bytes, at place g ^ 2 (n mod 4) for D = 128, g ^ 4 (n / 2 mod 2) for
 * D = 64) holds in word j entries 32 j + 4 g + r, r = 0..3, of the even position in nibble r, of the odd one in nibble 4 + r. */
size_t hbk_kv_q4_plane_bytes(int num_pages, int Hkv, int D); /* 0: refused sizes */
/* Rows k, v [T][>= Hkv * D] (bf16, k rotated) into the planes at slot_mapping [T] (a slot that is none, -1 say: the row is not stored; no slot may occur twice).
 * k_seen / v_seen (or NULL; may be k / v): the rows as the cache now stands for them, rounded to bf16: what a prompt's own attention reads
 * if it shall see what later steps will.  A group with an infinity or a NaN reads as NaN. */
int hbk_kv_write_q4(const void* k, int ldk, const void* v, int ldv, const int32_t* slot_mapping, void* k_cache, void* v_cache, void* k_seen, int ldks,
                    void* v_seen, int ldvs, int T, int Hkv, int D, int page_size, int num_pages, void* stream);
/* Attention over such planes: rows [cu_seqlens[b], cu_seqlens[b + 1]) of q are the last positions of the kv_lens[b]-long sequence b (at most max_q_len of them;
 * cu_seqlens NULL: one row per sequence, row b), each sees the positions up to its own. Any Hq / Hkv up to 4096, Hkv up to 65535, max_q_len * Hq up to 2^30.
 * window, softcap and sink as in hbk_attn_prefill_paged_with. A row that sees nothing (length 0) is 0; rows of no sequence keep what they hold. No kv_lens entry
 * is above max_kv_len or max_pages * 64 (what lies past either is cut off the sequence), positions of a page number outside the pool are not seen. Value scales
 * may differ by any factor (shares in which those of a group differ by more than 2^16 take up to fifty times as long); a weight counts to 2^-10 of itself or
 * 2^-23 of its row's largest. Entries of q below 2^-27 of the largest of their head's row lose bits, and with 256 columns key scales below 2^-25 of the largest
 * of their position; keys from 2^105 on overflow, however small the queries. split_pages: pages that one block reads of a sequence at most (a row's bits depend
 * on its sequence, on it and on whether max_q_len * Hq / Hkv is 256 or more, on nothing else); 0: hbk_attn_paged_q4_split's. Single tokens beside portions of
 * 256 columns (rows * Hq / Hkv) are quicker in a call of their own. workspace: as many floats as hbk_attn_paged_q4_workspace_floats says for the same arguments
 * (0: none, it may be NULL; on 16 bytes); launches that may run at the same time need one each. */
int hbk_attn_paged_q4(const void* q, int ldq, const void* k_cache, const void* v_cache, const int32_t* page_table, int max_pages, const int32_t* kv_lens,
                      const int32_t* cu_seqlens, void* out, int ldo, float* workspace, int B, int T, int max_q_len, int max_kv_len, int Hq, int Hkv, int D,
                      int page_size, int split_pages, float scale, int num_pages, int window, float softcap, const void* sink, void* stream);
/* Calls with 256 columns wait inside the kernel for one another's parts.  A wait that takes some seconds is given up: the rows it was for are NaN, the kernel ends, and
 * this says so: 0, or cudaErrorLaunchTimeout (702) where one was given up on the current device since it was last asked.  To be asked once the calls' stream is
 * synchronised, and not while a stream is captured. */
int hbk_attn_paged_q4_status(void);
/* cycles after which such a wait is given up by the calls that follow (below 0: at once), of the whole process; returns the former */
long long hbk_attn_paged_q4_wait_cycles(long long cycles);
/* pages per block by the rule for `sms` SMs (0: the current device's) and T = B * max_q_len rows (where a call has fewer, its own rule may take shorter shares: the
 * rule keeps the workspace within 2^28 floats); host arithmetic, -1 for refused sizes */
int hbk_attn_paged_q4_split(int B, int max_q_len, int max_kv_len, int Hq, int Hkv, int window, int sms);
size_t hbk_attn_paged_q4_workspace_floats(int B, int T, int max_q_len, int max_kv_len, int Hq, int Hkv, int D, int split_pages, int window);
/* 4-bit weights: N rows of K / 32 GGUF Q4_0 blocks (18 bytes: fp16 d, then byte i with entries i and i + 16; device memory) laid out as the product reads them, in
 * hbk_gemm_q4_bytes(N, K) bytes (K a multiple of 32 up to 2^30 - 128, N up to 65535 * 64): tiles [ceil(N / 16)][ceil(K / 128)] of 16 rows of 64 bytes as K
 * codes above with D = 128, then [16 rows][4 groups] fp16 scales. */
size_t hbk_gemm_q4_bytes(int N, int K); /* 0: refused sizes */
int hbk_gemm_q4_pack(const void* blocks, void* packed, int N, int K, void* stream);
/* out[M, N] = X[M, K] . W4[N, K]^T, M <= 256 (made for the rows of a decode step: beyond 32 rows hbk_gemm with bf16 weights is quicker); epi as in hbk_gemm: 0, 1, 3, 4
 * (bf16 out) or 6 (fp32 out); R may be out itself */
int hbk_gemm_q4(const void* X, int ldx, const void* W4, void* out, int ldo, const void* R, int ldr, const void* bias, int M, int N, int K, int epi,
                void* stream);

#ifdef __cplusplus
}
#endif
#endif
