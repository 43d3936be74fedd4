/*
 * libana -- MI355X (gfx950) decoder token loop for hhefesto/ana checkpoints.
 *
 * A plain C ABI over hand-written HIP kernels. It replaces the dense engine
 * seam of bend/Decode.bend (EDense, driven through Dd.dd.{load, feed, feeds,
 * logits, top, reset} of bend/Dense/Decode.bend:531-699) at engine
 * granularity: one call runs a whole decode step (every layer), not one
 * bulk op.
 *
 * Conventions
 *   - Every int-returning function answers 0 on success, or a nonzero
 *     ANA_E* code; ana_error(ctx) (or ana_error(NULL) after a failed
 *     ana_open) then holds the message, using the reference's wording where
 *     the reference has one (e.g. "checkpoint: short read").
 *   - Host buffers are the caller's, read or written only during the call.
 *     Device memory is the library's.
 *   - A context is single-threaded: the caller serialises calls on it, as
 *     the reference serialises the GPU with FT.mu (bend/effs/bulk.c:79-92).
 *     Every call returns after its device work has completed.
 *   - Sequences are slots 0 .. max_seqs-1 of a context; each keeps its own
 *     recurrent state (GLA S per layer and head, softmax K/V rings) and the
 *     residual row of the last token fed, as one dense store does for one
 *     sequence in the reference.
 *   - Positions count tokens from 0 per sequence; the softmax ring slot is
 *     pos mod ctx and the last live slot min(pos, ctx-1)
 *     (bend/Dense/Decode.bend:540-545).
 */
#ifndef ANA_H
#define ANA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ANA_ABI_VERSION 1

/* error codes */
#define ANA_OK 0
#define ANA_EINVAL 1     /* bad argument (sequence, position, token, size) */
#define ANA_ECKPT 2      /* checkpoint rejected (Manifest.problem, short read, ...) */
#define ANA_EDEVICE 3    /* HIP error: "device fault" */
#define ANA_ENOMEM 4     /* device allocation failed */
#define ANA_EUNSUP 5     /* configuration outside what the kernels handle */
#define ANA_ETOK 6       /* tokenizer artifact unreadable or rejected (Bpe.parse) */
#define ANA_ETIME 7      /* a wait between the persistent decode kernel's workgroups passed
                            its time limit (a stalled or heavily shared GPU): the call's
                            sequence is partly advanced and must be reset (ana_reset)
                            before it is fed again */

/* numerics modes */
#define ANA_EXACT_FP32 0 /* bit-exact with the reference's CPU kernels */
#define ANA_FAST_FP32 1  /* fp32, sums reassociated (split-K, fused multiply-add):
                            logits within 1e-4 of the reference, relative to their
                            largest magnitude */
#define ANA_BF16 2       /* matrices read as bfloat16 (rounded once at load); fp32
                            activations, accumulation and state: logits within 2e-2 */

/* ANA_FAST_FP32 | ANA_KV4 or ANA_BF16 | ANA_KV4: the softmax layers' K and V rings
 * in 4 bits, 7.5 times smaller than in fp32 (the cache of ana_kv4 below: at d 768 and ctx
 * 2048, 12.6 MB a layer and sequence become 1.7 MB). Every row attends
 * to keys and values as the rings hold them, its own too; all else is the mode's. The
 * rounding is the checkpoint's to bear: the modes' tolerances do not cover it. Head
 * dimensions of 32 and 64, positions below 2^31 (ANA_EINVAL past them); the one-sequence
 * loops take the step graphs. ANA_EUNSUP with ANA_EXACT_FP32 */
#define ANA_KV4 0x100

/* bend/Config.bend:7-10 */
typedef struct {
  uint32_t vocab, ctx, d, f, layers, heads;
  uint32_t rglru, qk, sinks, tied;
} ana_config;

typedef struct {
  int device;              /* HIP device ordinal */
  int numerics;            /* ANA_EXACT_FP32, ANA_FAST_FP32 or ANA_BF16, the last two
                              also with ANA_KV4 */
  uint32_t max_seqs;       /* sequences the context keeps state for (>= 1) */
  uint32_t prefill_chunk;  /* tokens of each sequence a prefill step takes; 0 = 64, as
                              ANA_PREFILL_CHUNK. In ANA_BF16, and past the ring's wrap, exactly
                              that; else at least that, and more where the step's rows (up to
                              8192 over its sequences) have room: a program that wants shorter
                              steps feeds shorter pieces. In the fast modes how a prompt's
                              values round follows its steps, so also what is fed beside it */
} ana_opts;

/* the decoding settings of bend/Decode.bend:147-148,546-548 */
typedef struct {
  float temperature;       /* <= 0: greedy (argmax, least index on ties) */
  uint32_t top_k;          /* on when < vocab (0xFFFFFFFF = off) */
  float top_p;             /* on when < 1 */
} ana_sampling;

/* Open an FTC2 checkpoint on a device.
 * Replaces dc.loaded.dense + Dd.dd.of.n + Dd.dd.load
 * (bend/Decode.bend:501-520, bend/Dense/Decode.bend:492-518,689-699): the
 * manifest is validated as Manifest.problem (bend/Checkpoint.bend:162-170),
 * the parameter count and a tied head are required, and the P big-endian
 * floats are read into device memory. All sequences start reset. */
int ana_open(const char* ftc2_path, const ana_opts* opts, struct ana_ctx** out);

/* The checkpoint's config and the Adam step it was saved at. */
int ana_config_of(const struct ana_ctx* ctx, ana_config* out, uint64_t* step);

/* Zero one sequence's states: dd.reset (bend/Dense/Decode.bend:534-538). */
int ana_reset(struct ana_ctx* ctx, uint32_t seq);

/* One token into each of n sequences (distinct seq[i]), no head:
 * dd.feed (bend/Dense/Decode.bend:548-551) for n sequences at once. One
 * sequence in ANA_EXACT_FP32 runs as one persistent launch where the device
 * and the model allow it, to the same bits as the step's kernels. A launch
 * whose waits pass their limit is undone and the token fed by the kernels,
 * which then take the context's later feeds too: ana_feed never returns
 * ANA_ETIME. */
int ana_feed(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, const uint32_t* pos,
             const uint32_t* tok);

/* len tokens into one sequence from pos, a chunk at a time: dd.feeds
 * (bend/Dense/Decode.bend:637-639). In ANA_EXACT_FP32 the states and the
 * residual row are bit-identical to len ana_feed calls. */
int ana_feeds(struct ana_ctx* ctx, uint32_t seq, uint32_t pos, const uint32_t* toks, uint32_t len);

/* dd.feeds for n sequences at once (distinct seq[i]): sequence seq[i] takes
 * len[i] tokens from pos[i]; toks holds the sequences' tokens one after
 * another. A chunk step feeds every sequence's next chunk together, so the
 * products run over all their rows at once (the reference prefills one
 * sequence per process and has no counterpart; its meaning is n ana_feeds
 * calls, and in ANA_EXACT_FP32 the states are bit-identical to them). */
int ana_feeds_n(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, const uint32_t* pos,
                const uint32_t* len, const uint32_t* toks);

/* Window scoring, Evaluate.bend's window.go (bend/Evaluate.bend:33-44) for
 * n sequences: sequence seq[i] feeds its first len[i] - 1 tokens from
 * pos[i] (as ana_feeds_n would), and after each fed token t, ce receives
 * G.lse(logits) - logits[token t + 1] (bend/Train/Grad.bend:795-797: the
 * tree max, plus F32.log of the tree sum of F32.exp(x - max)). ce holds
 * len[i] - 1 values per sequence, one sequence after another. In
 * ANA_EXACT_FP32 each value has the bits of ana_feed + ana_logits + that
 * lse; the fast modes are within their tolerance. The caller forms window
 * means and bits per byte from them (window.mean, report). */
int ana_score_n(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, const uint32_t* pos,
                const uint32_t* len, const uint32_t* toks, float* ce);

/* The head on each listed sequence's last fed token: n x vocab floats,
 * dd.logits (bend/Dense/Decode.bend:641-646). */
int ana_logits(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, float* out);

/* The model's own probability of a token after each listed sequence's
 * last fed token, and its likeliest rival: dc.prob.of
 * (bend/Decode.bend:199-202, the prob= of SAMPLE_STATS's lines,
 * bend/Generate.bend:40-49) and al.stat (bend/Agent/Loop.bend:284-288, the
 * agent's pass along a failed term). The head runs on the device and only
 * the three answers come back: with m the logits' tree max and z the tree
 * sum of F32.exp(x - m), prob[i] = exp(l[tok[i]] - m) / z; alt[i] is
 * Sample.argmax of the logits with l[tok[i]] set to -3e38, and alt_prob[i]
 * its probability the same way. Bit-exact with those formulas on the
 * reference's logits in ANA_EXACT_FP32. */
int ana_stats(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, const uint32_t* tok, float* prob,
              uint32_t* alt, float* alt_prob);

/* After each listed sequence's last fed token, what ana_row_logprobs gives of
 * the head's logits: the log probability and rank of tok[i] (tok NULL:
 * neither is written), the entropy, and the `top` (0 .. 64) likeliest tokens
 * with their log probabilities ([n][top]), ties to the lower index. No
 * counterpart in the reference (ana_stats gives its one rival); the sums are
 * f32 in every mode. */
int ana_logprobs(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, const uint32_t* tok, uint32_t top,
                 float* lp, float* ent, uint32_t* rank, uint32_t* top_tok, float* top_lp);

/* ana_score_n's windows with the same results in place of its summands:
 * after each fed token t, token t + 1's log probability and rank, the
 * entropy and the alternatives; len[i] - 1 of each a sequence, one sequence
 * after another. */
int ana_score_logprobs_n(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, const uint32_t* pos,
                         const uint32_t* len, const uint32_t* toks, uint32_t top, float* lp, float* ent,
                         uint32_t* rank, uint32_t* top_tok, float* top_lp);

/* Greedy's pick on the device: dd.top (bend/Dense/Decode.bend:475-484,
 * 648-660), the least index reaching the maximum logit; vocab when no logit
 * does (a NaN maximum), where the caller falls back to ana_pick. */
int ana_top(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, uint32_t* tok);

/* S.pick (bend/Sample.bend:246-254) on the device: greedy (tree argmax)
 * when temperature <= 0, else temperature, top-k and top-p by 40-step
 * bisections and one inverse-CDF draw in tree order. rng holds n x 4 u64
 * xoshiro words (bend/Sample.bend:49-93), advanced in place by one draw for
 * each sampled sequence (untouched when greedy). */
int ana_pick(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, const ana_sampling* s,
             uint64_t* rng, uint32_t* tok);

/* Rng.seeded (bend/Sample.bend:68-93): the 4 words for a seed. */
void ana_rng_seeded(uint64_t seed, uint64_t rng[4]);

/* The token loop of bend/Generate.bend:39-51 on the device, for n sequences
 * at once: steps times, feed each sequence's current token at its position,
 * run the head and pick (greedy when s is NULL or temperature <= 0), and
 * feed the pick back. tok[i] is sequence i's first token at pos[i]; out
 * receives n x steps picks (row i = sequence i). EOS does not stop the loop;
 * a caller wanting Generate's stop truncates each row after its first 1.
 * rng as ana_pick (NULL when greedy). One greedy sequence (n = 1) runs as
 * one persistent launch a call in every mode where the device and the model
 * allow it (the environment's ANA_PERSIST=0 keeps it on the step graphs);
 * its results are those of the graphs (bit for bit in ANA_EXACT_FP32), and
 * it can fail with ANA_ETIME (after 2 s in one wait; ANA_PERSIST_MS in the
 * environment sets another limit, in milliseconds). */
int ana_generate(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, const uint32_t* pos,
                 const uint32_t* tok, uint32_t steps, const ana_sampling* s, uint64_t* rng,
                 uint32_t* out);

/* ana_generate for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * No counterpart in the reference. Same arguments, semantics and results
 * as ana_generate, but the call allocates nothing: it calls no hipMalloc or
 * hipFree, captures no graph and records no timing events (kernels are
 * launched one by one), and its scratch (the rows' step counters and
 * picks) lives in a fixed device array of 2^18 words that each GPU holds
 * until the process ends. A call needs 64 * ceil(n / 64) + 2 * n * steps
 * words of it; larger calls fail with ANA_EINVAL. Every call on one GPU
 * shares that array, whatever the context, so calls on one GPU from several
 * threads run one at a time: each holds a per-device lock from clearing its
 * counters to its final synchronisation. */
int ana_generate_noalloc(struct ana_ctx* ctx, uint32_t n, const uint32_t* seq, const uint32_t* pos,
                         const uint32_t* tok, uint32_t steps, const ana_sampling* s, uint64_t* rng,
                         uint32_t* out);

/* Copy one sequence's state out (for parity checks): layer l's GLA S
 * (heads x hd x hd floats) or K ring then V ring (2 x ctx x d floats; with
 * ANA_KV4 the values that the codes stand for); l ==
 * layers gives the residual row (d floats). n is the float count of out. */
int ana_state(struct ana_ctx* ctx, uint32_t seq, uint32_t layer, float* out, size_t n);

/* Kernel timing (no counterpart in the reference; for benchmarks and
 * profiling). While on, every launch of the listed kinds is bracketed by HIP
 * events on the context's stream and its algorithmic bytes are counted;
 * ana_prof_read sums them since the last ana_prof(ctx, 1). */
#define ANA_K_GEMV 0     /* the layers' matrix-vector products */
#define ANA_K_HEAD 1     /* the LM head's product */
#define ANA_K_ATTN 2     /* softmax attention over the ring */
#define ANA_K_GLA 3      /* the GLA state update and readout */
#define ANA_K_PICK 4     /* greedy pick / sampler */
#define ANA_K_STEP 5     /* whole decode steps in one persistent launch (one greedy
                            sequence, any mode): every kind above at once */
#define ANA_K_KINDS 6
int ana_prof(struct ana_ctx* ctx, int on);
int ana_prof_read(struct ana_ctx* ctx, uint32_t kind, uint64_t* launches, double* ms,
                  double* bytes);

/* Phase stamps of the persistent one-sequence decode kernel (no counterpart
 * in the reference; for profiling the exchange between its workgroups).
 * ana_trace(ctx, steps) with 1 <= steps <= 64 arms it (allocating the
 * stamps' buffer; ANA_EUNSUP where the context has no persistent kernel or
 * more than 32 layers); steps == 0 disarms it. While armed, each persistent
 * launch records its first `steps` steps: per (step, phase, workgroup), four
 * readings of the device's constant-rate clock (100 MHz on gfx950; its low
 * 32 bits, so differences are taken modulo 2^32) taken by the
 * workgroup's first thread: the phase's start, all of its inputs seen, its
 * weights landed in LDS, its outputs published. A step's phases are, per
 * layer, q|k|v(|z), the mix (GLA; or the attention pieces, then their
 * combination), Wo, gate|up and down, then the head and the pick.
 * ana_trace_read copies the last launch's stamps, [steps][phases]
 * [workgroups][4], into out (cap entries) and their extents into dims;
 * with out NULL it gives the extents only. */
int ana_trace(struct ana_ctx* ctx, uint32_t steps);
int ana_trace_read(struct ana_ctx* ctx, uint32_t* out, size_t cap, uint32_t dims[3]);

/* A measurement probe with no counterpart in the reference (no context):
 * the rate of re-reading one zero-filled device buffer of `bytes` (at least
 * 4096, a multiple of 16) `reps` times with a streaming float4 read over
 * 8192 x 256 threads, after one untimed pass, in GB/s (HIP events). Where
 * the buffer fits a cache level (the XCDs' L2s, the Infinity Cache), the
 * rate is that level's; past it, HBM's. It allocates and frees its buffer. */
int ana_probe_reread(int device, uint64_t bytes, uint32_t reps, double* gbs);

/* The last error on ctx, or of the last failed ana_open when ctx is NULL. */
const char* ana_error(const struct ana_ctx* ctx);

void ana_close(struct ana_ctx* ctx);

typedef struct ana_ctx ana_ctx;

/* ---- the FTC2 manifest (bend/Checkpoint.bend:19-136) ----
 * Every field of Load.header's Manifest; the doubles as the reference forms
 * them in F32 (Load.double). Strings are UTF-8, NUL-terminated, cut at
 * ANA_MANIFEST_STR - 1 bytes. tokenizer_id names the tokenizer a caller
 * finds by identity (dc.tok.of). */
#define ANA_MANIFEST_STR 1024
typedef struct ana_manifest {
  uint32_t version;
  ana_config cfg;
  uint32_t count;                       /* the parameter count field */
  char layout[ANA_MANIFEST_STR];
  uint32_t layout_version;
  float lr, beta1, beta2, eps, weight_decay;   /* AdamW */
  uint32_t warmup, total_steps;
  uint32_t has_muon;
  float muon;
  char model_id[ANA_MANIFEST_STR], tokenizer_id[ANA_MANIFEST_STR], dataset_id[ANA_MANIFEST_STR];
  float clip;
  uint32_t numerics;
} ana_manifest;

/* Load.header's manifest of an FTC2 file, without Manifest.problem's
 * verdict (ana_open applies that): ANA_ECKPT and ana_error(NULL) on an
 * unreadable file, a wrong magic or a short header. */
int ana_manifest_read(const char* path, ana_manifest* out);

/* ---- operators on device memory ----
 * The kernels of a context's ANA_KV4 rings and of its log probabilities, for
 * programs that hold their own tensors on the device (no counterpart in the
 * reference). Unlike the calls on a context they take device pointers and
 * queue their work on `stream` (a hipStream_t; NULL the device's default
 * stream) without waiting for it: the memory stays the caller's, and stays
 * valid until the stream has passed the call. They allocate nothing,
 * synchronise nothing and can be captured into a graph. A call that needs a
 * workspace takes it from the caller; two calls that may run at the same
 * time need two. `device` is the pointers' device; the calling thread's
 * current device is left as it was. Any thread may call them; after a
 * nonzero answer ana_error(NULL) holds the calling thread's message.
 *
 * Tensors are [rows][heads][hd], the strides between rows and between heads
 * counted in elements, the last axis consecutive. Strides of hd elements or
 * more, in any order; a tensor whose rows or heads share elements (a
 * broadcast one, stride 0) is refused with ANA_EINVAL, an input as an output.
 * Addresses and strides on 16 bytes are read and written fastest. */
#define ANA_T_F32 0
#define ANA_T_BF16 1
#define ANA_T_F16 2

/* Keys and values of `seqs` sequences in 4 bits: rings of `slots` positions
 * (position p in slot p mod slots), `heads` key heads of hd = 32, 64 or 128
 * values. MXFP4: a value is an E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4 or 6 and a
 * sign), and 32 values next to each other along a head share a scale byte b,
 * 2^(b - 127). A block with largest magnitude a takes the least scale of
 * 2^-125 .. 2^125 with a <= 7 scale (past that the largest, and values past
 * its 6 are that), a value the nearest code, ties to the even one; a block
 * with an infinity or a NaN in it becomes NaN (b = 255). So stored scale bytes
 * are 2 .. 252 and 255, and every value is a bfloat16; a cache from elsewhere
 * keeps to them (zeros stand for slots that hold nothing).
 * data holds ana_kv4_bytes bytes on a 16-byte border, for each sequence and
 * head ceil(slots / 32) records of 32 slots and 34 hd bytes:
 *   keys    [4 j][16 m][2 h][hd / 8]  slot 16 h + m, dims j hd / 4 ..
 *   values  [4 j][16 m][8 e][hd / 32] slot 16 (e / 4) + 4 j + e % 4, dims m hd / 16 ..
 *   key scales   [hd / 32][16 m][2 h]
 *   value scales [hd / 32][4 j][8 e]
 * two codes a byte, the even dimension's in the low half. */
typedef struct {
  void* data;
  int device;
  uint32_t seqs, slots, heads, hd;
} ana_kv4;

/* The rows of a call, in device memory: sequence i of n has its place
 * seq[i] in the cache (seq NULL: i) and rows off[i] .. off[i + 1] - 1 of the
 * tensors, at positions pos[i] and on (off NULL: row i alone, rows == n). A
 * place outside 0 .. seqs - 1, or a first position outside 0 .. 2^31 - 1, is
 * none (-1 in a padded batch): nothing is stored for the sequence, and its
 * outputs are zeros. off does not go down, and ends at `rows` at most; rows
 * before off[0] and from off[n] on are not read, and their outputs are left
 * as they were. Up to 2^26 rows and sequences. */
typedef struct {
  uint32_t n, rows;
  const uint32_t *seq, *pos, *off;
} ana_kv4_rows;

/* a tensor: its address, and the elements from row to row and head to head */
typedef struct {
  void* p;
  uint64_t row, head;
} ana_mat;

/* the bytes of a cache; 0 where its shape is refused */
uint64_t ana_kv4_bytes(uint32_t seqs, uint32_t slots, uint32_t heads, uint32_t hd);

/* Keys k and values v (of ANA_T_ type `type`) into the cache. Of a
 * sequence with more rows than slots only the last `slots` are stored; of a
 * sequence that the call lists again, the first listing that has rows and a
 * place is. */
int ana_kv4_write(const ana_kv4* c, const ana_kv4_rows* r, int type, const ana_mat* k, const ana_mat* v,
                  void* stream);

/* The values that the cache holds at the rows' positions, to k and v. */
int ana_kv4_read(const ana_kv4* c, const ana_kv4_rows* r, int type, const ana_mat* k, const ana_mat* v,
                 void* stream);

/* Softmax attention of query rows [rows][hq][hd] over the cache; query head
 * a reads key head a / (hq / heads). The call's own keys and values have
 * been written. A row at position p, of a sequence whose last row is at P,
 * sees the positions up to p that the ring still holds (those above P -
 * slots): o = sum_j e^(scale q.k_j) v_j over (sum_j e^(scale q.k_j) +
 * e^sink[a]), sink (hq floats) NULL for none; 0 where it sees nothing.
 * What a row does not see, NaN included, does not change it. In f32 the
 * products are exact up to their f32 sums; 16-bit outputs take
 * probabilities to 2^-16, but bf16 ones of a sequence with more than 16 query
 * rows a key head (rows times hq / heads) each rounded to bf16, which adds to
 * an output as much again as its own rounding: a call's rows decide which. `live`, where not 0, is the most positions a
 * sequence holds after the call, as far as the caller knows: it only
 * chooses how the work is split. o may be q itself (the same address and
 * strides). ws: ana_kv4_attend_ws bytes of workspace for the same arguments,
 * on a 16-byte border. Up to 2^31 - 1 rows times hq, and with G = hq / heads
 * fewer than 2^24 of n heads ceil(G / 16), or with off of
 * (ceil(rows G / 64) + n) heads. */
int ana_kv4_attend(const ana_kv4* c, const ana_kv4_rows* r, int type, const ana_mat* q, uint32_t hq, float scale,
                   const float* sink, const ana_mat* o, uint64_t live, void* ws, uint64_t ws_bytes, void* stream);
uint64_t ana_kv4_attend_ws(const ana_kv4* c, const ana_kv4_rows* r, uint32_t hq, uint64_t live);

/* ana_kv4_attend where groups of rows also see a prefix that they have in
 * common (the prompt of many answers, a system prompt), held and read once for
 * all: group i of pre->n has rows pre->off[i] .. pre->off[i + 1] - 1 of the
 * tensors (off NULL: n is 1, and all rows are its), and each of them sees the
 * first pre->pos[i] positions of place pre->seq[i] (NULL: i) of the cache pc,
 * those of them that its ring holds, besides its own sequence's in c. One
 * softmax goes over both. pre->rows == r->rows. Rows of no group, a group
 * whose place is none, and one whose length is 0 or not below 2^31 see their
 * own positions alone; a sequence whose place in c is none has zeros. pc has
 * c's heads and head size, and may be c. pre->off as r->off; up to 2^26
 * groups. plive as live, of the prefixes. bf16 outputs' probabilities over a
 * prefix are taken to 2^-11, or 2^-32 of the largest one, over the own positions
 * as there. Scores are to be below 2^29 in size. ws: ana_kv4_attend_shared_ws bytes for the same arguments, on a
 * 16-byte border. */
int ana_kv4_attend_shared(const ana_kv4* c, const ana_kv4_rows* r, const ana_kv4* pc, const ana_kv4_rows* pre, int type,
                          const ana_mat* q, uint32_t hq, float scale, const float* sink, const ana_mat* o, uint64_t live,
                          uint64_t plive, void* ws, uint64_t ws_bytes, void* stream);
uint64_t ana_kv4_attend_shared_ws(const ana_kv4* c, const ana_kv4_rows* r, const ana_kv4* pc, const ana_kv4_rows* pre,
                                  uint32_t hq, uint64_t live, uint64_t plive);

/* How a head's values turn with its row's position: of the first `rot` (a
 * multiple of 16, hd at most; 0: none) the pairs (i, i + rot / 2), or with
 * near (2 i, 2 i + 1), by position times freq[i] (rot / 2 floats), in radians:
 * (a, b) becomes (a cos t - b sin t, b cos t + a sin t). gq and gk (hd
 * floats; NULL: no norm): before that each head of q, of k, is RMS-normed, x /
 * sqrt(mean x^2 + eps) * (1 + g), as a context's qk-norm. */
typedef struct {
  const float* freq;
  uint32_t rot;
  int near;
  const float *gq, *gk;
  float eps;
} ana_rope;

/* Queries q [rows][hq][hd] and keys k [rows][hk][hd], normed and turned, to qo
 * and ko (which may be q and k themselves: the same address and strides; else
 * they lie apart from them), in one pass; hd a multiple of 16 up to 256, either
 * of hq and hk may be 0 (its tensors are not looked at). r->seq is not read. A
 * sequence whose first position is none has zeros; rows of no sequence are left
 * as they were. Angles are right to f32's last bits at every position for
 * frequencies up to 256 in size. A norm's squares are summed in f32: a head where
 * they pass its largest number (values next to 2^64) comes out as zeros. Up to
 * 2^26 rows and sequences. */
int ana_qk_rope(int device, uint32_t hd, const ana_kv4_rows* r, int type, const ana_rope* f, uint32_t hq, const ana_mat* q,
                const ana_mat* qo, uint32_t hk, const ana_mat* k, const ana_mat* ko, void* stream);

/* How tokens are drawn: one setting for every row, or (arrays of n, where not
 * NULL) each row its own. temperature 0: the likeliest token. top_k: the first
 * k tokens by value, then lower index (0, or the vocabulary and more: all).
 * top_p: of these, the fewest first ones whose mass is top_p of theirs or more
 * (1: all). min_p: of these, the ones of min_p or more of the likeliest one's
 * probability (0: all). The first is always kept. In the arrays a temperature
 * that is not above 0 is 0, a top_p of 1 or more (or NaN) is 1, of 0 or less
 * 0, a min_p above 1 is 1 and one not above 0 (or NaN) is 0. */
typedef struct {
  float temperature, top_p, min_p;
  uint32_t top_k;
  const float *temperatures, *top_ps, *min_ps;
  const uint32_t* top_ks;
} ana_draw;

/* A token of each of n rows of `vocab` logits (of ANA_T_ type `type`, ld
 * elements from row to row, vocab or more) from a given number u[i], 0 <= u <
 * 1 (others count as the nearest): tok[i], the first in the order of value,
 * then lower index, at which the running probability of what is kept, e^(x /
 * temperature) over its sum, passes u; and lp[i], the log of its own (0 for a
 * temperature of 0). Probabilities below 2^-43 of the likeliest one's are 0, and
 * the sums are exact in units of 2^-42 of it, so that a row's token does not
 * depend on the other rows or on how the work is split. -inf and NaN are never
 * drawn; tokens at +inf are alike and have all; with no number above -inf tok
 * is 2^32 - 1 and lp NaN. Finite logits are to be within 2^128 of each other. Up to 2^21 logits and 2^22 - 1 rows. ws:
 * ana_row_sample_ws bytes, on an 8-byte border (0 bytes but for few long rows). */
int ana_row_sample(int device, int type, const void* logits, uint64_t ld, uint32_t n, uint32_t vocab, const float* u,
                   const ana_draw* s, uint32_t* tok, float* lp, void* ws, uint64_t ws_bytes, void* stream);
uint64_t ana_row_sample_ws(uint32_t n, uint32_t vocab);

/* Of n rows of `vocab` logits (of ANA_T_ type `type`, ld elements from row
 * to row, vocab or more), in one read of them: lp[i], the log probability of the given
 * token tok[i] (NaN for a token outside the vocabulary), and rank[i], the
 * tokens before it in the order of value, then of lower index (0: it is the
 * greedy pick; 2^32 - 1 outside the vocabulary); tok NULL: neither is
 * written. ent[i], the entropy in nats; top_tok and top_lp [n][top], the
 * first `top` (0 .. 64, at most vocab) tokens in that order and their log
 * probabilities. A logit of -inf has probability 0; in a row with nothing
 * else every log probability is -inf and the entropy 0. NaN comes after
 * every number in the order; a NaN or +inf in a row makes its log
 * probabilities and entropy NaN. Sums are f32. vocab up to 2^21; up to
 * 2^22 - 1 rows of 32768 logits (2^16 - 1 of the longest). ws:
 * ana_row_logprobs_ws bytes, on a 4-byte border. */
int ana_row_logprobs(int device, int type, const void* logits, uint64_t ld, uint32_t n, uint32_t vocab,
                     const uint32_t* tok, uint32_t top, float* lp, float* ent, uint32_t* rank, uint32_t* top_tok,
                     float* top_lp, void* ws, uint64_t ws_bytes, void* stream);
uint64_t ana_row_logprobs_ws(uint32_t n, uint32_t vocab, uint32_t top);

/* ---- the fast BPE tokenizer (bend/Tokenizer.bend), host side ----
 * Tokens: 0 = BOS, 1 = EOS, 2..257 the bytes, then one per merge in id
 * order. The GPU path sees ids only; these serve the prompts and the
 * outputs around it (dc.tok.of, Bpe.encode, Bpe.decode). */
struct ana_bpe;

/* Bpe.parse of a .bpe artifact ("BPE <vocab> [v2]", then "a b new" rows,
 * ids contiguous from 258): ANA_ETOK when unreadable or rejected. */
int ana_bpe_open(const char* path, struct ana_bpe** out);
/* the byte tokenizer (no merges, V2 rule; dc.tok.btc, bend/Decode.bend:264-268) */
int ana_bpe_bytes(struct ana_bpe** out);
void ana_bpe_close(struct ana_bpe* t);
uint32_t ana_bpe_vocab(const struct ana_bpe* t);
/* Bpe.identity (bend/Tokenizer.bend:330-336): "fastbpe-word-v1:bos=0:eos=1:
 * bytes=2..257:pretoken=<rule>:vocab=<v>:sha256=<digest of the merges>",
 * NUL-terminated into buf (ANA_EINVAL if cap is too small) */
int ana_bpe_identity(const struct ana_bpe* t, char* buf, size_t cap);
/* Bpe.encode (bend/Tokenizer.bend:631-634): pretokenize, then BPE per
 * word; *nids receives the count, ids the ids when cap holds them
 * (ANA_EINVAL otherwise, *nids still set) */
int ana_bpe_encode(const struct ana_bpe* t, const uint8_t* bytes, size_t n, uint32_t* ids, size_t cap,
                   size_t* nids);
/* Bpe.decode of each id, concatenated (BOS and EOS give no bytes) */
int ana_bpe_decode(const struct ana_bpe* t, const uint32_t* ids, size_t n, uint8_t* bytes, size_t cap,
                   size_t* nbytes);
/* H.sha256 (bend/Sha256.bend): 64 lowercase hex digits and a NUL */
int ana_sha256_hex(const uint8_t* bytes, size_t n, char* out65);

#ifdef __cplusplus
}
#endif
#endif
