/*
 * pesti_sampler.h -- C ABI of the B200 (sm_100a) token sampler.
 *
 * Drop-in boundary for the PESTI sampling step
 *   temperature -> softmax -> top-k -> top-p -> inverse-CDF draw
 * that the reference implements in Rust as
 *   pub fn sample(logits: &[f32], config: &SamplingConfig, rng: &mut StdRng) -> u32
 *                                       (llm-runner/src/transformer/sampling.rs:39)
 *   pub fn argmax(logits: &[f32]) -> u32 (llm-runner/src/transformer/sampling.rs:115)
 * called from LlamaModel::generate (llm-runner/src/transformer/model.rs:517-521) and
 * CpuModel::run (llm-runner/src/model.rs:823-828).  The reference has no GPU
 * sampler; this library takes the place of the stubbed GPU crate
 * (cuda-oxide/src/main.rs:1-3) and is the sampling entry the kernel layer
 * (llm-runner/src/kernel/mod.rs) lacks.
 *
 * Results are those of the reference algorithm, bit for bit, given the same
 * per-row uniform draw u (the value `rng.random::<f32>()` returns at
 * sampling.rs:98) and given exp correctly rounded (the reference calls the
 * platform expf, which differs from the correctly rounded value by one ulp on
 * about 6e-4 of its inputs).
 *
 * Conventions (mirroring the reference kernel layer):
 *  - every call returns 0 on success or a negative PESTI_E_* code; the message
 *    of the last failure on the calling thread is pesti_last_error();
 *  - device pointers are plain addresses (RawHandle(u64) in
 *    llm-runner/src/kernel/memory.rs:22); the caller owns every buffer;
 *  - batch calls are stream-ordered and never synchronize the host;
 *  - there is no CPU fallback: without a usable sm_100 device the calls fail.
 */
#ifndef PESTI_SAMPLER_H
#define PESTI_SAMPLER_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PESTI_OK 0
#define PESTI_E_INVALID_ARG (-1)
#define PESTI_E_CUDA (-2)
#define PESTI_E_NCCL (-3)
#define PESTI_E_TIMEOUT (-4)
#define PESTI_E_UNSUPPORTED (-5)
#define PESTI_E_NO_DEVICE (-6)

/* Logit element types.  BF16 and F16 logits are widened to f32 exactly, so
 * results are those of the reference on the widened values (a caller of the
 * reference's &[f32] API would widen them the same way).
 *
 * FP8_E4M3 (OCP E4M3FN: no infinities, S.1111.111 is NaN) and FP8_E5M2 (IEEE
 * layout with infinities and NaNs), the float8 crate's F8E4M3 and F8E5M2,
 * are taken by pesti_sample_batch and pesti_argmax_batch only.  Every value
 * of both formats is an f16 value: the call first widens the [B, V] logits
 * exactly into f16 in the handle's workspace (2 bytes per logit, on the
 * call's stream), then samples those.  The other entry points refuse them
 * with PESTI_E_INVALID_ARG. */
typedef enum { PESTI_F32 = 0, PESTI_BF16 = 1, PESTI_F16 = 2, PESTI_FP8_E4M3 = 3, PESTI_FP8_E5M2 = 4 } pesti_dtype;

/* Per-row sampling parameters: SamplingConfig (sampling.rs:12-21) without the
 * seed, which sample() never reads. */
typedef struct {
  float temperature; /* sampling.rs:14; > 0 scales the logits, otherwise none */
  float top_p;       /* sampling.rs:16; used only when top_k == 0 (sampling.rs:66) */
  uint32_t top_k;    /* sampling.rs:18; 0 = disabled */
  uint32_t flags;    /* PESTI_FLAG_* */
} pesti_sampling_params;

/* Apply the caller branch of generate()/run(): temperature == 0.0 -> argmax
 * (transformer/model.rs:517-521, model.rs:823-828).  Without it a zero
 * temperature means "no scaling", as in sample() itself (sampling.rs:43). */
#define PESTI_FLAG_GREEDY_IF_ZERO_T 1u
/* argmax ties go to the lowest index.  Default: the last index, as
 * Iterator::max_by returns (sampling.rs:115-122). */
#define PESTI_FLAG_ARGMAX_FIRST 2u

typedef struct pesti_sampler pesti_sampler;

/* Creates a sampler bound to CUDA device `device`: events, a workspace that
 * grows on demand, and a private stream for pesti_sample_row_host.  Replaces
 * the context set-up of CudaRuntime::new (llm-runner/src/cuda_runtime.rs:92-176)
 * for this path.  A handle may be used from one thread at a time. */
int pesti_sampler_create(int device, pesti_sampler** out);
void pesti_sampler_destroy(pesti_sampler* s);

/*
 * Batched sample over row-major logits [B, ld] (first V columns of each row),
 * dtype F32, BF16 or F16, on device memory.  Replaces, per row, the call
 *   generate():  if T == 0 { argmax(row) } else { sample(row, cfg, rng) }
 * (model.rs:517-521) when params carry PESTI_FLAG_GREEDY_IF_ZERO_T, and
 * sample(row, cfg, rng) (sampling.rs:39) otherwise.
 *
 *  params          host pointer: B entries if params_per_row, else 1 entry.
 *                  When params_on_device != 0 it is a device pointer instead.
 *  d_u             device [B] f32: the draw r of each row (sampling.rs:98).
 *  d_out_tokens    device [B] u32.
 *  d_kept_p/idx    optional device [B, kept_width]: the first kept_width
 *                  entries of each row's kept list (the (probability, index)
 *                  pairs left after top-k / top-p, sampling.rs:56-78), padded
 *                  with 0 / 0xffffffff.  Either may be NULL.
 *  d_kept_count    optional device [B] i64: length of each kept list (0 for
 *                  greedy rows).
 *  stream          cudaStream_t; NULL is the legacy default stream, as for
 *                  CUDA's own calls (PyTorch's default stream is that stream).
 */
int pesti_sample_batch(pesti_sampler* s, const void* d_logits, pesti_dtype dtype, int64_t B,
                       int64_t V, int64_t ld, const pesti_sampling_params* params,
                       int params_per_row, int params_on_device, const float* d_u,
                       uint32_t* d_out_tokens, float* d_kept_p, uint32_t* d_kept_idx,
                       int64_t kept_width, int64_t* d_kept_count, void* stream);

/* Batched argmax (sampling.rs:115-122, last of equal maxima; NaN handled as
 * Iterator::max_by does) over device logits.  flags: PESTI_FLAG_ARGMAX_FIRST. */
int pesti_argmax_batch(pesti_sampler* s, const void* d_logits, pesti_dtype dtype, int64_t B,
                       int64_t V, int64_t ld, uint32_t flags, uint32_t* d_out_tokens,
                       void* stream);

/* One row from HOST memory, synchronous: the drop-in for
 * sample(&logits, &cfg, &mut rng) (sampling.rs:39) with r drawn by the caller;
 * honours PESTI_FLAG_GREEDY_IF_ZERO_T like the batch call. */
int pesti_sample_row_host(pesti_sampler* s, const float* h_logits, int64_t V,
                          const pesti_sampling_params* params, float u, uint32_t* out_token);

/*
 * No counterpart in the reference.
 *
 * pesti_sample_batch without a handle and without any device allocation, for
 * callers that cannot allocate device memory while they sample: a decode loop
 * that has handed the rest of HBM to its KV-cache page pool, where a
 * cudaMalloc would fail, or one that must not stall its other streams, which
 * cudaMalloc and cudaFree do (pesti_sample_batch grows its workspace with them
 * whenever it meets a larger batch).
 *
 * Arguments and results are those of pesti_sample_batch.  It runs on the
 * calling thread's current device; stream NULL is the legacy default stream.
 * Its only device memory besides the caller's buffers is one static array of
 * PESTI_NOALLOC_SCRATCH_BYTES on each device, shared by every call:
 *  - a call that needs more scratch than the array holds fails with
 *    PESTI_E_INVALID_ARG and launches nothing.  A call needs about 16 bytes
 *    per logit (B*V) when every row is greedy or uses top_k <= 1024, 36 bytes
 *    per logit otherwise (top-p, no filter, larger top_k, or params on the
 *    device), plus host per-row params and at most about 0.3 MB per row:
 *    8 rows of V = 128256 with top-p need about 37 MB;
 *  - calls whose GPU work overlaps (on streams with no order between them)
 *    race on the array: order them on one stream;
 *  - host per-row params are copied into the array on the stream.  From
 *    ordinary (pageable) host memory the copy has taken the values when the
 *    call returns, so the caller may reuse them at once.  From page-locked
 *    host memory (cudaMallocHost, cudaHostRegister, torch's pin_memory) the
 *    copy runs later, when the stream reaches it: the caller must leave those
 *    params unchanged until then (synchronize the stream, or wait on an event
 *    recorded after the call, before rewriting them);
 *  - a single params entry on the device is read back with a stream
 *    synchronization, as in pesti_sample_batch.
 * The first call on a device does the set-up: it looks the array up with
 * cudaGetSymbolAddress, which loads it onto that device.  Make that first call
 * before any stream capture.  No call allocates: none calls cudaMalloc,
 * cudaFree or an allocating library routine.
 */
#define PESTI_NOALLOC_SCRATCH_BYTES (64ull << 20)
int pesti_sample_batch_noalloc(const void* d_logits, pesti_dtype dtype, int64_t B, int64_t V,
                               int64_t ld, const pesti_sampling_params* params,
                               int params_per_row, int params_on_device, const float* d_u,
                               uint32_t* d_out_tokens, float* d_kept_p, uint32_t* d_kept_idx,
                               int64_t kept_width, int64_t* d_kept_count, void* stream);

/*
 * No counterpart in the reference (it has no multi-GPU path).
 *
 * Vocabulary-sharded sampling: each of the communicator's ranks holds one
 * contiguous column range of every row, all ranges V_shard wide and in rank
 * order (rank r holds columns [r*V_shard, (r+1)*V_shard) of rows that are
 * world*V_shard long).  Every rank calls pesti_sample_batch_sharded with the
 * same B, V_shard, params and u (the draws of all B rows), its own shard as
 * d_logits [B, ld], and receives the tokens and kept lists of ALL B rows.
 * Results are those of pesti_sample_batch on the whole rows, bit for bit.
 *
 * Top-k rows (1 <= top_k <= 256) and greedy rows are sampled without moving
 * logits: three NCCL all-gathers of per-row summaries (a few hundred bytes
 * per row and shard).  Other rows (top-p, no filter, larger top_k, NaN, and
 * the rare row the sharded algorithm cannot settle) take a gathered path:
 * their shards are all-gathered into whole rows on every rank and sampled
 * there.  The call synchronizes the stream once, to learn which rows those
 * are.
 *
 * A communicator is made once per rank: one rank calls pesti_comm_id, the
 * caller broadcasts its PESTI_COMM_ID_BYTES bytes to the others, and every
 * rank calls pesti_comm_create with them (ncclGetUniqueId /
 * ncclCommInitRank; NCCL is loaded from libnccl.so.2 on first use).  The
 * sampler and the communicator must be on the same device.
 */
typedef struct pesti_comm pesti_comm;
#define PESTI_COMM_ID_BYTES 128
int pesti_comm_id(void* id);
int pesti_comm_create(int world_size, int rank, const void* id, int device, pesti_comm** out);
/*
 * No counterpart in the reference, whose only failure detection is the HTTP
 * health check of a remote runner with a 3 s limit
 * (llm-runner/src/remote_discovery.rs:36-70).
 *
 * pesti_comm_create with a deadline (pesti_comm_create uses 120000 ms).  The
 * communicator is made non-blocking (ncclCommInitRankConfig with blocking = 0)
 * and its set-up is polled with ncclCommGetAsyncError: if every rank has not
 * joined after timeout_ms, the set-up is aborted (ncclCommAbort) and the call
 * returns PESTI_E_TIMEOUT, so a rank that exits or never starts does not hang
 * the others.  The same deadline bounds, on the host, each
 * pesti_sample_batch_sharded call's exchanges: a call whose all-gathers do not
 * complete within timeout_ms of its start, or that reports an NCCL error,
 * aborts the communicator and returns PESTI_E_TIMEOUT (or PESTI_E_NCCL);
 * every later call on that communicator fails with PESTI_E_NCCL, and
 * pesti_comm_destroy releases it.
 */
int pesti_comm_create_timed(int world_size, int rank, const void* id, int device, int timeout_ms, pesti_comm** out);
void pesti_comm_destroy(pesti_comm* c);
int pesti_sample_batch_sharded(pesti_sampler* s, pesti_comm* c, const void* d_logits, pesti_dtype dtype,
                               int64_t B, int64_t V_shard, int64_t ld, const pesti_sampling_params* params,
                               int params_per_row, int params_on_device, const float* d_u,
                               uint32_t* d_out_tokens, float* d_kept_p, uint32_t* d_kept_idx,
                               int64_t kept_width, int64_t* d_kept_count, void* stream);

/*
 * No counterpart in the reference, whose draw comes from StdRng on the host
 * (sampling.rs:98) once per sample() call.
 *
 * Per-row draws on the device, for a decode loop that keeps its generators
 * on the GPU: no draw crosses from the host each step, and the draws feed
 * d_u of the batch calls directly.  Each row has its own PCG32 generator
 * (O'Neill 2014, XSH-RR 64->32) in d_state: [B][2] u64, state then
 * increment, owned by the caller.
 *  - pesti_pcg32_seed: row b's generator is the one seeded with `seed` on
 *    stream first_stream + b;
 *  - pesti_pcg32_draw: d_u[b] = (next_u32 >> 8) * 2^-24 (the [0, 1) 24-bit
 *    grid of the reference's f32 draw), and row b's generator advances.
 * Both are stream-ordered (NULL: the legacy default stream) and allocate
 * nothing.
 */
int pesti_pcg32_seed(uint64_t* d_state, int64_t B, uint64_t seed, uint64_t first_stream, void* stream);
int pesti_pcg32_draw(uint64_t* d_state, int64_t B, float* d_u, void* stream);

/*
 * The loop control of generate() (transformer/model.rs:508-531: stop tokens,
 * the max_tokens bound, pos >= max_seq_len) on the device, for B sequences
 * decoded together.  Called after each step's sample, it keeps each
 * sequence's tokens on the GPU and feeds the next step's input, so a decode
 * loop reads nothing back per step.  For every row b with d_done[b] == 0,
 * t = d_next[b] (the step's sampled token):
 *  - t in d_stop[0..n_stop): the row finishes (d_done[b] = 1) and t is not
 *    kept (the reference breaks before pushing it);
 *  - otherwise d_generated[b*cap + d_count[b]] = t, d_count[b] += 1 and
 *    d_last[b] = t (the next forward's input token); the row finishes when
 *    d_count[b] reaches max_seq_len (d_done[b] = 3) or max_tokens (2).
 * A row whose d_count[b] is already max_tokens finishes without taking t.
 * Finished rows are left as they are, whatever d_next holds for them.
 * d_active (optional; mapped host memory works) receives the number of rows
 * still running, for a host that checks it now and then instead of
 * synchronising every step.  The caller zeroes d_count and d_done before the
 * first step; cap >= min(max_tokens, max_seq_len).  Stream-ordered (NULL: the
 * legacy default stream); allocates nothing.
 */
int pesti_generate_advance(const uint32_t* d_next, int64_t B, const uint32_t* d_stop, int64_t n_stop,
                           int64_t max_tokens, int64_t max_seq_len, uint32_t* d_generated, int64_t cap,
                           int32_t* d_count, uint8_t* d_done, uint32_t* d_last, int32_t* d_active, void* stream);

/*
 * The sampler chain of PESTI's llama.cpp backend: `build_sampler`
 * (llm-runner/src/llama.rs:465-508) over the fields of its SamplingConfig
 * (llm-runner/src/llama/sampler.rs:19-79), for B rows with one parameter set.
 * The stages run in build_sampler's order and under its gates:
 *   temperature         temperature > 0
 *   top-k               top_k > 0
 *   top-p (min_keep 0)  top_p > 0 (1 or more keeps every candidate)
 *   min-p (min_keep 256) min_p > 0: p >= min_p * p_max, at least 256 kept
 *   top-n-sigma         0 < tfs < 1, n = tfs: logit >= max - n * sigma
 *   typical (min_keep 0) 0 < typical_p < 1
 *   penalties           repetition_penalty != 1, over the last repeat_last_n
 *                       tokens of the row's history (all of it when
 *                       repeat_last_n < 0, none when 0), with
 *                       frequency_penalty and presence_penalty (0.0 in the
 *                       reference)
 * and end with an inverse-CDF draw on d_u[b] over the candidates sorted by
 * logit (the chain as built has no selecting stage; the draw is the Rust
 * sampler's, sampling.rs:97-111).  The stages restate the published filters
 * of llama.cpp, whose sources are not in the reference tree; probabilities
 * are computed in f64.  NaN logits count as -inf.
 *
 * d_history: [B, history_ld] int32 token ids (the row's recent tokens, oldest
 * first), d_history_len (optional): [B] counts of valid leading entries
 * (history_ld for every row when NULL); ids outside [0, V) are ignored.  The
 * window (min(repeat_last_n, history_ld), or history_ld) is at most 8192.
 * d_out_kept (optional): [B] candidates left before the draw.
 * Logits: PESTI_F32, PESTI_BF16, PESTI_F16, and the fp8 types (widened to f16
 * in the handle's workspace first).  Scratch: 16 bytes per logit in the
 * handle's workspace.  Stream-ordered; one 1024-thread block per row.
 */
typedef struct {
  float temperature;        /* llama/sampler.rs:33 */
  int32_t top_k;            /* :36 */
  float top_p;              /* :40 */
  float min_p;              /* :44 */
  float tfs;                /* :47, passed to top-n-sigma (llama.rs:488-491) */
  float typical_p;          /* :50 */
  float repetition_penalty; /* :62 */
  int32_t repeat_last_n;    /* :65 */
  float frequency_penalty;  /* 0.0 in build_sampler (llama.rs:502-503) */
  float presence_penalty;   /* 0.0 in build_sampler */
} pesti_llama_chain_params;

int pesti_llama_chain_batch(pesti_sampler* s, const void* d_logits, pesti_dtype dtype, int64_t B, int64_t V,
                            int64_t ld, const pesti_llama_chain_params* params, const int32_t* d_history,
                            const int32_t* d_history_len, int64_t history_ld, const float* d_u,
                            int32_t* d_out_tokens, int32_t* d_out_kept, void* stream);

/*
 * Beam search: the third way to choose tokens beside pesti_sample_batch and
 * pesti_argmax_batch.  No counterpart in the reference, whose generate()
 * (transformer/model.rs:508-531) follows one sequence.
 *
 * G groups (prompts) of W beams each, W <= PESTI_BEAM_MAX_WIDTH.  None of
 * these calls needs a handle or allocates: they run on the calling thread's
 * current device, stream-ordered (NULL: the legacy default stream), in the
 * caller's buffers, and may be captured into a graph.
 *
 * pesti_beam_select: the K best continuations of each group, for logits
 * [G*W, ld] (first V columns of each row; beam w of group g is row g*W + w;
 * F32, BF16 or F16):
 *   score(w, v) = cum[w] + log softmax(x[w])[v]
 *  - scores are compared in 64 bits; within a beam candidates rank by their
 *    logits, equal logits by the lower token id; equal scores of two beams
 *    rank by the lower beam;
 *  - NaN logits count as -inf.  Tokens of probability 0 are never chosen.  In
 *    a row that holds +inf, the +inf entries share its probability equally;
 *  - d_cum: [G, W] f32 scores so far (NULL: all 0).  A beam whose score is
 *    -inf or NaN has no candidates, and its logits are not read (unless d_lse
 *    is given);
 *  - d_done: optional [G] u8; groups with a non-zero entry are not read and
 *    get no candidates;
 *  - d_score, d_token, d_parent: [G, K], best first, K <= PESTI_BEAM_MAX_CAND:
 *    score (f32), token, and the beam (0..W-1) it continues.  Slots without a
 *    candidate hold -inf, -1, -1;
 *  - d_lse: optional [G, W]: log sum exp of each row's logits (-inf for the
 *    rows of finished groups);
 *  - d_ws: device scratch of pesti_beam_select_workspace(...) bytes, 256-byte
 *    aligned, any contents.  Calls whose GPU work may overlap need scratch of
 *    their own.
 * Outputs overlap neither inputs nor one another (d_score may be d_cum if
 * K == W: a group's scores are read before they are written).
 * With W = 1 and no d_cum it gives the K largest log-probabilities of each row
 * (a distillation teacher's list).
 */
#define PESTI_BEAM_MAX_WIDTH 64
#define PESTI_BEAM_MAX_CAND 128
/* Bytes of scratch, or a negative PESTI_E_* code for refused sizes. */
int64_t pesti_beam_select_workspace(pesti_dtype dtype, int64_t G, int64_t W, int64_t V, int64_t K);
int pesti_beam_select(const void* d_logits, pesti_dtype dtype, int64_t G, int64_t W, int64_t V, int64_t ld,
                      const float* d_cum, const uint8_t* d_done, int64_t K, float* d_score, int32_t* d_token,
                      int32_t* d_parent, float* d_lse, void* d_ws, int64_t ws_bytes, void* stream);

/*
 * The loop control of a beam search on the device: pesti_generate_advance's
 * counterpart for beams.  The state of G groups of W beams is a set of the
 * caller's device arrays; pesti_beam_reset fills them for a new search (one
 * live beam per group, score 0).
 *
 * pesti_beam_advance takes one step's candidates (pesti_beam_select's outputs)
 * and, for every group with done == 0, goes through them in rank order:
 *  - a candidate whose token is in d_stop[0..n_stop) ends a hypothesis if it is
 *    among the first W ranks: the tokens of its parent (the stop token is not
 *    kept), with the score s / (count + 1)^length_penalty;
 *  - the first W others become the live beams 0, 1, ...: tokens[w] is the
 *    parent's tokens and the new one, cum[w] the candidate's score, last[w] the
 *    new token, parent[w] its parent.  Beams left over are dead: cum -inf,
 *    parent -1, the rest as it was;
 *  - padding (token or parent -1, a parent outside [0, W)) is passed over; a
 *    dead parent (which pesti_beam_select never names) is taken with the tokens
 *    that its row holds.
 * Ended hypotheses go to the group's pool of the W best: a full pool's lowest
 * score (of equal ones the highest slot) gives way to a higher one.  count
 * grows by 1.  Then the group finishes:
 *  - when count reaches min(max_tokens, max_seq_len): the live beams go to the
 *    pool with cum / count^length_penalty; done = 3 if count is max_seq_len,
 *    else 2 (a group that is there before the step, as with a limit of 0, ends
 *    with the same codes and nothing more);
 *  - without a live beam: done = 1;
 *  - with a full pool, if early_stop is set or no live beam can still reach the
 *    pool's lowest score (the larger of best / (count + 1)^length_penalty and
 *    best / limit^length_penalty is no higher): done = 1.
 * Groups that are done keep their state; their parent entries become -1.
 * Scores are divided in 64 bits and held in f32.
 */
typedef struct {
  float* cum;          /* [G, W] scores of the live beams */
  int32_t* last;       /* [G, W] the next step's input tokens */
  int32_t* parent;     /* [G, W] for pesti_beam_reorder; -1: the beam stays */
  int32_t* tokens;     /* [G, W, cap] tokens of the live beams */
  int32_t* count;      /* [G] steps taken: the length of every live beam */
  uint8_t* done;       /* [G] */
  int32_t* fin_tokens; /* [G, W, cap] the pool */
  int32_t* fin_len;    /* [G, W] */
  float* fin_score;    /* [G, W] -inf in empty slots */
  int32_t* fin_count;  /* [G] */
  int64_t cap;         /* >= min(max_tokens, max_seq_len) */
} pesti_beam_state;
typedef struct {
  int64_t max_tokens;
  int64_t max_seq_len;
  double length_penalty;
  int32_t early_stop;
} pesti_beam_limits;
int pesti_beam_reset(const pesti_beam_state* state, int64_t G, int64_t W, void* stream);
int pesti_beam_advance(const pesti_beam_state* state, const float* d_score, const int32_t* d_token,
                       const int32_t* d_parent, int64_t G, int64_t W, int64_t K, const uint32_t* d_stop,
                       int64_t n_stop, const pesti_beam_limits* limits, void* stream);

/*
 * Reorders per-beam states (caches, generator states, page tables, histories)
 * after a step: for every group g and beam w, row g*W + w of each state's dst
 * becomes row g*W + d_parent[g*W + w] of its src; a parent outside [0, W) means
 * the beam itself.  src and dst are the same memory with the same strides (in
 * place; beams that stay are not touched) or do not overlap.  States must not
 * share memory with one another (the same dst twice is refused), and no dst
 * with d_parent (refused).
 * A row is `blocks` runs of block_bytes bytes, block_stride bytes apart (for a
 * cache [rows, heads, room, dim] of which `used` positions are filled: blocks =
 * heads, block_bytes = used*dim*esize).  Strides are in bytes and not negative.
 * states: host array, read before the call returns.
 */
typedef struct {
  const void* src;
  void* dst;
  int64_t src_row_stride, dst_row_stride;
  int64_t src_block_stride, dst_block_stride;
  int64_t blocks, block_bytes;
} pesti_beam_rows;
int pesti_beam_reorder(const pesti_beam_rows* states, int64_t n_states, const int32_t* d_parent, int64_t G,
                       int64_t W, void* stream);

/*
 * Distillation from a teacher's top logits: the training side of the kept
 * lists and of pesti_beam_select's log-probabilities.  No counterpart in the
 * reference.
 *
 * Student logits [N, ld] (first V columns; F32, BF16 or F16) at temperature T:
 * p = softmax(x / T) over all V tokens.  The teacher of row n lists k entries
 * (token d_idx[n*idx_ld + j], logit or log-probability t = d_val[n*val_ld + j],
 * val_dtype F32, BF16 or F16), 1 <= k <= PESTI_DISTILL_MAX_TOP; entries whose
 * token is outside [0, V) (padding) are ignored, a token listed more than once
 * counts with the sum of its entries.
 *  - d_teacher_lse NULL: q_j = softmax(t / T) over the listed entries;
 *  - d_teacher_lse [N] f32, the log sum exp of t / T over the teacher's whole
 *    vocabulary: q_j = exp(t_j / T - lse), and the rest q_t = max(0, 1 - sum q)
 *    stands against p_t, the student's mass outside the list.  Where p_t is 0 in
 *    64 bits, q_t counts as 0.
 *   loss = w T^2 [ sum_j q_j log(q_j / p_j) + q_t log(q_t / p_t) ]
 *   grad = d loss / d x (the teacher is a constant)
 * w = d_weight[n] (NULL: 1).  A row of weight 0 (padding) is not read: its loss
 * and gradient are 0.  A row without teacher entries has loss and gradient 0.
 * Where the largest logit is 2^29 T ln 2 or more in magnitude (masks of a
 * type's lowest value), smaller ones count as p = 0.
 * Entries with q = 0 add nothing to the loss.  A student logit of -inf has
 * p = 0 (loss +inf where q > 0); a row of -inf alone has p = 0 everywhere.  NaN
 * and +inf logits make the row's loss and gradient NaN, as NaN in its list does.
 *
 * pesti_distill_topk: d_loss [N] f32.  With d_grad ([N, grad_ld], the logits'
 * type) it writes the gradient of the losses' sum as well; d_grad may be
 * d_logits itself (with grad_ld == ld).  With d_stats ([N,
 * PESTI_DISTILL_STATS(k)] f64) it keeps what pesti_distill_topk_backward needs.
 * Other outputs overlap neither inputs nor one another.  d_ws: device scratch of
 * pesti_distill_topk_workspace(...) bytes, 256-byte aligned, any contents; calls
 * whose GPU work may overlap need scratch of their own.
 * pesti_distill_topk_backward: the gradient of sum_n d_up[n*up_stride] *
 * loss_n (up_stride 0: one value for all rows) from the forward call's inputs
 * and stats.
 * Both run on the calling thread's current device, stream-ordered (NULL: the
 * legacy default stream), allocate nothing, add in a fixed order (the same
 * inputs give the same bits) and may be captured into a graph.
 */
#define PESTI_DISTILL_MAX_TOP 256
#define PESTI_DISTILL_STATS(k) (8 + (k))
/* Bytes of scratch, or a negative PESTI_E_* code for refused sizes. */
int64_t pesti_distill_topk_workspace(pesti_dtype dtype, int64_t N, int64_t V, int64_t k);
int pesti_distill_topk(const void* d_logits, pesti_dtype dtype, int64_t N, int64_t V, int64_t ld,
                       const int32_t* d_idx, int64_t idx_ld, const void* d_val, pesti_dtype val_dtype,
                       int64_t val_ld, int64_t k, const float* d_teacher_lse, const float* d_weight,
                       double temperature, float* d_loss, double* d_stats, void* d_grad, int64_t grad_ld,
                       void* d_ws, int64_t ws_bytes, void* stream);
int pesti_distill_topk_backward(const void* d_logits, pesti_dtype dtype, int64_t N, int64_t V, int64_t ld,
                                const int32_t* d_idx, int64_t idx_ld, const void* d_val, pesti_dtype val_dtype,
                                int64_t val_ld, int64_t k, const float* d_teacher_lse, const float* d_weight,
                                double temperature, const double* d_stats, const float* d_up, int64_t up_stride,
                                void* d_grad, int64_t grad_ld, void* stream);

/*
 * Cross entropy straight from the hidden states that the vocabulary projection
 * (Linear::forward, llm-runner/src/transformer/linear.rs:51-70) makes logits of:
 * the loss of training and of scoring, with its gradients.  The logits z =
 * hidden * head^T are not kept.  No counterpart in the reference.
 *
 * hidden [N, h_ld] (first D columns) and head [V, w_ld] (first D columns), both
 * BF16 or both F16; head 16-byte aligned, w_ld a multiple of 8.  d_target [N]
 * of target_bytes 4 (int32) or 8 (int64).  Rows whose target is outside [0, V)
 * and rows of weight 0 are padding: they are not read and cost nothing, their
 * loss and gradients are 0.  w = d_weight[n] (NULL: 1).
 *   lse  = log sum_v exp z_v
 *   loss = w [ lse - (1 - label_smoothing) z_t - label_smoothing / V sum_v z_v
 *              + z_loss lse^2 ]
 *   G_v  = up w [ (1 + 2 z_loss lse) exp(z_v - lse) - (1 - label_smoothing) [v = t]
 *              - label_smoothing / V ]
 *   grad_hidden = G head,  grad_head = G^T hidden      (in the inputs' type)
 * Products are summed in f32, which cuts off after every 16 of K; logits, those
 * of the loss and the same again for G, in runs of 1024 of K whose sums are
 * rounded.  A row's exponentials are summed without its target's, in f32 over a
 * tile and in 64 bits over the tiles, and -log p_t and G_t are made of that sum:
 * their errors are relative to themselves, where p_t is near 1 too.  The other G
 * are off by up to 2^-22 (2 + |lse|) of themselves besides their logits' errors.
 * G is rounded once to the inputs' type, or (up to 64 rows) held as the sum of two
 * such values (F16: times a power of two that brings its largest value to about
 * 2^14, of the rows whose loss and upstream gradient are finite; what is 2^38 below
 * that is lost).  Logits that are NaN or +inf make their row's loss NaN, and the
 * gradients that the row has part in.
 *
 * pesti_linear_ce: d_loss [N] f32, optionally d_lse [N] f32 (0 for padding) and
 * the gradients of the losses' sum (either may be NULL): d_grad_hidden [N,
 * gh_ld], d_grad_head [V, gw_ld] (16-byte aligned, gw_ld a multiple of 8).
 * pesti_linear_ce_backward: the gradients of sum_n d_up[n*up_stride] * loss_n
 * (up_stride 0: one value for all rows) from the forward call's inputs and lse.
 * G_t of that lse, an f32, is off by up to 2^-22 (1 + |lse|) w up.  The two _nll
 * calls pass on d_nll [N] f32 besides (lse - z_t, 0 for padding; NULL: as without),
 * from which G_t is made as in the gradients of pesti_linear_ce.
 * Outputs overlap neither inputs nor one another.  d_ws: device scratch of
 * pesti_linear_ce_workspace(...) bytes for what the call computes (passes:
 * PESTI_LINEAR_CE_FORWARD, _GRADS, or both), 256-byte aligned, any contents;
 * calls whose GPU work may overlap need scratch of their own.
 * Both run on the calling thread's current device, stream-ordered (NULL: the
 * legacy default stream), allocate nothing, add in a fixed order (the same
 * inputs give the same bits) and may be captured into a graph.  If a wait inside
 * a kernel ever gives up, after about a second, what it leaves unfinished is NaN.
 */
#define PESTI_LINEAR_CE_FORWARD 1
#define PESTI_LINEAR_CE_GRADS 2
/* Bytes of scratch, or a negative PESTI_E_* code for refused sizes. */
int64_t pesti_linear_ce_workspace(pesti_dtype dtype, int64_t N, int64_t V, int64_t D, int passes);
int pesti_linear_ce(const void* d_hidden, pesti_dtype dtype, int64_t N, int64_t D, int64_t h_ld, const void* d_head,
                    int64_t V, int64_t w_ld, const void* d_target, int target_bytes, const float* d_weight,
                    double label_smoothing, double z_loss, float* d_loss, float* d_lse, void* d_grad_hidden,
                    int64_t gh_ld, void* d_grad_head, int64_t gw_ld, void* d_ws, int64_t ws_bytes, void* stream);
int pesti_linear_ce_backward(const void* d_hidden, pesti_dtype dtype, int64_t N, int64_t D, int64_t h_ld,
                             const void* d_head, int64_t V, int64_t w_ld, const void* d_target, int target_bytes,
                             const float* d_weight, double label_smoothing, double z_loss, const float* d_lse,
                             const float* d_up, int64_t up_stride, void* d_grad_hidden, int64_t gh_ld,
                             void* d_grad_head, int64_t gw_ld, void* d_ws, int64_t ws_bytes, void* stream);
int pesti_linear_ce_nll(const void* d_hidden, pesti_dtype dtype, int64_t N, int64_t D, int64_t h_ld,
                        const void* d_head, int64_t V, int64_t w_ld, const void* d_target, int target_bytes,
                        const float* d_weight, double label_smoothing, double z_loss, float* d_loss, float* d_lse,
                        float* d_nll, void* d_grad_hidden, int64_t gh_ld, void* d_grad_head, int64_t gw_ld, void* d_ws,
                        int64_t ws_bytes, void* stream);
int pesti_linear_ce_nll_backward(const void* d_hidden, pesti_dtype dtype, int64_t N, int64_t D, int64_t h_ld,
                                 const void* d_head, int64_t V, int64_t w_ld, const void* d_target, int target_bytes,
                                 const float* d_weight, double label_smoothing, double z_loss, const float* d_lse,
                                 const float* d_nll, const float* d_up, int64_t up_stride, void* d_grad_hidden,
                                 int64_t gh_ld, void* d_grad_head, int64_t gw_ld, void* d_ws, int64_t ws_bytes,
                                 void* stream);

/*
 * The vocabulary projection's weight in 4 bits with group scales, and logits
 * from it for the few rows of a decode step.  No counterpart in the reference
 * (its Linear is f32, llm-runner/src/transformer/linear.rs).
 *
 * Of head [V, ld] (first D columns; F32, BF16 or F16) every `group` (32, 64 or
 * 128) columns of a row share a scale:
 *   s = bf16(-m / 8), m the group's largest value by magnitude, the first of
 *       equal ones;  q = clamp(round-half-even(w / s), -8, 7)  (0 where s is 0)
 * A group with an infinity or a NaN is held as NaN.
 * Layout: tiles of 64 rows and 128 columns.  d_q: 4096 bytes a tile, [ceil(V /
 * 64)][ceil(D / 128)][64 rows][4 chunks][4 words]; d_scale: bf16 [ceil(V / 64)]
 * [ceil(D / 128)][64 rows][128 / group]; both 16-byte aligned.  Chunk c of row r
 * (0 to 63) of a tile has t = c ^ (r / 2 % 4); its 32-bit word j holds the tile's
 * columns 32j + 8t to 32j + 8t + 7 as q + 8, the first in its lowest 4 bits.
 * Columns from D on and rows from V on hold 8 (q = 0), rows from V on scales of 0.
 * pesti_q4_quantize fills d_q and d_scale.  pesti_q4_dequantize writes q s
 * (exact in F32, else rounded once).  Buffers do not overlap (refused).
 * pesti_q4_logits: d_logits [B, ld] (first V columns; F32, BF16 or F16) = x
 * [B, x_ld] (first D columns; F32, BF16 or F16) times the held weight.
 * Sums are f32.  Up to 8 rows of x (4 of F32): over a group of exact products with
 * q, then over the groups with their scales.  More rows: of products with q s,
 * which is exact, over 512 columns (256 for F32 x), then over those; scales below
 * 2^-25 of the largest of these columns of their row lose bits.  16-bit x enters
 * as it is (more rows of BF16: down to 2^-39 of their largest finite value), F32 x
 * within 2^-24 of itself or 2^-39 of its row's largest finite value.  Products of
 * BF16 x with q (up to 8 rows) overflow from some 2^117 of x on.  The weight is
 * read once for every 64 rows of x.  The logits overlap no input (refused).  If a
 * wait inside a kernel ever gives up, after about a second, the logits that it
 * leaves unfinished are NaN.  d_ws: device scratch of
 * pesti_q4_logits_workspace(...) bytes (0 for few rows: NULL will do), 256-byte
 * aligned, any contents; calls whose GPU work may overlap need scratch of their own.
 * All run on the calling thread's current device, stream-ordered (NULL: the
 * legacy default stream), allocate nothing, add in a fixed order (the same
 * inputs give the same bits) and may be captured into a graph.
 */
int pesti_q4_quantize(const void* d_head, pesti_dtype dtype, int64_t V, int64_t D, int64_t ld, int64_t group,
                      void* d_q, void* d_scale, void* stream);
int pesti_q4_dequantize(const void* d_q, const void* d_scale, int64_t V, int64_t D, int64_t group, void* d_head,
                        pesti_dtype dtype, int64_t ld, void* stream);
/* Bytes of scratch, or a negative PESTI_E_* code for refused sizes. */
int64_t pesti_q4_logits_workspace(pesti_dtype dtype, int64_t B, int64_t D);
int pesti_q4_logits(const void* d_x, pesti_dtype dtype, int64_t B, int64_t D, int64_t x_ld, const void* d_q,
                    const void* d_scale, int64_t V, int64_t group, void* d_logits, pesti_dtype out_dtype, int64_t ld,
                    void* d_ws, int64_t ws_bytes, void* stream);

/* Message of the last failure on the calling thread ("" if none). */
const char* pesti_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* PESTI_SAMPLER_H */
