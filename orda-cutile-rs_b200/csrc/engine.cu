// engine.cu -- the chunk-loop orchestrator and the C ABI entry points.
//
// Device flow of one `distillation_loss` call (src/api.rs:188-422), all
// enqueued on the caller's stream with no host synchronisation:
//   label pass      count non-ignored labels, range check, mean scale,
//                   target-row flags for the quantiser
//   for each chunk (the resolver's plan, src/resolver.rs:53-99):
//     [teacher GEMM] teacher logits (Tied/Separate) -> fp32 chunk buffer
//     student GEMM   student logits -> fp32 chunk buffer + online-softmax
//                    records (own and paired-teacher statistics, KL term)
//     row kernel     per-row NLL / KL, bf16 logit gradients into the group
//                    buffer (the merged CE + KL gradient of src/api.rs:319-344)
//   per group of chunks (all chunks when the dlogits of the whole batch fit
//   the memory budget, which holds for every BASELINE configuration):
//     dgrad GEMM     grad_hidden rows = mean_scale * dlogits @ W
//     wgrad GEMM     grad_W (+)= mean_scale * dlogits^T @ hidden
//                    (Tied: student and teacher rows as two K segments)
//   finalize        deterministic f64 reduction of the per-row losses
//   quantise        optional INT8 round trip of grad_W (src/quant.rs)
// Deferring the backward GEMMs to a group turns the per-chunk K=chunk_size
// wgrad (a read-modify-write of the fp32 grad_W per chunk) into one GEMM with
// K = group rows; the loss and gradients are chunk-invariant
// (tests/end_to_end.rs:230-278), so results do not depend on the grouping.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <condition_variable>
#include <functional>
#include <map>
#include <unordered_map>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <memory>
#include <mutex>
#include <optional>
#include <thread>
#include <vector>

#include "../../include/orda.h"
#include "host_io.h"
#include "host_logic.h"
#include "kernels.h"
#include "ptx.cuh"

struct OrdaContext {
  int device = 0;
  int num_sms = 148;
  // [0] status of the last call that clears it, [1] n_non_ignore, [2] a label and
  // [3] a token id out of range, [6] an expired wait of a call before a linear
  // cross entropy (each kept until it is reported), [4] live tokens and [5]
  // finished blocks of a linear cross entropy call (0 between calls)
  int* d_words = nullptr;
  float* d_mean_scale = nullptr;  // [0] distillation loss, [1] linear cross entropy
  void* ws = nullptr;
  size_t ws_bytes = 0;
  size_t ws_refused = 0;  // the smallest size that could not be had, 0 once that has changed
  // A graph captured with this workspace replays with its address: once that
  // has happened a workspace that is outgrown lives on until the context ends.
  bool ws_in_graph = false;
  std::vector<void*> ws_retired;
  void* stage = nullptr;
  size_t stage_bytes = 0;
  int inject_fail = 0;
  cudaStream_t last_stream = nullptr;
  cudaStream_t own_stream = nullptr;  // host-Mat entry: compute stream
  cudaStream_t copy_in = nullptr;     // host-Mat entry: host->device copies
  cudaStream_t copy_out = nullptr;    // host-Mat entry: device->host copies
  // Concurrency of bandwidth-bound kernels with the tensor-bound GEMMs: the
  // persistent GEMM grid leaves `spare_sms` SMs free and the teacher
  // statistics (during the logits GEMM) and the INT8 quantiser (during
  // dgrad) run on the low-priority auxiliary stream. 0 = serial, the
  // default: at c4 the side kernels cost the GEMMs more than they saved
  // (they compete for HBM, L2 and power: GEMM DRAM traffic per step rose from
  // 33.9 to 49.4 GB and the step did not get faster with 2 to 8 spare SMs).
  int spare_sms = 0;
  cudaStream_t aux_stream = nullptr;
  cudaEvent_t aux_ev[3] = {nullptr, nullptr, nullptr};
  std::mutex mu;
  // phase timing (see orda_context_enable_timing)
  bool timing = false;
  bool capturing = false;  // a call under stream capture is being enqueued: events that are only captured have no times
  struct PhaseEvents {
    int phase;
    cudaEvent_t begin, end;
    int launches;
  };
  std::vector<PhaseEvents> pending;
  std::vector<cudaEvent_t> event_pool;
  double phase_ms[ORDA_NUM_PHASES] = {};
  uint64_t phase_launches[ORDA_NUM_PHASES] = {};
  uint64_t launches = 0;
  // Slot buffers of the fused grad_W reduce-scatter (orda_context_slots_*):
  // this rank owns grad_W rows [rank*slice, (rank+1)*slice) and receives
  // every rank's partial of them, fp32 [world][slice][h].
  float* slots = nullptr;
  int slot_world = 0;
  int slot_rank = -1;
  long long slot_slice = 0;
  long long slot_h = 0;
  long long slot_total = 0;  // rows over all owners (owner o: [o*slice, min((o+1)*slice, total)))
  int slot_copies = 1;  // independent [world][slice][h] sets in one buffer
  // INT8 wire format: this rank's local fp32 grad_W partial before it is
  // quantised into the owners' slots
  float* wire_local = nullptr;
  size_t wire_local_bytes = 0;
  float* slot_peer[orda::kMaxSlotRanks] = {};  // rank -> its slot buffer (IPC mapping for other ranks)
  bool slots_attached = false;
  // Persisting-L2 limit set by orda_context_set_l2_persisting, and the
  // value it replaced (restored by orda_context_destroy).
  bool l2_set = false;
  size_t l2_prev = 0;
  // Vocabulary-sharded calls: the workspace layout and shapes of the last
  // orda_vocab_forward_device, whose slice logits the backward phase reuses.
  bool vocab_ready = false;
  size_t vocab_bt = 0, vocab_v = 0, vocab_h = 0;
  int vocab_flags = 0;  // the options that shape the workspace layout
  OrdaChunkPlan vocab_plan{};
  size_t vocab_layout[24] = {};
};

namespace orda {
namespace {

size_t round_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

struct DevInputs {
  MatRef hs, w, ht, wt;     // bf16
  const void* t_logits = nullptr;
  long long ld_t_logits = 0;
  bool t_logits_bf16 = true;
  const int64_t* labels = nullptr;
  size_t bt = 0, h = 0, v = 0, ht_dim = 0;
  OrdaTeacherMode mode = ORDA_TEACHER_TIED;
};

struct Flags {
  float w_s, w_t, kd, temperature, alpha;
  bool need_teacher, teacher_rows, teacher_grad, teacher_ce, quant;
  // Profile::Fast (KernelConfig::fast_math): fp16 logits storage, exact label
  // logits from a dot-product kernel, part of the exp2 work on the FMA pipe
  bool fast;
};

struct WsLayout {
  size_t logits = 0, rec_own = 0, rec_own_t = 0, dlog_s = 0, dlog_t = 0, nll_s = 0, nll_t = 0, kl_base = 0,
         s_part = 0, flags = 0, row_const = 0, x_label = 0, t_label = 0, total = 0;
  size_t ldv = 0, ldd = 0, parts = 0, parts_t = 0, nseg = 0, cs = 0, fwd_rows = 0, group_rows = 0;
};

// Workspace for one rung of the OOM ladder. `fwd_rows` rows (a whole number
// of the plan's chunks, fwd_rows <= group_rows) go through each launch of the
// forward-side kernels (logits GEMMs, statistics, gradient pass);
// `group_rows` rows of bf16 logit gradients are kept for each backward GEMM
// launch. Both are chunk-invariant groupings of the resolver's plan.
WsLayout make_layout(const DevInputs& in, const Flags& f, size_t cs, size_t fwd_rows, size_t group_rows) {
  WsLayout L;
  L.cs = cs;
  L.fwd_rows = fwd_rows;
  L.group_rows = group_rows;
  L.ldv = round_up(in.v, 8);
  L.ldd = round_up(in.v, 8);
  L.parts = (in.v + 127) / 128;
  L.parts_t = f.teacher_rows ? L.parts : 1;  // teacher GEMM records, or one pre-pass record per row
  L.nseg = f.kd > 0.0f ? (in.v + kGradSegCols - 1) / kGradSegCols : 0;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = round_up(off + bytes, 256);
    return o;
  };
  L.logits = take((f.teacher_rows ? 2 : 1) * fwd_rows * L.ldv * (f.fast ? 2 : 4));
  L.rec_own = take(fwd_rows * L.parts * 16);
  L.rec_own_t = take(f.need_teacher ? fwd_rows * L.parts_t * 16 : 0);
  L.dlog_s = take(group_rows * L.ldd * 2);
  L.dlog_t = take(f.teacher_grad ? group_rows * L.ldd * 2 : 0);
  L.nll_s = take(in.bt * sizeof(float));
  L.nll_t = take(in.bt * sizeof(float));
  L.kl_base = take(in.bt * sizeof(double));
  L.s_part = take(in.bt * L.nseg * sizeof(float));
  L.flags = take(f.quant ? in.v : 0);
  L.row_const = take(fwd_rows * kRowConstBytes);
  L.x_label = take(f.fast ? fwd_rows * sizeof(float) : 0);
  L.t_label = take(f.fast && f.teacher_rows && f.teacher_ce ? fwd_rows * sizeof(float) : 0);
  L.total = off;
  return L;
}

// With `keeps`, for what outlives the call: not a workspace that a graph holds,
// whose replay would write over it.
cudaError_t ensure_ws(OrdaContext* ctx, size_t bytes, bool keeps = false) {
  auto refused = [&] {
    ctx->ws_refused = ctx->ws_refused ? std::min(ctx->ws_refused, bytes) : bytes;
    return cudaErrorMemoryAllocation;
  };
  if (ctx->inject_fail > 0) {
    --ctx->inject_fail;
    return refused();
  }
  if (ctx->ws_bytes >= bytes && !(keeps && ctx->ws_in_graph)) return cudaSuccess;
  // a workspace that a graph holds frees no memory for the larger one: it stays
  // the context's until that one has been had
  if (ctx->ws && !ctx->ws_in_graph) {
    cudaFree(ctx->ws);
    ctx->ws = nullptr;
    ctx->ws_bytes = 0;
  }
  void* p = nullptr;
  cudaError_t e = cudaMalloc(&p, bytes);
  if (e != cudaSuccess) {
    cudaGetLastError();  // clear the sticky-free allocation error
    return refused();
  }
  if (bytes >= ctx->ws_refused) ctx->ws_refused = 0;
  if (ctx->ws) ctx->ws_retired.push_back(ctx->ws);
  ctx->ws = p;
  ctx->ws_bytes = bytes;
  ctx->ws_in_graph = false;
  return cudaSuccess;
}

struct AllocTry {
  OrdaContext* ctx;
  const DevInputs* in;
  const Flags* f;
  WsLayout layout;
};

// Allocation for a rung of the OOM ladder: the largest forward and backward
// groups (in whole chunks) whose workspace stays within 60% of the memory
// this call may use; every chunk in one group when that fits, which holds
// for all BASELINE configurations on a 180 GB B200.
int try_alloc_cb(size_t num_chunks, size_t chunk_size, void* user) {
  AllocTry* t = static_cast<AllocTry*>(user);
  const size_t bt = t->in->bt;
  const size_t all_rows = std::min(num_chunks * chunk_size, bt);
  // Fast path (no device query): the held workspace already fits one group
  // of every chunk.
  {
    const WsLayout full = make_layout(*t->in, *t->f, chunk_size, all_rows, all_rows);
    if (t->ctx->inject_fail <= 0 && t->ctx->ws_bytes >= full.total) {
      t->layout = full;
      return 0;
    }
  }
  size_t free_b = 0, total_b = 0;
  cudaMemGetInfo(&free_b, &total_b);
  const size_t budget = static_cast<size_t>((free_b + t->ctx->ws_bytes) * 0.6);
  WsLayout L = make_layout(*t->in, *t->f, chunk_size, chunk_size, chunk_size);
  for (size_t g = num_chunks; g >= 1; g = g / 2) {
    bool found = false;
    for (size_t fw = g; fw >= 1; fw = fw / 2) {
      const WsLayout c = make_layout(*t->in, *t->f, chunk_size, std::min(fw * chunk_size, bt),
                                     std::min(g * chunk_size, bt));
      if (c.total <= budget) {
        L = c;
        found = true;
        break;
      }
      if (fw == 1) break;
    }
    if (found || g == 1) break;
  }
  if (ensure_ws(t->ctx, L.total) != cudaSuccess) return 1;
  t->layout = L;
  return 0;
}

// Records the span of one kernel phase on the launch stream when timing is
// enabled; counts kernel launches always.
struct Phase {
  OrdaContext* ctx;
  int phase;
  cudaStream_t st;
  cudaEvent_t begin = nullptr;
  int n = 0;
  Phase(OrdaContext* c, int p, cudaStream_t s) : ctx(c), phase(p), st(s) {
    if (ctx->timing && !ctx->capturing) {
      begin = take_event(ctx);
      cudaEventRecord(begin, st);
    }
  }
  void launched(int k = 1) {
    n += k;
    ctx->launches += static_cast<uint64_t>(k);
  }
  ~Phase() {
    if (!ctx->timing || !begin) return;
    cudaEvent_t end = take_event(ctx);
    cudaEventRecord(end, st);
    ctx->pending.push_back({phase, begin, end, n});
  }
  static cudaEvent_t take_event(OrdaContext* c) {
    if (!c->event_pool.empty()) {
      cudaEvent_t e = c->event_pool.back();
      c->event_pool.pop_back();
      return e;
    }
    cudaEvent_t e = nullptr;
    cudaEventCreate(&e);
    return e;
  }
};

int cuda_fail(cudaError_t e, const char* what, char* err, size_t len) {
  set_error(err, len, "CUDA error in %s: %s", what, cudaGetErrorString(e));
  return ORDA_ERR_CUDA;
}

// A vocabulary-sharded call: this rank's W (and teacher) rows are
// [v0, v0 + V) of v_total. Phase 1 runs the slice's logits GEMMs and writes
// one partial statistics tuple per row; phase 2 (after the caller gathered
// every rank's tuples) merges them and runs the gradient pass and the
// backward GEMMs of the slice.
static_assert(kVocabTuple == ORDA_VOCAB_TUPLE, "tuple size of the C ABI");

struct VocabCall {
  int phase = 0;
  long long v_total = 0, v0 = 0;
  float* partials_out = nullptr;
  const float* partials_in = nullptr;
  int world = 1;
  int include_rows = 1;
  int scatter_hidden = 0;  // phase 2: dgrad rows go to their owners' slot buffers
};

// Hooks through which the host-Mat entry overlaps its host<->device copies
// with the device work: run_device calls them, on the host, at fixed points
// of its launch order on the compute stream.
struct HostPipe {
  size_t group_rows = 0;  // > 0: forward and backward groups of this many rows (whole chunks)
  // before the row pass of the forward group of rows [s, s + n) (its teacher
  // logits must have landed); a non-zero return aborts the call
  std::function<int(size_t s, size_t n)> before_rows;
  // after the dgrad launches of the backward group [g0, g1) (its grad_hidden
  // rows are final)
  std::function<int(size_t g0, size_t g1)> after_dgrad;
};

// Rank r's slot set `copy` (each set is [world][slice][h] fp32).
float* slot_set(const OrdaContext* ctx, int r, int copy) {
  return ctx->slot_peer[r] + static_cast<long long>(copy) * ctx->slot_world * ctx->slot_slice * ctx->slot_h;
}

// The slot buffers read in the INT8 wire format: codes int8 [world][slice][h],
// then scales f32 [world][slice] at the next 256-byte boundary (the fp32
// buffer holds 4 bytes per element, so both fit for h >= 2).
WireSlots wire_slots(const OrdaContext* ctx) {
  WireSlots w;
  const size_t codes = static_cast<size_t>(ctx->slot_world) * ctx->slot_slice * ctx->slot_h;
  for (int r = 0; r < ctx->slot_world; ++r) {
    uint8_t* b = reinterpret_cast<uint8_t*>(ctx->slot_peer[r]);
    w.codes[r] = reinterpret_cast<int8_t*>(b);
    w.scales[r] = reinterpret_cast<float*>(b + round_up(codes, 256));
  }
  return w;
}

// The auxiliary stream (lowest priority, so the GEMM's CTAs are placed
// first) and its dependency events; created on first use.
cudaError_t aux_init(OrdaContext* ctx) {
  if (ctx->aux_stream) return cudaSuccess;
  int least = 0, greatest = 0;
  cudaError_t e = cudaDeviceGetStreamPriorityRange(&least, &greatest);
  if (e == cudaSuccess) e = cudaStreamCreateWithPriority(&ctx->aux_stream, cudaStreamNonBlocking, least);
  for (int i = 0; i < 3 && e == cudaSuccess; ++i) e = cudaEventCreateWithFlags(&ctx->aux_ev[i], cudaEventDisableTiming);
  return e;
}

// `to` waits for the work queued on `from` so far (through event ev).
cudaError_t stream_after(cudaStream_t to, cudaStream_t from, cudaEvent_t ev) {
  cudaError_t e = cudaEventRecord(ev, from);
  return e == cudaSuccess ? cudaStreamWaitEvent(to, ev, 0) : e;
}

// Rows of this rank's slice (the last owner may hold fewer than slot_slice).
long long slot_rows_mine(const OrdaContext* ctx) {
  const long long r0 = static_cast<long long>(ctx->slot_rank) * ctx->slot_slice;
  return std::max(0ll, std::min(ctx->slot_slice, ctx->slot_total - r0));
}

int run_device(OrdaContext* ctx, const DevInputs& in, const OrdaLossOptions& o, const OrdaDeviceOutputs& out,
               const OrdaShardOptions* shard, cudaStream_t st, OrdaChunkPlan* plan_out, char* err, size_t len,
               const VocabCall* vc = nullptr, const HostPipe* hp = nullptr) {
  const int vphase = vc ? vc->phase : 0;
  // any other call reuses the workspace that holds a vocabulary forward
  // phase's slice logits: its backward phase must not run after this
  if (vphase == 0) ctx->vocab_ready = false;
  Flags f{};
  f.w_s = o.student_ce_weight;
  f.w_t = o.has_teacher_ce_weight ? o.teacher_ce_weight : orda_default_teacher_ce_weight(in.mode);
  if (f.w_t < 0.0f) {
    set_error(err, len, "teacher_ce_weight must be >= 0, got %s", fmt_f32(f.w_t).c_str());
    return ORDA_ERR_INVALID;
  }
  f.kd = o.kd_weight;
  f.temperature = o.temperature;
  f.alpha = o.label_smoothing;
  f.need_teacher = f.kd > 0.0f || f.w_t > 0.0f;
  const bool live_teacher = in.mode == ORDA_TEACHER_TIED || in.mode == ORDA_TEACHER_SEPARATE;
  f.teacher_rows = f.need_teacher && live_teacher;
  f.teacher_grad = f.w_t > 0.0f && live_teacher;
  f.teacher_ce = f.w_t > 0.0f;
  f.fast = o.config.fast_math != 0;
  const bool scatter = shard && shard->scatter_grad_weight;
  f.quant = o.config.quantize_grad_weight != 0 && !(shard && shard->skip_quantize) && !scatter;

  const bool scatter_hidden = vphase == 2 && vc->scatter_hidden;
  if (scatter_hidden) {
    const long long need = f.teacher_grad ? 2 : 1;
    if (!ctx->slots_attached || ctx->slot_total != static_cast<long long>(in.bt) ||
        ctx->slot_h != static_cast<long long>(in.h) || ctx->slot_copies < need ||
        (f.teacher_grad && in.ht_dim != in.h)) {
      set_error(err, len, "scatter_grad_hidden needs slot buffers made for BT rows x H with %lld set(s) "
                          "(orda_context_slots_create / _attach) and H_t == H", need);
      return ORDA_ERR_INVALID;
    }
  }
  if (vphase == 1) {
    if (!vc->partials_out) {
      set_error(err, len, "row_partials output is required");
      return ORDA_ERR_INVALID;
    }
  } else if ((!out.grad_student_hidden && !scatter_hidden) || (!out.grad_weight && !scatter) || !out.scalars) {
    set_error(err, len, "grad_student_hidden, grad_weight and scalars outputs are required");
    return ORDA_ERR_INVALID;
  }
  if (vphase && (vc->v0 < 0 || vc->v0 + static_cast<long long>(in.v) > vc->v_total || vc->world < 1 ||
                 (vphase == 2 && !vc->partials_in))) {
    set_error(err, len, "vocabulary shard out of range (v0 = %lld, slice rows = %zu, v_total = %lld)", vc->v0, in.v,
              vc->v_total);
    return ORDA_ERR_INVALID;
  }
  if (scatter) {
    if (!ctx->slots_attached) {
      set_error(err, len, "scatter_grad_weight needs slot buffers (orda_context_slots_create / _attach)");
      return ORDA_ERR_INVALID;
    }
    if (static_cast<long long>(in.v) != ctx->slot_total || static_cast<long long>(in.h) != ctx->slot_h) {
      set_error(err, len, "slot buffers were made for V=%lld, H=%lld; this call has V=%zu, H=%zu",
                ctx->slot_total, ctx->slot_h, in.v, in.h);
      return ORDA_ERR_INVALID;
    }
  }
  const bool wire = scatter && shard->int8_wire;
  if (wire) {
    // the local fp32 partial, quantised into the owners' slots after wgrad
    const size_t need = in.v * in.h * sizeof(float);
    if (ctx->wire_local_bytes < need) {
      cudaFree(ctx->wire_local);
      ctx->wire_local = nullptr;
      ctx->wire_local_bytes = 0;
      if (cudaMalloc(&ctx->wire_local, need) != cudaSuccess) {
        cudaGetLastError();
        set_error(err, len, "INT8 wire: %zu bytes for the local grad_W partial are not available", need);
        return ORDA_ERR_OOM;
      }
      ctx->wire_local_bytes = need;
    }
  }
  if (vphase != 1 && !scatter_hidden && f.teacher_grad && !out.grad_teacher_hidden) {
    set_error(err, len, "grad_teacher_hidden output is required (teacher CE weight > 0 with a live teacher)");
    return ORDA_ERR_INVALID;
  }
  if (vphase != 1 && f.teacher_grad && in.mode == ORDA_TEACHER_SEPARATE && !out.grad_teacher_weight) {
    set_error(err, len, "grad_teacher_weight output is required (Separate teacher with teacher CE weight > 0)");
    return ORDA_ERR_INVALID;
  }

  const size_t bt = in.bt, v = in.v, h = in.h, ht = in.ht_dim;
  // the plan of the full vocabulary (a vocabulary-sharded call reports the
  // plan the single-device call would use)
  OrdaChunkPlan plan = resolve_chunk_size(bt, o.chunk_size, true, vphase ? static_cast<size_t>(vc->v_total) : v,
                                          o.config.has_max_chunks != 0, o.config.max_chunks);
  const size_t limit = o.config.has_max_chunks ? o.config.max_chunks : default_max_chunks_limit(bt);
  AllocTry at{ctx, &in, &f, {}};
  OrdaChunkPlan used{};
  static_assert(sizeof(WsLayout) <= sizeof(ctx->vocab_layout), "saved layout");
  const int layout_flags = (f.fast ? 64 : 0) | (f.need_teacher ? 1 : 0) | (f.teacher_rows ? 2 : 0) |
                           (f.teacher_grad ? 4 : 0) |
                           (f.quant ? 8 : 0) | (f.kd > 0.0f ? 16 : 0) | (f.teacher_ce ? 32 : 0);
  bool have = false;
  if (vphase == 2) {
    // the forward phase's workspace, with its slice logits and statistics
    if (!ctx->vocab_ready || ctx->vocab_bt != bt || ctx->vocab_v != v || ctx->vocab_h != h ||
        ctx->vocab_flags != layout_flags) {
      set_error(err, len, "orda_vocab_backward_device must follow orda_vocab_forward_device on the same context "
                          "with the same shapes and options");
      return ORDA_ERR_INVALID;
    }
    std::memcpy(&at.layout, ctx->vocab_layout, sizeof(WsLayout));
    used = ctx->vocab_plan;
    have = true;
  } else if (vphase == 1) {
    // the slice logits of the whole batch stay in the workspace until the
    // backward phase: one forward and one backward group
    ctx->vocab_ready = false;
    at.layout = make_layout(in, f, plan.chunk_size, bt, bt);
    if (ensure_ws(ctx, at.layout.total, true) != cudaSuccess) {
      set_error(err, len, "vocabulary-sharded calls keep the whole batch's slice logits between the two phases: "
                          "%zu bytes of workspace are not available", at.layout.total);
      return ORDA_ERR_OOM;
    }
    used = plan;
    have = true;
  } else {
    if (hp && hp->group_rows > 0) {
      // the host entry's pipelined grouping (whole chunks), if it fits
      const size_t gr = std::min(bt, round_up(hp->group_rows, plan.chunk_size));
      const WsLayout c = make_layout(in, f, plan.chunk_size, gr, gr);
      if (ensure_ws(ctx, c.total) == cudaSuccess) {
        at.layout = c;
        used = plan;
        have = true;
      }
    }
    // Rung 0 is the resolver's plan itself (a Fixed chunk size keeps its row
    // count); after an allocation failure the ladder doubles the chunk count
    // along chunk_doubling_schedule, as the upstream dispatcher does.
    if (!have) have = try_alloc_cb(plan.num_chunks, plan.chunk_size, &at) == 0;
    if (have) used = plan;
  }
  if (!have) {
    for (size_t nc : chunk_doubling_schedule(bt, plan.num_chunks, std::max(limit, plan.num_chunks))) {
      if (nc <= plan.num_chunks) continue;
      const size_t cs_r = ceil_div(bt, nc);
      if (try_alloc_cb(nc, cs_r, &at) == 0) {
        used = OrdaChunkPlan{cs_r, nc};
        have = true;
        break;
      }
    }
  }
  if (!have) {
    set_error(err, len, "device workspace allocation failed for every chunk count of the OOM ladder");
    return ORDA_ERR_OOM;
  }
  const WsLayout& L = at.layout;
  if (plan_out) *plan_out = used;

  uint8_t* ws = static_cast<uint8_t*>(ctx->ws);
  void* logits = ws + L.logits;
  void* logits_t = ws + L.logits + L.fwd_rows * L.ldv * (f.fast ? 2 : 4);
  float* x_label = f.fast ? reinterpret_cast<float*>(ws + L.x_label) : nullptr;
  float* t_label = f.fast && f.teacher_rows && f.teacher_ce ? reinterpret_cast<float*>(ws + L.t_label) : nullptr;
  float* rec_own = reinterpret_cast<float*>(ws + L.rec_own);
  float* rec_own_t = reinterpret_cast<float*>(ws + L.rec_own_t);
  uint16_t* dlog_s = reinterpret_cast<uint16_t*>(ws + L.dlog_s);
  uint16_t* dlog_t = reinterpret_cast<uint16_t*>(ws + L.dlog_t);
  float* nll_s = reinterpret_cast<float*>(ws + L.nll_s);
  float* nll_t = reinterpret_cast<float*>(ws + L.nll_t);
  double* kl_base = reinterpret_cast<double*>(ws + L.kl_base);
  float* s_part = reinterpret_cast<float*>(ws + L.s_part);
  uint8_t* tflags = f.quant ? ws + L.flags : nullptr;
  void* row_const = ws + L.row_const;
  int* status = ctx->d_words;

  cudaError_t e;
  const long long denom_override = shard ? shard->global_non_ignore : 0;
  if (vphase != 2) {
    if ((e = cudaMemsetAsync(ctx->d_words, 0, 2 * sizeof(int), st)) != cudaSuccess)
      return cuda_fail(e, "memset", err, len);
    if (tflags && (e = cudaMemsetAsync(tflags, 0, v, st)) != cudaSuccess) return cuda_fail(e, "memset", err, len);
    Phase ph_prep(ctx, 5, st);
    ph_prep.launched();
    // labels are checked against the full vocabulary; a slice's target rows
    // are the labels that fall in it
    launch_label_prep(in.labels, static_cast<long long>(bt),
                      vphase ? vc->v_total : static_cast<long long>(v), o.ignore_index,
                      o.reduction == ORDA_REDUCTION_SUM, denom_override, ctx->d_words + 1, ctx->d_mean_scale,
                      vphase ? nullptr : tflags, status, st);
    if (vphase && tflags) {
      ph_prep.launched();
      launch_target_flags(in.labels, static_cast<long long>(bt), static_cast<long long>(v), o.ignore_index, tflags,
                          st, vc->v0);
    }
  }

  const float inv_t = 1.0f / f.temperature;
  const char* why = nullptr;
  const size_t fwd_rows = L.fwd_rows;
  const size_t group_rows = L.group_rows;
  const size_t t_esz = in.t_logits_bf16 ? 2 : 4;
  bool quant_async = false;  // the INT8 round trip was queued on the auxiliary stream
  for (size_t g0 = 0; g0 < bt; g0 += group_rows) {
    const size_t g1 = std::min(g0 + group_rows, bt);
    for (size_t s = g0; s < g1; s += fwd_rows) {
      const size_t n = std::min(fwd_rows, g1 - s);
      const void* t_rows = live_teacher ? static_cast<const void*>(logits_t)
                                        : static_cast<const void*>(static_cast<const uint8_t*>(in.t_logits) +
                                                                   s * in.ld_t_logits * t_esz);
      const long long t_ld = live_teacher ? static_cast<long long>(L.ldv) : in.ld_t_logits;
      const int t_bf16 = live_teacher ? 0 : static_cast<int>(in.t_logits_bf16);
      const int t_dtype = live_teacher ? (f.fast ? kLogitF16 : kLogitF32) : (in.t_logits_bf16 ? kLogitBF16 : kLogitF32);
      // given teacher logits: their statistics run on the auxiliary stream
      // while the logits GEMM runs on all SMs but spare_sms
      const bool conc_t = ctx->spare_sms > 0 && vphase != 2 && f.need_teacher && !live_teacher && !hp;
      if (conc_t) {
        if ((e = aux_init(ctx)) != cudaSuccess) return cuda_fail(e, "auxiliary stream", err, len);
        if ((e = stream_after(ctx->aux_stream, st, ctx->aux_ev[0])) != cudaSuccess)
          return cuda_fail(e, "event", err, len);
        Phase ph_t(ctx, 1, ctx->aux_stream);
        ph_t.launched();
        launch_teacher_stats(t_rows, t_ld, t_bf16, static_cast<int>(n), static_cast<int>(v), inv_t, rec_own_t,
                             ctx->aux_stream, f.teacher_ce, f.fast);
        if ((e = cudaEventRecord(ctx->aux_ev[1], ctx->aux_stream)) != cudaSuccess)
          return cuda_fail(e, "event", err, len);
      }
      if (vphase != 2) {
        Phase ph_fwd(ctx, 0, st);
        // ---- teacher logits + statistics (Tied / Separate)
        if (f.teacher_rows) {
          int nl = 0;  // the GEMM and, with an L2 carve-out, the demotion kernel
          GemmDesc gd;
          const MatRef& tw = in.mode == ORDA_TEACHER_TIED ? in.w : in.wt;
          const size_t kdim = in.mode == ORDA_TEACHER_TIED ? h : ht;
          gd.a[0] = MatRef{static_cast<const uint16_t*>(in.ht.ptr) + s * in.ht.ld, static_cast<long long>(n),
                           static_cast<long long>(kdim), in.ht.ld};
          gd.b[0] = tw;
          gd.k_seg[0] = static_cast<long long>(kdim);
          gd.M = static_cast<long long>(n);
          gd.N = static_cast<long long>(v);
          gd.epi = Epi::Logits;
          gd.status = status;
          gd.args.logits = logits_t;
          gd.args.logits_f16 = f.fast;
          gd.args.ldl = static_cast<long long>(L.ldv);
          gd.args.rec_own = rec_own_t;
          gd.args.n_parts = static_cast<int>(L.parts);
          gd.args.inv_t = inv_t;
          gd.args.own_dT = f.kd > 0.0f;
          gd.demote_kept = ctx->l2_set;
          gd.launches = &nl;
          if ((e = gemm_launch(gd, ctx->num_sms, st, &why)) != cudaSuccess)
            return cuda_fail(e, why ? why : "teacher logits GEMM", err, len);
          ph_fwd.launched(nl);
        }
        // ---- student logits + statistics
        int nl = 0;  // the GEMM and, with an L2 carve-out, the demotion kernel
        GemmDesc gd;
        gd.a[0] = MatRef{static_cast<const uint16_t*>(in.hs.ptr) + s * in.hs.ld, static_cast<long long>(n),
                         static_cast<long long>(h), in.hs.ld};
        gd.b[0] = in.w;
        gd.k_seg[0] = static_cast<long long>(h);
        gd.M = static_cast<long long>(n);
        gd.N = static_cast<long long>(v);
        gd.epi = Epi::Logits;
        gd.status = status;
        gd.args.logits = logits;
        gd.args.logits_f16 = f.fast;
        gd.spare_sms = conc_t ? ctx->spare_sms : 0;
        gd.args.ldl = static_cast<long long>(L.ldv);
        gd.args.rec_own = rec_own;
        gd.args.n_parts = static_cast<int>(L.parts);
        gd.args.inv_t = inv_t;
        gd.args.own_dT = f.kd > 0.0f;
        gd.demote_kept = ctx->l2_set;
        gd.launches = &nl;
        if ((e = gemm_launch(gd, ctx->num_sms, st, &why)) != cudaSuccess)
          return cuda_fail(e, why ? why : "student logits GEMM", err, len);
        ph_fwd.launched(nl);
      }
      // ---- row pass: teacher statistics (given logits), losses, logit gradients
      if (hp && hp->before_rows) {
        if (int rc = hp->before_rows(s, n)) return rc;
      }
      {
        Phase ph_rows(ctx, 1, st);
        if (conc_t) {
          if ((e = cudaStreamWaitEvent(st, ctx->aux_ev[1], 0)) != cudaSuccess) return cuda_fail(e, "event", err, len);
        } else if (vphase != 2 && f.need_teacher && !live_teacher) {
          ph_rows.launched();
          launch_teacher_stats(t_rows, t_ld, t_bf16, static_cast<int>(n), static_cast<int>(v), inv_t, rec_own_t, st,
                               f.teacher_ce, f.fast);
        }
        if (f.fast && vphase != 2) {
          // exact fp32 label logits (the 16-bit logits buffer is rounded)
          const long long lv0 = vphase ? vc->v0 : 0;
          ph_rows.launched();
          launch_label_logits(static_cast<const uint16_t*>(in.hs.ptr) + s * in.hs.ld, in.hs.ld, in.w.ptr, in.w.ld,
                              static_cast<long long>(h), in.labels + s, static_cast<long long>(n), lv0,
                              static_cast<long long>(v), o.ignore_index, x_label, st);
          if (t_label) {
            const MatRef& tw = in.mode == ORDA_TEACHER_TIED ? in.w : in.wt;
            ph_rows.launched();
            launch_label_logits(static_cast<const uint16_t*>(in.ht.ptr) + s * in.ht.ld, in.ht.ld, tw.ptr, tw.ld,
                                static_cast<long long>(in.mode == ORDA_TEACHER_TIED ? h : ht), in.labels + s,
                                static_cast<long long>(n), lv0, static_cast<long long>(v), o.ignore_index, t_label, st);
          }
        }
        ph_rows.launched(vphase == 1 ? 1 : kRowLaunches);
        RowArgs r{};
        r.n = static_cast<int>(n);
        r.v = static_cast<int>(v);
        r.n_parts = static_cast<int>(L.parts);
        r.n_parts_t = static_cast<int>(L.parts_t);
        r.logits_s = logits;
        r.logits_f16 = f.fast;
        r.x_label = x_label;
        r.t_label = t_label;
        r.fast = f.fast;
        r.ldl = static_cast<long long>(L.ldv);
        r.teacher = t_rows;
        r.ld_teacher = t_ld;
        r.teacher_dtype = t_dtype;
        r.rec_own = rec_own;
        r.rec_own_t = rec_own_t;
        r.labels = in.labels + s;
        r.ignore_index = o.ignore_index;
        r.w_s = f.w_s;
        r.w_t = f.w_t;
        r.kd = f.kd;
        r.temperature = f.temperature;
        r.inv_t = inv_t;
        r.alpha = f.alpha;
        r.need_kl = f.kd > 0.0f;
        r.teacher_ce = f.teacher_ce;
        r.teacher_grad = f.teacher_grad;
        r.dlog_s = dlog_s + (s - g0) * L.ldd;
        r.dlog_t = f.teacher_grad ? dlog_t + (s - g0) * L.ldd : nullptr;
        r.ldd = static_cast<long long>(L.ldd);
        r.nll_s_rows = nll_s + s;
        r.nll_t_rows = nll_t + s;
        r.kl_base_rows = kl_base + s;
        r.s_part = s_part + s * L.nseg;
        r.nseg = static_cast<int>(L.nseg);
        r.row_const = row_const;
        r.num_sms = ctx->num_sms;
        if (vphase) {
          r.v_total = static_cast<int>(vc->v_total);
          r.v0 = vc->v0;
          r.world = vc->world;
          r.partials_out = vphase == 1 ? vc->partials_out + s * kVocabTuple : nullptr;
          r.partials_in = vphase == 2 ? vc->partials_in : nullptr;
        }
        if (vphase == 1) launch_vocab_partials(r, st);
        else if (vphase == 2) launch_vocab_rows(r, st);
        else launch_rows(r, st);
        if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "row kernels", err, len);
      }
    }
    if (vphase == 1) continue;  // the backward phase follows the exchange of the partials
    const long long rows_g = static_cast<long long>(g1 - g0);
    const long long vv = static_cast<long long>(v);
    // Last backward group with the INT8 round trip: wgrad first, then the
    // quantiser on the auxiliary stream while dgrad runs on all SMs but
    // spare_sms (dgrad does not touch grad_W; the order of the two GEMMs does
    // not change any result).
    const bool conc_q = ctx->spare_sms > 0 && f.quant && g1 == bt && !hp;
    auto do_wgrad = [&]() -> int {
      // ---- wgrad: grad_W (+)= mean_scale * dlogits^T @ hidden
      {
        Phase ph(ctx, 3, st);
        int nl = 0;  // the GEMM and, with an L2 carve-out, the demotion kernel
        GemmDesc gd;
        gd.a_mn_major = true;
        gd.b_mn_major = true;
        gd.a[0] = MatRef{dlog_s, rows_g, vv, static_cast<long long>(L.ldd)};
        gd.b[0] = MatRef{static_cast<const uint16_t*>(in.hs.ptr) + g0 * in.hs.ld, rows_g, static_cast<long long>(h),
                         in.hs.ld};
        gd.k_seg[0] = rows_g;
        if (f.teacher_grad && in.mode == ORDA_TEACHER_TIED) {
          gd.nseg = 2;
          gd.a[1] = MatRef{dlog_t, rows_g, vv, static_cast<long long>(L.ldd)};
          gd.b[1] = MatRef{static_cast<const uint16_t*>(in.ht.ptr) + g0 * in.ht.ld, rows_g, static_cast<long long>(h),
                           in.ht.ld};
          gd.k_seg[1] = rows_g;
        }
        gd.M = vv;
        gd.N = static_cast<long long>(h);
        gd.raster_n_fastest = true;
        gd.status = status;
        if (wire) {
          // INT8 wire: the local fp32 partial first (quantised into the owners'
          // slots once complete)
          gd.args.out0 = ctx->wire_local;
          gd.args.ld0 = static_cast<long long>(h);
        } else if (scatter) {
          // each owner's rows go straight to its slot buffer: the reduce-scatter
          // transfer overlaps this GEMM
          gd.args.scatter = 1;
          gd.args.slot_rank = ctx->slot_rank;
          gd.args.slot_slice = ctx->slot_slice;
          gd.args.slot_ld = ctx->slot_h;
          for (int r = 0; r < kMaxSlotRanks; ++r) gd.args.slot[r] = ctx->slot_peer[r];
        } else {
          gd.args.out0 = out.grad_weight;
          gd.args.ld0 = static_cast<long long>(out.ld_grad_weight);
        }
        gd.args.alpha_ptr = ctx->d_mean_scale;
        gd.args.beta = g0 > 0 ? 1.0f : 0.0f;
        gd.demote_kept = ctx->l2_set;
        gd.launches = &nl;
        if ((e = gemm_launch(gd, ctx->num_sms, st, &why)) != cudaSuccess)
          return cuda_fail(e, why ? why : "wgrad GEMM", err, len);
        ph.launched(nl);
      }
      if (f.teacher_grad && in.mode == ORDA_TEACHER_SEPARATE) {
        Phase ph(ctx, 3, st);
        int nl = 0;  // the GEMM and, with an L2 carve-out, the demotion kernel
        GemmDesc gd;
        gd.a_mn_major = true;
        gd.b_mn_major = true;
        gd.a[0] = MatRef{dlog_t, rows_g, vv, static_cast<long long>(L.ldd)};
        gd.b[0] = MatRef{static_cast<const uint16_t*>(in.ht.ptr) + g0 * in.ht.ld, rows_g, static_cast<long long>(ht),
                         in.ht.ld};
        gd.k_seg[0] = rows_g;
        gd.M = vv;
        gd.N = static_cast<long long>(ht);
        gd.raster_n_fastest = true;
        gd.status = status;
        gd.args.out0 = out.grad_teacher_weight;
        gd.args.ld0 = static_cast<long long>(out.ld_grad_teacher_weight);
        gd.args.alpha_ptr = ctx->d_mean_scale;
        gd.args.beta = g0 > 0 ? 1.0f : 0.0f;
        gd.demote_kept = ctx->l2_set;
        gd.launches = &nl;
        if ((e = gemm_launch(gd, ctx->num_sms, st, &why)) != cudaSuccess)
          return cuda_fail(e, why ? why : "teacher wgrad GEMM", err, len);
        ph.launched(nl);
      }
      return ORDA_OK;
    };
    // ---- dgrad: grad_h rows = mean_scale * dlogits @ W
    auto dgrad = [&](const uint16_t* dl, const MatRef& wmat, long long ncols, float* outp, size_t ldo,
                     int copy) -> int {
      Phase ph(ctx, 2, st);
      ph.launched();
      GemmDesc gd;
      gd.a[0] = MatRef{dl, rows_g, vv, static_cast<long long>(L.ldd)};
      gd.b_mn_major = true;
      gd.b[0] = MatRef{wmat.ptr, vv, ncols, wmat.ld};
      gd.k_seg[0] = vv;
      gd.M = rows_g;
      gd.N = ncols;
      gd.raster_n_fastest = true;
      gd.status = status;
      gd.spare_sms = conc_q ? ctx->spare_sms : 0;
      if (scatter_hidden) {
        // vocabulary-sharded: this rank's partial of every owner's rows goes
        // straight to the owner's slot set `copy` (a reduce-scatter over rows)
        gd.args.scatter = 1;
        gd.args.slot_rank = ctx->slot_rank;
        gd.args.slot_slice = ctx->slot_slice;
        gd.args.slot_ld = ctx->slot_h;
        for (int r = 0; r < ctx->slot_world; ++r) gd.args.slot[r] = slot_set(ctx, r, copy);
      } else {
        gd.args.out0 = outp + g0 * ldo;
        gd.args.ld0 = static_cast<long long>(ldo);
      }
      gd.args.alpha_ptr = ctx->d_mean_scale;
      cudaError_t ee = gemm_launch(gd, ctx->num_sms, st, &why);
      if (ee != cudaSuccess) return cuda_fail(ee, why ? why : "dgrad GEMM", err, len);
      return ORDA_OK;
    };
    if (conc_q) {
      if (int rc = do_wgrad()) return rc;
      if ((e = aux_init(ctx)) != cudaSuccess) return cuda_fail(e, "auxiliary stream", err, len);
      if ((e = stream_after(ctx->aux_stream, st, ctx->aux_ev[0])) != cudaSuccess)
        return cuda_fail(e, "event", err, len);
      Phase ph(ctx, 4, ctx->aux_stream);
      ph.launched();
      const uint64_t seed = o.config.has_stochastic_seed ? o.config.stochastic_seed : 0;
      launch_quant(out.grad_weight, static_cast<long long>(v), static_cast<long long>(h),
                   static_cast<long long>(out.ld_grad_weight), tflags, o.config.stochastic_rounding, seed,
                   out.grad_weight_q, out.grad_weight_scale, ctx->aux_stream, vphase == 2 ? vc->v0 : 0);
      if ((e = cudaEventRecord(ctx->aux_ev[2], ctx->aux_stream)) != cudaSuccess)
        return cuda_fail(e, "event", err, len);
      quant_async = true;
    }
    if (int rc = dgrad(dlog_s, in.w, static_cast<long long>(h), out.grad_student_hidden, out.ld_grad_student_hidden,
                       0))
      return rc;
    if (f.teacher_grad) {
      const MatRef& tw = in.mode == ORDA_TEACHER_TIED ? in.w : in.wt;
      const long long tn = static_cast<long long>(in.mode == ORDA_TEACHER_TIED ? h : ht);
      if (int rc = dgrad(dlog_t, tw, tn, out.grad_teacher_hidden, out.ld_grad_teacher_hidden, 1)) return rc;
    }
    if (hp && hp->after_dgrad) {
      if (int rc = hp->after_dgrad(g0, g1)) return rc;
    }
    if (!conc_q) {
      if (int rc = do_wgrad()) return rc;
    }
  }
  if (wire) {
    // row-wise INT8 partials (and scales) into the owners' slots
    Phase ph(ctx, 3, st);
    ph.launched();
    launch_quant_send(ctx->wire_local, static_cast<long long>(v), static_cast<long long>(h),
                      static_cast<long long>(h), ctx->slot_slice, ctx->slot_rank, ctx->slot_world,
                      wire_slots(ctx), st);
  }
  if (vphase == 1) {
    if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "vocabulary forward phase", err, len);
    std::memcpy(ctx->vocab_layout, &L, sizeof(WsLayout));
    ctx->vocab_bt = bt;
    ctx->vocab_v = v;
    ctx->vocab_h = h;
    ctx->vocab_plan = used;
    ctx->vocab_flags = layout_flags;
    ctx->vocab_ready = true;
    ctx->last_stream = st;
    return ORDA_OK;
  }
  {
    Phase ph(ctx, 5, st);
    ph.launched();
    const double t_sq = static_cast<double>(f.temperature * f.temperature);
    launch_finalize(nll_s, nll_t, kl_base, s_part, static_cast<int>(L.nseg), t_sq, static_cast<long long>(bt),
                    ctx->d_mean_scale, f.w_s, f.w_t, f.kd, out.scalars, st, vphase == 2 ? vc->include_rows : 1);
  }
  if (quant_async) {
    // the call ends on `st` after the auxiliary stream's quantiser
    if ((e = cudaStreamWaitEvent(st, ctx->aux_ev[2], 0)) != cudaSuccess) return cuda_fail(e, "event", err, len);
  } else if (f.quant) {
    Phase ph(ctx, 4, st);
    ph.launched();
    const uint64_t seed = o.config.has_stochastic_seed ? o.config.stochastic_seed : 0;
    launch_quant(out.grad_weight, static_cast<long long>(v), static_cast<long long>(h),
                 static_cast<long long>(out.ld_grad_weight), tflags, o.config.stochastic_rounding, seed,
                 out.grad_weight_q, out.grad_weight_scale, st, vphase == 2 ? vc->v0 : 0);
  }
  if (vphase == 2) ctx->vocab_ready = false;
  if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "kernel launch", err, len);
  ctx->last_stream = st;
  return ORDA_OK;
}

// ------------------------------------------------- linear cross entropy
// Makes the context's device current and the caller's device current again.
struct DeviceScope {
  int prev = -1, dev;
  explicit DeviceScope(int d) : dev(d) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceScope() {
    if (prev >= 0 && prev != dev) cudaSetDevice(prev);
  }
};

int stream_capturing(cudaStream_t st, bool* capturing, char* err, size_t len) {
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(st, &cap);
  if (e != cudaSuccess) return cuda_fail(e, "cudaStreamIsCapturing", err, len);
  *capturing = cap != cudaStreamCaptureStatusNone;
  return ORDA_OK;
}

// The workspace for a call. Under stream capture nothing may be allocated, and
// the graph keeps the workspace's address.
int call_ws(OrdaContext* ctx, size_t bytes, bool capturing, char* err, size_t len) {
  if (capturing) {
    if (ctx->ws_bytes < bytes) {
      set_error(err, len, "a captured call cannot allocate its %zu bytes of workspace: make the same call once "
                          "before the capture", bytes);
      return ORDA_ERR_OOM;
    }
    ctx->ws_in_graph = true;
    return ORDA_OK;
  }
  if (ensure_ws(ctx, bytes) != cudaSuccess) {
    set_error(err, len, "device workspace allocation of %zu bytes failed", bytes);
    return ORDA_ERR_OOM;
  }
  return ORDA_OK;
}

// Bytes of 16-bit logits that a call with gradients keeps by default: the
// whole batch of the largest benchmark shape (8192 rows x 131072) is half of it.
constexpr size_t kCePieceBytes = size_t{4} << 30;
constexpr size_t kCePieceCols = 512;  // pieces are whole 512-column tiles

struct CeLayout {
  size_t h_clean = 0, ref = 0, rec = 0, sx = 0, row_const = 0, nll = 0, piece = 0, dgrad = 0, total = 0;
  size_t cols = 0;      // vocabulary columns of one piece
  size_t n_parts = 0, rec_ld = 0, clean_rows = 0, ld_clean = 0, ld_piece = 0, ld_dgrad = 0, slab_rows = 0;
  int slabs = 1;
  bool few = false;           // logits by few_kernel
  bool dgrad_direct = false;  // the dgrad product writes the fp32 output itself
};

// K slabs of the dgrad product: with fewer 256 x 256 tiles than CTA pairs its
// long K (the vocabulary) is cut so that every pair has a tile, each at least
// eight K blocks deep (the depth of the ring and a little more); the slabs'
// partial sums are added in order afterwards. One token at H = 4096, V =
// 131072: 16 tiles would leave 58 of 74 pairs idle while all of W is read.
int ce_slabs(size_t rows, size_t h, size_t cols, int num_sms) {
  const size_t pairs = static_cast<size_t>(std::max(1, num_sms / 2));
  const size_t tiles = ceil_div(rows, 256) * ceil_div(h, 256);
  const size_t k_blocks = ceil_div(cols, 64);
  if (tiles >= pairs) return 1;
  return static_cast<int>(std::max<size_t>(1, std::min(pairs / tiles, k_blocks / 8)));
}

CeLayout ce_layout(size_t bt, size_t h, size_t v, size_t cols, bool smooth, const OrdaLinearCeOutputs& o,
                   int num_sms) {
  CeLayout L;
  const bool grads = o.grad_hidden || o.grad_weight;
  L.cols = cols;
  L.few = bt <= kCeFewRows;
  L.n_parts = ceil_div(v, L.few ? kCeFewPartCols : kCePartCols);
  L.rec_ld = round_up(L.n_parts, 4);  // rows of records start on 32-byte sectors
  // rows on 128-byte lines: a TMA box row (128 bytes) then is one line, not two
  // (1999 x 1000 x 100003 with gradients: 1.42 ms, 1.67 ms with 16-byte rows)
  L.ld_clean = round_up(h, 64);
  L.ld_piece = round_up(cols, 64);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = round_up(off + bytes, 256);
    return at;
  };
  // few tokens: as many rows as the kernel reads (zeros behind the last token). Rows
  // of a TMA box beyond the matrix are fetched too, all from one place, and 148 SMs
  // asking for the same lines cost a quarter of the time
  L.clean_rows = L.few ? static_cast<size_t>(few_rows(static_cast<long long>(bt))) : bt;
  L.h_clean = take(L.clean_rows * L.ld_clean * 2);
  L.ref = take(bt * sizeof(float2));
  L.rec = take(bt * L.rec_ld * sizeof(float2));
  L.sx = take(smooth ? bt * L.rec_ld * sizeof(float) : 0);
  L.row_const = take(bt * sizeof(float4));
  L.nll = take(o.nll ? 0 : bt * sizeof(float));
  L.piece = take(grads ? bt * L.ld_piece * 2 : 0);
  if (o.grad_hidden) {
    L.slabs = ce_slabs(bt, h, cols, num_sms);
    L.slab_rows = round_up(bt, 32);
    L.ld_dgrad = round_up(h, 4);
    L.dgrad_direct = L.slabs == 1 && o.grad_hidden_dtype == ORDA_DTYPE_F32;
    L.dgrad = take(L.dgrad_direct ? 0 : static_cast<size_t>(L.slabs) * L.slab_rows * L.ld_dgrad * 4);
  }
  L.total = off;
  return L;
}

// One call: label pass, logits product (the statistics of every piece but
// one, then that piece with its 16-bit logits kept), losses, and for each
// piece its logit gradients (from the kept logits, or by the logits product
// again) and the two gradient products. No [BT, V] buffer exists unless it fits
// piece_bytes; each further piece costs its share of one more product.
int run_linear_ce(OrdaContext* ctx, const OrdaDeviceMat& hm, const OrdaDeviceMat& wm, const int64_t* labels, size_t bt,
                  const OrdaLinearCeOptions& o, const OrdaLinearCeOutputs& out, cudaStream_t st, char* err,
                  size_t len) {
  const size_t h = hm.cols, v = wm.rows;
  const bool grads = out.grad_hidden || out.grad_weight;
  const bool smooth = o.label_smoothing > 0.0f;
  ctx->vocab_ready = false;  // the workspace no longer holds a vocabulary forward phase

  // the piece: all of the vocabulary if that fits, else even pieces of whole tiles
  const size_t limit = o.piece_bytes ? o.piece_bytes : kCePieceBytes;
  size_t pieces = 1, cols = v;
  if (grads) {
    const size_t fit = std::max(kCePieceCols, limit / (2 * bt) / kCePieceCols * kCePieceCols);
    if (fit < v) {
      pieces = ceil_div(v, fit);
      cols = round_up(ceil_div(v, pieces), kCePieceCols);
    }
  }
  auto layout = [&](size_t c) { return ce_layout(bt, h, v, c, smooth, out, ctx->num_sms); };
  auto narrower = [](size_t c) { return round_up(ceil_div(c, 2), kCePieceCols); };
  CeLayout L = layout(cols);
  const bool capturing = ctx->capturing;
  // Where as much workspace was refused before: the widest of the ladder's pieces
  // that the present one holds, if any. A call that had to take smaller pieces,
  // and the same call made again or captured, then take the same ones.
  if (grads && ctx->inject_fail <= 0 && ctx->ws_refused && L.total >= ctx->ws_refused) {
    size_t c = cols;
    while (layout(c).total > ctx->ws_bytes && c > kCePieceCols) c = narrower(c);
    if (layout(c).total <= ctx->ws_bytes) cols = c;
  }
  while (true) {
    L = layout(cols);
    const int rc = call_ws(ctx, L.total, capturing, err, len);
    if (rc == ORDA_OK) break;
    // smaller pieces where the memory is short, as the chunk ladder does
    if (rc != ORDA_ERR_OOM || capturing || !grads || cols <= kCePieceCols) return rc;
    cols = narrower(cols);
  }
  pieces = ceil_div(v, cols);

  uint8_t* ws = static_cast<uint8_t*>(ctx->ws);
  CeArgs a;
  a.h = hm.data;
  a.ldh = static_cast<long long>(hm.ld);
  a.w = wm.data;
  a.ldw = static_cast<long long>(wm.ld);
  a.bt = static_cast<long long>(bt);
  a.hd = static_cast<long long>(h);
  a.v = static_cast<long long>(v);
  a.labels = labels;
  a.ignore_index = o.ignore_index;
  a.alpha = o.label_smoothing;
  a.reduction_sum = o.reduction == ORDA_REDUCTION_SUM;
  a.denom_override = o.global_non_ignore;
  a.h_clean = reinterpret_cast<uint16_t*>(ws + L.h_clean);
  a.clean_rows = static_cast<long long>(L.clean_rows);
  a.ld_clean = static_cast<long long>(L.ld_clean);
  a.ref = reinterpret_cast<float2*>(ws + L.ref);
  a.rec = reinterpret_cast<float2*>(ws + L.rec);
  a.sx = smooth ? reinterpret_cast<float*>(ws + L.sx) : nullptr;
  a.rec_ld = static_cast<long long>(L.rec_ld);
  a.n_parts = static_cast<int>(L.n_parts);
  a.part_shift = L.few ? 5 : 6;
  static_assert(kCeFewPartCols == 1 << 5 && kCePartCols == 1 << 6, "part_shift");
  a.row_const = reinterpret_cast<float4*>(ws + L.row_const);
  a.nll = out.nll ? out.nll : reinterpret_cast<float*>(ws + L.nll);
  a.lse = out.lse;
  a.loss = out.loss;
  a.scale = ctx->d_mean_scale + 1;
  a.status = ctx->d_words;
  a.bad_label = ctx->d_words + 2;
  a.earlier = ctx->d_words + 6;
  a.count = ctx->d_words + 4;
  a.done = ctx->d_words + 5;
  uint16_t* piece = grads ? reinterpret_cast<uint16_t*>(ws + L.piece) : nullptr;

  cudaError_t e;
  const char* why = nullptr;
  {
    Phase ph(ctx, 5, st);
    ph.launched();
    if ((e = launch_ce_prep(a, st)) != cudaSuccess) return cuda_fail(e, "label pass", err, len);
  }
  const MatRef hmat{a.h_clean, a.bt, a.hd, a.ld_clean};
  // logits of vocabulary columns [v0, v0 + n): statistics (and kept 16-bit logits), or the gradients
  auto logits = [&](size_t v0, size_t n, Epi epi, uint16_t* keep) -> int {
    Phase ph(ctx, 0, st);
    int nl = 0;
    GemmDesc gd;
    gd.a[0] = hmat;
    gd.a[0].rows = a.clean_rows;
    gd.b[0] = MatRef{static_cast<const uint16_t*>(wm.data) + v0 * wm.ld, static_cast<long long>(n), a.hd, a.ldw};
    gd.k_seg[0] = a.hd;
    gd.M = a.bt;
    gd.N = static_cast<long long>(n);
    gd.epi = epi;
    gd.status = ctx->d_words;
    gd.args.out16 = keep;
    gd.args.ld16 = static_cast<long long>(L.ld_piece);
    gd.args.ce_v0 = static_cast<long long>(v0);
    gd.args.ce_ref = a.ref;
    gd.args.ce_rec = a.rec + (v0 >> a.part_shift);
    gd.args.ce_sx = smooth ? a.sx + (v0 >> a.part_shift) : nullptr;
    gd.args.ce_rec_ld = a.rec_ld;
    gd.args.ce_const = a.row_const;
    gd.args.pdl = kPdlWaitFirst;
    gd.demote_kept = ctx->l2_set;
    gd.launches = &nl;
    e = L.few && epi == Epi::CeStats ? few_launch(gd, ctx->num_sms, st, &why) : gemm_launch(gd, ctx->num_sms, st, &why);
    if (e != cudaSuccess) return cuda_fail(e, why ? why : "logits GEMM", err, len);
    ph.launched(nl);
    return ORDA_OK;
  };
  if (pieces > 1) {
    if (int rc = logits(cols, v - cols, Epi::CeStats, nullptr)) return rc;
  }
  if (int rc = logits(0, std::min(cols, v), Epi::CeStats, piece)) return rc;
  {
    Phase ph(ctx, 1, st);
    ph.launched();
    if ((e = launch_ce_rows(a, piece, static_cast<long long>(L.ld_piece),
                            grads ? static_cast<long long>(std::min(cols, v)) : 0, st)) != cudaSuccess)
      return cuda_fail(e, "row kernel", err, len);
  }
  for (size_t v0 = 0; grads && v0 < v; v0 += cols) {
    const size_t n = std::min(cols, v - v0);
    if (v0 > 0) {
      if (int rc = logits(v0, n, Epi::CeGrad, piece)) return rc;
    }
    const MatRef dl{piece, a.bt, static_cast<long long>(n), static_cast<long long>(L.ld_piece)};
    if (out.grad_hidden) {
      Phase ph(ctx, 2, st);
      int nl = 0;
      GemmDesc gd;
      gd.a[0] = dl;
      gd.b_mn_major = true;
      gd.b[0] = MatRef{static_cast<const uint16_t*>(wm.data) + v0 * wm.ld, static_cast<long long>(n), a.hd, a.ldw};
      gd.k_seg[0] = static_cast<long long>(n);
      gd.M = a.bt;
      gd.N = a.hd;
      gd.raster_n_fastest = true;
      gd.status = ctx->d_words;
      gd.args.beta = v0 > 0 ? 1.0f : 0.0f;
      if (L.dgrad_direct) {
        gd.args.out0 = static_cast<float*>(out.grad_hidden);
        gd.args.ld0 = static_cast<long long>(out.ld_grad_hidden);
        gd.args.alpha_ptr = a.scale;
      } else {
        gd.args.out0 = reinterpret_cast<float*>(ws + L.dgrad);
        gd.args.ld0 = static_cast<long long>(L.ld_dgrad);
        // the last piece may be narrower than its slabs are many: every slab
        // that earlier pieces wrote stays in the sum
        gd.args.slabs = std::min<int>(L.slabs, static_cast<int>(ceil_div(n, 64)));
        gd.args.slab_rows = static_cast<long long>(L.slab_rows);
      }
      gd.args.pdl = kPdlWaitFirst;
      gd.demote_kept = ctx->l2_set;
      gd.launches = &nl;
      if ((e = gemm_launch(gd, ctx->num_sms, st, &why)) != cudaSuccess)
        return cuda_fail(e, why ? why : "dgrad GEMM", err, len);
      ph.launched(nl);
    }
    if (out.grad_weight) {
      Phase ph(ctx, 3, st);
      int nl = 0;
      GemmDesc gd;
      gd.a_mn_major = true;
      gd.b_mn_major = true;
      gd.a[0] = dl;
      gd.b[0] = hmat;
      gd.k_seg[0] = a.bt;
      gd.M = static_cast<long long>(n);
      gd.N = a.hd;
      gd.raster_n_fastest = true;
      gd.status = ctx->d_words;
      gd.args.alpha_ptr = a.scale;
      if (out.grad_weight_dtype == ORDA_DTYPE_BF16) {
        gd.epi = Epi::StoreBf16;
        gd.args.out16 = static_cast<uint16_t*>(out.grad_weight) + v0 * out.ld_grad_weight;
        gd.args.ld16 = static_cast<long long>(out.ld_grad_weight);
        // it may run beside the dgrad product, which began with the gradients complete
        gd.args.pdl = out.grad_hidden ? kPdlWaitLast : kPdlWaitFirst;
      } else {
        gd.args.out0 = static_cast<float*>(out.grad_weight) + v0 * out.ld_grad_weight;
        gd.args.ld0 = static_cast<long long>(out.ld_grad_weight);
      }
      gd.demote_kept = ctx->l2_set;
      gd.launches = &nl;
      if ((e = gemm_launch(gd, ctx->num_sms, st, &why)) != cudaSuccess)
        return cuda_fail(e, why ? why : "wgrad GEMM", err, len);
      ph.launched(nl);
    }
  }
  if (out.grad_hidden && !L.dgrad_direct) {
    Phase ph(ctx, 2, st);
    ph.launched();
    if ((e = launch_slab_sum(reinterpret_cast<const float*>(ws + L.dgrad), L.slabs,
                             static_cast<long long>(L.slab_rows), static_cast<long long>(L.ld_dgrad), a.bt, a.hd,
                             a.scale, out.grad_hidden, static_cast<long long>(out.ld_grad_hidden),
                             out.grad_hidden_dtype == ORDA_DTYPE_BF16, st)) != cudaSuccess)
      return cuda_fail(e, "dgrad sum", err, len);
  }
  if (!capturing) ctx->last_stream = st;  // what is captured runs elsewhere, and its stream may end before the context
  return ORDA_OK;
}

// --------------------------------------------------------------- helpers
bool device_is_sm100(int dev) {
  cudaDeviceProp p;
  if (cudaGetDeviceProperties(&p, dev) != cudaSuccess) return false;
  return p.major == 10;
}

int check_status(OrdaContext* ctx, char* err, size_t len) {
  int words[7] = {};
  cudaError_t e = cudaStreamSynchronize(ctx->last_stream);
  if (e != cudaSuccess) return cuda_fail(e, "stream synchronize", err, len);
  e = cudaMemcpy(words, ctx->d_words, sizeof words, cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return cuda_fail(e, "status read", err, len);
  // one report a call; a word is cleared with its own report, so that what else
  // happened is reported by the next calls. Word 0 stays until the next loss call
  // clears it, marked as reported unless that has happened already: kernels give
  // their waits up while it is set.
  auto put = [&](int word, int value) {
    return cudaMemcpy(ctx->d_words + word, &value, sizeof value, cudaMemcpyHostToDevice);
  };
  int status = words[0] & ~kStatusReported;
  if (words[3] != DEV_OK) {
    if ((e = put(3, DEV_OK)) != cudaSuccess) return cuda_fail(e, "status write", err, len);
    set_error(err, len, "a token id is out of range [0, V) (device id check)");
    return ORDA_ERR_LABEL;
  }
  if (words[2] != DEV_OK) {
    if ((e = put(2, DEV_OK)) != cudaSuccess) return cuda_fail(e, "status write", err, len);
    status = DEV_LABEL_RANGE;
  } else if (words[6] != DEV_OK) {
    if ((e = put(6, DEV_OK)) != cudaSuccess) return cuda_fail(e, "status write", err, len);
    status = words[6];
  } else if (status != DEV_OK) {
    if ((e = launch_mark_reported(ctx->d_words, status, ctx->last_stream)) != cudaSuccess ||
        (e = cudaStreamSynchronize(ctx->last_stream)) != cudaSuccess)
      return cuda_fail(e, "status write", err, len);
  }
  if (status == DEV_LABEL_RANGE) {
    set_error(err, len, "a label is out of range [0, V) and != ignore_index (device label check)");
    return ORDA_ERR_LABEL;
  }
  if (status != DEV_OK) {
    set_error(err, len, "a bounded device wait expired (status 0x%x); results are invalid", status);
    return ORDA_ERR_TIMEOUT;
  }
  return ORDA_OK;
}

// Teacher-logit slab of the host entry's copy pipeline (bytes).
std::atomic<size_t> g_host_slab_bytes{size_t{512} << 20};
// bytes the last successful host-Mat call copied each way (orda_last_call_bytes)
std::atomic<uint64_t> g_last_h2d{0}, g_last_d2h{0};

// The host-Mat entry's compressed grad_W download (on unless
// ORDA_HOST_DEQUANT=0, a diagnostic switch read on every call).
bool host_dequant_enabled() {
  const char* v = std::getenv("ORDA_HOST_DEQUANT");
  return !(v && v[0] == '0');
}

// The host-Mat entry's bf16 uploads: GEMM operands rounded on the host and
// teacher-logit chunks that hold bf16 values sent as bf16, while the copy
// engine is busy (1, the default); 0: fp32 copies only; 2: every chunk
// through the host passes (a diagnostic switch read on every call, which the
// tests use to cover the host conversion on small inputs).
int host_convert_mode() {
  const char* v = std::getenv("ORDA_HOST_CONVERT");
  if (!v || !v[0]) return 1;
  return v[0] == '0' ? 0 : v[0] == '2' ? 2 : 1;
}

std::mutex g_default_mu;
OrdaContext* g_default_ctx[64] = {nullptr};

// Output buffers of the host-Mat entry: page-locked host memory recycled
// through a pool, so the gradients come back at full PCIe bandwidth without
// page faults on every call. orda_output_free returns a buffer to the pool;
// at most kPinnedPoolCap bytes of free buffers are kept.
constexpr size_t kPinnedPoolCap = size_t{16} << 30;
std::mutex g_pinned_mu;
std::multimap<size_t, void*> g_pinned_free;      // capacity -> buffer
std::unordered_map<void*, size_t> g_pinned_cap;  // live and free buffers
size_t g_pinned_free_bytes = 0;

float* pinned_alloc(size_t bytes) {
  bytes = std::max<size_t>(bytes, 256);
  {
    std::lock_guard<std::mutex> lock(g_pinned_mu);
    auto it = g_pinned_free.lower_bound(bytes);
    if (it != g_pinned_free.end() && it->first <= 2 * bytes) {
      void* p = it->second;
      g_pinned_free_bytes -= it->first;
      g_pinned_free.erase(it);
      return static_cast<float*>(p);
    }
  }
  void* p = nullptr;
  if (cudaHostAlloc(&p, bytes, cudaHostAllocDefault) != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  std::lock_guard<std::mutex> lock(g_pinned_mu);
  g_pinned_cap[p] = bytes;
  return static_cast<float*>(p);
}

void pinned_release(void* p) {
  if (!p) return;
  std::lock_guard<std::mutex> lock(g_pinned_mu);
  auto it = g_pinned_cap.find(p);
  if (it == g_pinned_cap.end()) return;
  const size_t cap = it->second;
  if (g_pinned_free_bytes + cap > kPinnedPoolCap) {
    g_pinned_cap.erase(it);
    cudaFreeHost(p);
    return;
  }
  g_pinned_free.emplace(cap, p);
  g_pinned_free_bytes += cap;
}

}  // namespace
}  // namespace orda

using namespace orda;

extern "C" {

int orda_is_available(void) {
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 0;
  }
  return device_is_sm100(0) ? 1 : 0;
}

int orda_context_create(int device, OrdaContext** out, char* err, size_t err_len) {
  *out = nullptr;
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || device < 0 || device >= n) {
    cudaGetLastError();
    set_error(err, err_len, "no CUDA device %d available (this library has no CPU path)", device);
    return ORDA_ERR_BACKEND;
  }
  if (!device_is_sm100(device)) {
    set_error(err, err_len, "device %d is not an sm_100 (B200-class) GPU", device);
    return ORDA_ERR_BACKEND;
  }
  cudaError_t e = cudaSetDevice(device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice", err, err_len);
  std::unique_ptr<OrdaContext> ctx(new OrdaContext());
  ctx->device = device;
  cudaDeviceGetAttribute(&ctx->num_sms, cudaDevAttrMultiProcessorCount, device);
  if ((e = cudaMalloc(&ctx->d_words, 8 * sizeof(int))) != cudaSuccess) return cuda_fail(e, "cudaMalloc", err, err_len);
  if ((e = cudaMalloc(&ctx->d_mean_scale, 4 * sizeof(float))) != cudaSuccess)
    return cuda_fail(e, "cudaMalloc", err, err_len);
  cudaMemset(ctx->d_words, 0, 8 * sizeof(int));
  *out = ctx.release();
  return ORDA_OK;
}

static void release_slots(OrdaContext* ctx) {
  for (int r = 0; r < orda::kMaxSlotRanks; ++r) {
    if (ctx->slot_peer[r] && r != ctx->slot_rank) cudaIpcCloseMemHandle(ctx->slot_peer[r]);
    ctx->slot_peer[r] = nullptr;
  }
  if (ctx->slots) cudaFree(ctx->slots);
  ctx->slots = nullptr;
  ctx->slot_world = 0;
  ctx->slot_rank = -1;
  ctx->slot_slice = 0;
  ctx->slot_h = 0;
  ctx->slot_total = 0;
  ctx->slot_copies = 1;
  ctx->slots_attached = false;
}

int orda_context_slots_create(OrdaContext* ctx, int world, int rank, size_t total_rows, size_t h, int copies,
                              OrdaIpcHandle* handle_out, char* err, size_t err_len) {
  if (!ctx || !handle_out || world < 1 || world > orda::kMaxSlotRanks || rank < 0 || rank >= world ||
      total_rows == 0 || h < 2 || copies < 1 || copies > 4) {
    set_error(err, err_len,
              "invalid argument (world in [1, %d], rank in [0, world), total_rows > 0, h >= 2, copies in [1, 4])",
              orda::kMaxSlotRanks);
    return ORDA_ERR_INVALID;
  }
  // owner slices: ceil(total / world) rounded up to 8 rows; the last owner
  // holds the remainder
  const size_t slice_rows = round_up(ceil_div(total_rows, static_cast<size_t>(world)), 8);
  if (static_cast<size_t>(world - 1) * slice_rows >= total_rows) {
    set_error(err, err_len, "%zu rows leave rank %d of %d no rows in slices of %zu", total_rows, world - 1, world,
              slice_rows);
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  cudaDeviceSynchronize();
  release_slots(ctx);
  void* p = nullptr;
  const size_t bytes = static_cast<size_t>(copies) * world * slice_rows * h * sizeof(float);
  cudaError_t e = cudaMalloc(&p, bytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error(err, err_len, "slot buffer allocation failed (%zu bytes)", bytes);
    return ORDA_ERR_OOM;
  }
  cudaIpcMemHandle_t hd;
  if ((e = cudaIpcGetMemHandle(&hd, p)) != cudaSuccess) {
    cudaFree(p);
    return cuda_fail(e, "cudaIpcGetMemHandle", err, err_len);
  }
  static_assert(sizeof(hd) <= sizeof(handle_out->bytes), "IPC handle size");
  std::memset(handle_out->bytes, 0, sizeof(handle_out->bytes));
  std::memcpy(handle_out->bytes, &hd, sizeof(hd));
  ctx->slots = static_cast<float*>(p);
  ctx->slot_world = world;
  ctx->slot_rank = rank;
  ctx->slot_slice = static_cast<long long>(slice_rows);
  ctx->slot_h = static_cast<long long>(h);
  ctx->slot_total = static_cast<long long>(total_rows);
  ctx->slot_copies = copies;
  return ORDA_OK;
}

int orda_context_slots_attach(OrdaContext* ctx, const OrdaIpcHandle* handles, char* err, size_t err_len) {
  if (!ctx || !handles || !ctx->slots) {
    set_error(err, err_len, "invalid argument (create the slot buffer first)");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  for (int r = 0; r < ctx->slot_world; ++r) {
    if (r == ctx->slot_rank) {
      ctx->slot_peer[r] = ctx->slots;
      continue;
    }
    cudaIpcMemHandle_t hd;
    std::memcpy(&hd, handles[r].bytes, sizeof(hd));
    void* p = nullptr;
    cudaError_t e = cudaIpcOpenMemHandle(&p, hd, cudaIpcMemLazyEnablePeerAccess);
    if (e != cudaSuccess) {
      cudaGetLastError();
      for (int k = 0; k < r; ++k)
        if (k != ctx->slot_rank && ctx->slot_peer[k]) {
          cudaIpcCloseMemHandle(ctx->slot_peer[k]);
          ctx->slot_peer[k] = nullptr;
        }
      return cuda_fail(e, "cudaIpcOpenMemHandle (peer slot buffer)", err, err_len);
    }
    ctx->slot_peer[r] = static_cast<float*>(p);
  }
  ctx->slots_attached = true;
  return ORDA_OK;
}

int orda_reduce_slots_device(OrdaContext* ctx, float* grad_w_slice, size_t ld, const int64_t* labels, size_t n_labels,
                             int64_t ignore_index, int quantize, int stochastic, uint64_t seed, int8_t* q, float* scale,
                             int int8_wire, void* stream, char* err, size_t err_len) {
  if (!ctx || !grad_w_slice || (n_labels > 0 && !labels) || !ctx->slots ||
      ld < static_cast<size_t>(ctx->slot_h)) {
    set_error(err, err_len, "invalid argument (slot buffer, output slice and its ld >= H)");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long slice = ctx->slot_slice, h = ctx->slot_h, rows = slot_rows_mine(ctx);
  const long long row0 = static_cast<long long>(ctx->slot_rank) * slice;
  uint8_t* flags = nullptr;
  if (quantize) {
    ctx->vocab_ready = false;  // the flags below overwrite the workspace
    if (ensure_ws(ctx, round_up(static_cast<size_t>(slice), 256)) != cudaSuccess) {
      set_error(err, err_len, "device workspace allocation failed");
      return ORDA_ERR_OOM;
    }
    flags = static_cast<uint8_t*>(ctx->ws);
    cudaError_t e = cudaMemsetAsync(flags, 0, static_cast<size_t>(slice), st);
    if (e != cudaSuccess) return cuda_fail(e, "memset", err, err_len);
    orda::launch_target_flags(labels, static_cast<long long>(n_labels), rows, ignore_index, flags, st, row0);
    ctx->launches += 1;
  }
  if (int8_wire) {
    // dequantise the INT8 partials, sum them in rank order (and quantise)
    WireSlots mine;
    const WireSlots all = wire_slots(ctx);
    mine.codes[0] = all.codes[ctx->slot_rank];
    mine.scales[0] = all.scales[ctx->slot_rank];
    if (!orda::launch_wire_reduce(mine, ctx->slot_world, slice, rows, h, grad_w_slice, static_cast<long long>(ld),
                                  flags, quantize, stochastic, seed, q, scale, row0, st)) {
      set_error(err, err_len, "INT8 wire: rows of H=%lld do not fit the reduction's shared memory", h);
      return ORDA_ERR_INVALID;
    }
    ctx->launches += 1;
  } else if (!quantize) {
    orda::launch_slot_reduce(ctx->slots, ctx->slot_world, slice, rows, h, grad_w_slice, static_cast<long long>(ld),
                             st);
    ctx->launches += 1;
  } else if (orda::launch_slot_reduce_quant(ctx->slots, ctx->slot_world, slice, rows, h, grad_w_slice,
                                            static_cast<long long>(ld), flags, stochastic, seed, q, scale, row0,
                                            st)) {
    // one pass: rank-ordered sum and INT8 round trip of each row
    ctx->launches += 1;
  } else {
    orda::launch_slot_reduce(ctx->slots, ctx->slot_world, slice, rows, h, grad_w_slice, static_cast<long long>(ld),
                             st);
    orda::launch_quant(grad_w_slice, rows, h, static_cast<long long>(ld), flags, stochastic, seed, q, scale, st,
                       row0);
    ctx->launches += 2;
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "slot reduction", err, err_len);
  ctx->last_stream = st;
  return ORDA_OK;
}

int orda_reduce_slot_set_device(OrdaContext* ctx, int copy, float* out, size_t ld, void* stream, char* err,
                                size_t err_len) {
  if (!ctx || !out || !ctx->slots || copy < 0 || copy >= ctx->slot_copies || ld < static_cast<size_t>(ctx->slot_h)) {
    set_error(err, err_len, "invalid argument (slot buffer, set index in range, output ld >= H)");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  orda::launch_slot_reduce(ctx->slots + static_cast<long long>(copy) * ctx->slot_world * ctx->slot_slice * ctx->slot_h,
                           ctx->slot_world, ctx->slot_slice, slot_rows_mine(ctx), ctx->slot_h, out,
                           static_cast<long long>(ld), st);
  ctx->launches += 1;
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "slot reduction", err, err_len);
  ctx->last_stream = st;
  return ORDA_OK;
}

int orda_context_set_l2_persisting(OrdaContext* ctx, size_t bytes, size_t* granted, char* err, size_t err_len) {
  if (!ctx) {
    set_error(err, err_len, "null context");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  int max_bytes = 0;
  cudaError_t e = cudaDeviceGetAttribute(&max_bytes, cudaDevAttrMaxPersistingL2CacheSize, ctx->device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute", err, err_len);
  size_t prev = 0;
  if ((e = cudaDeviceGetLimit(&prev, cudaLimitPersistingL2CacheSize)) != cudaSuccess)
    return cuda_fail(e, "cudaDeviceGetLimit", err, err_len);
  const size_t want = std::min(bytes, static_cast<size_t>(max_bytes > 0 ? max_bytes : 0));
  if ((e = cudaDeviceSetLimit(cudaLimitPersistingL2CacheSize, want)) != cudaSuccess)
    return cuda_fail(e, "cudaDeviceSetLimit", err, err_len);
  if (!ctx->l2_set) {
    ctx->l2_set = true;
    ctx->l2_prev = prev;
  }
  // the driver rounds the carve-out to its own granularity: report what holds
  size_t now = want;
  if ((e = cudaDeviceGetLimit(&now, cudaLimitPersistingL2CacheSize)) != cudaSuccess)
    return cuda_fail(e, "cudaDeviceGetLimit", err, err_len);
  if (granted) *granted = now;
  return ORDA_OK;
}

void orda_context_destroy(OrdaContext* ctx) {
  if (!ctx) return;
  cudaSetDevice(ctx->device);
  cudaDeviceSynchronize();
  if (ctx->l2_set) cudaDeviceSetLimit(cudaLimitPersistingL2CacheSize, ctx->l2_prev);
  release_slots(ctx);
  cudaFree(ctx->ws);
  for (void* p : ctx->ws_retired) cudaFree(p);
  cudaFree(ctx->stage);
  cudaFree(ctx->wire_local);
  cudaFree(ctx->d_words);
  cudaFree(ctx->d_mean_scale);
  for (cudaStream_t sp : {ctx->own_stream, ctx->copy_in, ctx->copy_out, ctx->aux_stream})
    if (sp) cudaStreamDestroy(sp);
  for (cudaEvent_t ev : ctx->aux_ev)
    if (ev) cudaEventDestroy(ev);
  for (auto& pe : ctx->pending) {
    cudaEventDestroy(pe.begin);
    cudaEventDestroy(pe.end);
  }
  for (cudaEvent_t e : ctx->event_pool) cudaEventDestroy(e);
  delete ctx;
}

int orda_context_check(OrdaContext* ctx, char* err, size_t err_len) {
  if (!ctx) return ORDA_ERR_INVALID;
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  return check_status(ctx, err, err_len);
}

size_t orda_context_workspace_bytes(const OrdaContext* ctx) { return ctx ? ctx->ws_bytes : 0; }

void orda_context_inject_alloc_failures(OrdaContext* ctx, int count) {
  if (ctx) ctx->inject_fail = count;
}

static bool dev_mat_ok(const OrdaDeviceMat& m, bool need_bf16) {
  if (need_bf16 && m.dtype != ORDA_DTYPE_BF16) return false;
  const size_t esz = m.dtype == ORDA_DTYPE_BF16 ? 2 : 4;
  if (!m.data) return false;
  if ((reinterpret_cast<uintptr_t>(m.data) & 15) != 0) return false;
  if ((m.ld * esz) % 16 != 0 || m.ld < m.cols) return false;
  return true;
}

// Validates the device-entry arguments (shapes, scalars, dtypes, alignment)
// and describes the inputs for run_device.
static int build_dev_inputs(const OrdaDeviceMat* student_hidden, const OrdaDeviceMat* weight, const int64_t* labels,
                            size_t bt, const OrdaDeviceTeacher* teacher, const OrdaLossOptions* opts, DevInputs* out_in,
                            char* err, size_t err_len) {
  const Shape2 sh{student_hidden->rows, student_hidden->cols}, w{weight->rows, weight->cols};
  const Shape2 th{teacher->hidden.rows, teacher->hidden.cols}, tw{teacher->weight.rows, teacher->weight.cols},
      tl{teacher->logits.rows, teacher->logits.cols};
  size_t v = 0, h = 0, bt_chk = 0;
  if (int rc = validate_shapes(sh, w, bt, teacher->mode, th, tw, tl, *opts, &v, &h, &bt_chk, err, err_len)) return rc;
  if (int rc = validate_scalars_and_teacher(bt_chk, h, v, teacher->mode, th, tw, tl, *opts, err, err_len)) return rc;
  if (opts->backend == ORDA_BACKEND_CPU) {
    set_error(err, err_len, "Backend::Cpu is not available: this library is the B200 path and has no CPU backend");
    return ORDA_ERR_BACKEND;
  }
  if (!dev_mat_ok(*student_hidden, true) || !dev_mat_ok(*weight, true)) {
    set_error(err, err_len, "student_hidden and weight must be bf16, 16-byte aligned, with ld*2 a multiple of 16");
    return ORDA_ERR_INVALID;
  }
  DevInputs& in = *out_in;
  in.bt = bt;
  in.h = h;
  in.v = v;
  in.mode = teacher->mode;
  in.labels = labels;
  in.hs = MatRef{student_hidden->data, static_cast<long long>(bt), static_cast<long long>(h),
                 static_cast<long long>(student_hidden->ld)};
  in.w = MatRef{weight->data, static_cast<long long>(v), static_cast<long long>(h), static_cast<long long>(weight->ld)};
  in.ht_dim = h;
  if (teacher->mode == ORDA_TEACHER_TIED || teacher->mode == ORDA_TEACHER_SEPARATE) {
    if (!dev_mat_ok(teacher->hidden, true)) {
      set_error(err, err_len, "teacher hidden must be bf16, 16-byte aligned, with ld*2 a multiple of 16");
      return ORDA_ERR_INVALID;
    }
    in.ht_dim = teacher->hidden.cols;
    in.ht = MatRef{teacher->hidden.data, static_cast<long long>(bt), static_cast<long long>(in.ht_dim),
                   static_cast<long long>(teacher->hidden.ld)};
  }
  if (teacher->mode == ORDA_TEACHER_SEPARATE) {
    if (!dev_mat_ok(teacher->weight, true)) {
      set_error(err, err_len, "teacher weight must be bf16, 16-byte aligned, with ld*2 a multiple of 16");
      return ORDA_ERR_INVALID;
    }
    in.wt = MatRef{teacher->weight.data, static_cast<long long>(v), static_cast<long long>(in.ht_dim),
                   static_cast<long long>(teacher->weight.ld)};
  }
  if (teacher->mode == ORDA_TEACHER_PRECOMPUTED) {
    if (!dev_mat_ok(teacher->logits, false)) {
      set_error(err, err_len, "teacher logits must be 16-byte aligned with ld*elem a multiple of 16");
      return ORDA_ERR_INVALID;
    }
    in.t_logits = teacher->logits.data;
    in.ld_t_logits = static_cast<long long>(teacher->logits.ld);
    in.t_logits_bf16 = teacher->logits.dtype == ORDA_DTYPE_BF16;
  }
  return ORDA_OK;
}

int orda_distillation_loss_device(OrdaContext* ctx, const OrdaDeviceMat* student_hidden, const OrdaDeviceMat* weight,
                                  const int64_t* labels, size_t bt, const OrdaDeviceTeacher* teacher,
                                  const OrdaLossOptions* opts, const OrdaDeviceOutputs* out,
                                  const OrdaShardOptions* shard, void* stream, OrdaChunkPlan* plan_out, char* err,
                                  size_t err_len) {
  if (!ctx || !student_hidden || !weight || !labels || !teacher || !opts || !out) {
    set_error(err, err_len, "null argument");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  DevInputs in;
  if (int rc = build_dev_inputs(student_hidden, weight, labels, bt, teacher, opts, &in, err, err_len)) return rc;
  cudaSetDevice(ctx->device);
  return run_device(ctx, in, *opts, *out, shard, static_cast<cudaStream_t>(stream), plan_out, err, err_len);
}

int orda_vocab_forward_device(OrdaContext* ctx, const OrdaDeviceMat* student_hidden, const OrdaDeviceMat* weight_slice,
                              const int64_t* labels, size_t bt, const OrdaDeviceTeacher* teacher,
                              const OrdaLossOptions* opts, const OrdaVocabShard* vs, float* row_partials, void* stream,
                              char* err, size_t err_len) {
  if (!ctx || !student_hidden || !weight_slice || !labels || !teacher || !opts || !vs || !row_partials) {
    set_error(err, err_len, "null argument");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  DevInputs in;
  if (int rc = build_dev_inputs(student_hidden, weight_slice, labels, bt, teacher, opts, &in, err, err_len)) return rc;
  cudaSetDevice(ctx->device);
  VocabCall vc;
  vc.phase = 1;
  vc.v_total = vs->v_total;
  vc.v0 = vs->v0;
  vc.world = vs->world;
  vc.partials_out = row_partials;
  OrdaDeviceOutputs none{};
  return run_device(ctx, in, *opts, none, nullptr, static_cast<cudaStream_t>(stream), nullptr, err, err_len, &vc);
}

int orda_vocab_backward_device(OrdaContext* ctx, const OrdaDeviceMat* student_hidden,
                               const OrdaDeviceMat* weight_slice, const int64_t* labels, size_t bt,
                               const OrdaDeviceTeacher* teacher, const OrdaLossOptions* opts, const OrdaVocabShard* vs,
                               const float* all_partials, const OrdaDeviceOutputs* out, void* stream,
                               OrdaChunkPlan* plan_out, char* err, size_t err_len) {
  if (!ctx || !student_hidden || !weight_slice || !labels || !teacher || !opts || !vs || !all_partials || !out) {
    set_error(err, err_len, "null argument");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  DevInputs in;
  if (int rc = build_dev_inputs(student_hidden, weight_slice, labels, bt, teacher, opts, &in, err, err_len)) return rc;
  cudaSetDevice(ctx->device);
  VocabCall vc;
  vc.phase = 2;
  vc.v_total = vs->v_total;
  vc.v0 = vs->v0;
  vc.world = vs->world;
  vc.include_rows = vs->include_rows;
  vc.scatter_hidden = vs->scatter_grad_hidden;
  vc.partials_in = all_partials;
  return run_device(ctx, in, *opts, *out, nullptr, static_cast<cudaStream_t>(stream), plan_out, err, err_len, &vc);
}

void orda_linear_ce_options_default(OrdaLinearCeOptions* out) {
  if (!out) return;
  std::memset(out, 0, sizeof *out);
  out->ignore_index = -100;
  out->reduction = ORDA_REDUCTION_MEAN;
}

// A gradient output of the linear cross entropy: any alignment of its element
// type (an output that TMA cannot address is stored from registers).
static bool grad_out_ok(const void* p, size_t ld, OrdaDType dt, size_t cols) {
  if (!p) return true;
  if (dt != ORDA_DTYPE_BF16 && dt != ORDA_DTYPE_F32) return false;
  return ld >= cols && reinterpret_cast<uintptr_t>(p) % (dt == ORDA_DTYPE_BF16 ? 2 : 4) == 0;
}

int orda_linear_cross_entropy_device(OrdaContext* ctx, const OrdaDeviceMat* hidden, const OrdaDeviceMat* weight,
                                     const int64_t* labels, size_t bt, const OrdaLinearCeOptions* opts,
                                     const OrdaLinearCeOutputs* out, void* stream, char* err, size_t err_len) {
  if (!ctx || !hidden || !weight || (bt > 0 && !labels) || !opts || !out) {
    set_error(err, err_len, "null argument");
    return ORDA_ERR_INVALID;
  }
  if (hidden->rows == 0) {
    set_error(err, err_len, "BT must be > 0");
    return ORDA_ERR_INVALID;
  }
  if (weight->rows == 0 || hidden->cols == 0 || weight->cols != hidden->cols) {
    set_error(err, err_len, "weight must be (V, %zu), got (%zu, %zu)", hidden->cols, weight->rows, weight->cols);
    return ORDA_ERR_INVALID;
  }
  if (bt != hidden->rows) {
    set_error(err, err_len, "labels must have BT=%zu entries, got %zu", hidden->rows, bt);
    return ORDA_ERR_INVALID;
  }
  constexpr size_t kMax = size_t{1} << 30;  // tile coordinates are 32-bit
  if (bt > kMax || weight->rows > kMax || hidden->cols > kMax) {
    set_error(err, err_len, "BT, V and H must be at most 2^30, got %zu, %zu and %zu", bt, weight->rows, hidden->cols);
    return ORDA_ERR_INVALID;
  }
  if (!(opts->label_smoothing >= 0.0f && opts->label_smoothing <= 1.0f)) {
    set_error(err, err_len, "label_smoothing must be in [0,1], got %s", fmt_f32(opts->label_smoothing).c_str());
    return ORDA_ERR_INVALID;
  }
  if (opts->reduction != ORDA_REDUCTION_MEAN && opts->reduction != ORDA_REDUCTION_SUM) {
    set_error(err, err_len, "unknown reduction %d", static_cast<int>(opts->reduction));
    return ORDA_ERR_INVALID;
  }
  if (opts->global_non_ignore < 0) {
    set_error(err, err_len, "global_non_ignore must be >= 0, got %lld", static_cast<long long>(opts->global_non_ignore));
    return ORDA_ERR_INVALID;
  }
  if (!dev_mat_ok(*hidden, true) || !dev_mat_ok(*weight, true)) {
    set_error(err, err_len, "hidden and weight must be bf16, 16-byte aligned, with ld*2 a multiple of 16");
    return ORDA_ERR_INVALID;
  }
  if (!out->loss) {
    set_error(err, err_len, "loss output is required");
    return ORDA_ERR_INVALID;
  }
  if (!grad_out_ok(out->grad_hidden, out->ld_grad_hidden, out->grad_hidden_dtype, hidden->cols) ||
      !grad_out_ok(out->grad_weight, out->ld_grad_weight, out->grad_weight_dtype, hidden->cols)) {
    set_error(err, err_len, "gradient outputs must be bf16 or f32 with ld >= H=%zu", hidden->cols);
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  DeviceScope dev(ctx->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = stream_capturing(st, &ctx->capturing, err, err_len)) return rc;
  const int rc = run_linear_ce(ctx, *hidden, *weight, labels, bt, *opts, *out, st, err, err_len);
  ctx->capturing = false;
  // a call that broke off leaves its counters as a whole one does
  if (rc == ORDA_ERR_CUDA) cudaMemsetAsync(ctx->d_words + 4, 0, 2 * sizeof(int), st);
  return rc;
}

static bool elem_mat_ok(const void* data, size_t rows, size_t cols, size_t ld, OrdaDType dt) {
  if (dt != ORDA_DTYPE_BF16 && dt != ORDA_DTYPE_F32) return false;
  if (!data && rows > 0) return false;
  return ld >= cols && reinterpret_cast<uintptr_t>(data) % (dt == ORDA_DTYPE_BF16 ? 2 : 4) == 0;
}

// Sizes and scale of the two embedding entries.
static int embedding_args_ok(size_t v, size_t h, size_t n, const int64_t* ids, float scale, char* err, size_t err_len) {
  constexpr size_t kMax = size_t{1} << 30;   // positions and keys are 32-bit
  constexpr size_t kMaxH = size_t{1} << 20;  // column blocks are the grid's y
  if (v == 0 || h == 0 || v > kMax || h > kMaxH || n > kMax) {
    set_error(err, err_len, "V must be in [1, 2^30], H in [1, 2^20] and n at most 2^30, got %zu, %zu and %zu", v, h, n);
    return ORDA_ERR_INVALID;
  }
  if (n > 0 && !ids) {
    set_error(err, err_len, "null argument");
    return ORDA_ERR_INVALID;
  }
  if (!(scale - scale == 0.0f)) {
    set_error(err, err_len, "scale must be finite, got %s", fmt_f32(scale).c_str());
    return ORDA_ERR_INVALID;
  }
  return ORDA_OK;
}

int orda_embedding_device(OrdaContext* ctx, const OrdaDeviceMat* table, const int64_t* ids, size_t n, float scale,
                          const OrdaDeviceMatMut* out, void* stream, char* err, size_t err_len) {
  if (!ctx || !table || !out) {
    set_error(err, err_len, "null argument");
    return ORDA_ERR_INVALID;
  }
  if (int rc = embedding_args_ok(table->rows, table->cols, n, ids, scale, err, err_len)) return rc;
  if (out->rows != n || out->cols != table->cols) {
    set_error(err, err_len, "out must be (%zu, %zu), got (%zu, %zu)", n, table->cols, out->rows, out->cols);
    return ORDA_ERR_INVALID;
  }
  if (!elem_mat_ok(table->data, table->rows, table->cols, table->ld, table->dtype) ||
      !elem_mat_ok(out->data, out->rows, out->cols, out->ld, out->dtype)) {
    set_error(err, err_len, "table and out must be bf16 or f32, with ld >= H");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  DeviceScope dev(ctx->device);
  EmbedArgs a;
  a.table = table->data;
  a.ld = static_cast<long long>(table->ld);
  a.v = static_cast<long long>(table->rows);
  a.h = static_cast<long long>(table->cols);
  a.in_bf16 = table->dtype == ORDA_DTYPE_BF16;
  a.out_bf16 = out->dtype == ORDA_DTYPE_BF16;
  a.ids = ids;
  a.n = static_cast<long long>(n);
  a.scale = scale;
  a.out = out->data;
  a.ldo = static_cast<long long>(out->ld);
  a.bad = ctx->d_words + 3;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  bool capturing = false;
  if (int rc = stream_capturing(st, &capturing, err, err_len)) return rc;
  if (!capturing) ctx->last_stream = st;
  if (n == 0) return ORDA_OK;
  launch_embed(a, st);
  ctx->launches += 1;
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ORDA_OK : cuda_fail(e, "embedding", err, err_len);
}

int orda_embedding_grad_device(OrdaContext* ctx, const OrdaDeviceMat* grad_out, const int64_t* ids, size_t n,
                               float scale, int has_padding_id, int64_t padding_id, const OrdaDeviceMatMut* grad_table,
                               int accumulate, void* stream, char* err, size_t err_len) {
  if (!ctx || !grad_out || !grad_table) {
    set_error(err, err_len, "null argument");
    return ORDA_ERR_INVALID;
  }
  if (int rc = embedding_args_ok(grad_table->rows, grad_table->cols, n, ids, scale, err, err_len)) return rc;
  if (grad_out->rows != n || grad_out->cols != grad_table->cols) {
    set_error(err, err_len, "grad_out must be (%zu, %zu), got (%zu, %zu)", n, grad_table->cols, grad_out->rows,
              grad_out->cols);
    return ORDA_ERR_INVALID;
  }
  if (!elem_mat_ok(grad_out->data, grad_out->rows, grad_out->cols, grad_out->ld, grad_out->dtype) ||
      !elem_mat_ok(grad_table->data, grad_table->rows, grad_table->cols, grad_table->ld, grad_table->dtype)) {
    set_error(err, err_len, "grad_out and grad_table must be bf16 or f32, with ld >= H");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  DeviceScope dev(ctx->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  EmbedGradArgs a;
  a.g = grad_out->data;
  a.ldg = static_cast<long long>(grad_out->ld);
  a.v = static_cast<long long>(grad_table->rows);
  a.h = static_cast<long long>(grad_table->cols);
  a.in_bf16 = grad_out->dtype == ORDA_DTYPE_BF16;
  a.out_bf16 = grad_table->dtype == ORDA_DTYPE_BF16;
  a.ids = ids;
  a.n = static_cast<long long>(n);
  a.scale = scale;
  a.has_padding = has_padding_id;
  a.padding_id = padding_id;
  a.out = grad_table->data;
  a.ldo = static_cast<long long>(grad_table->ld);
  a.accumulate = accumulate;
  a.bad = ctx->d_words + 3;
  ctx->vocab_ready = false;  // the workspace no longer holds a vocabulary forward phase
  bool capturing = false;
  if (int rc = stream_capturing(st, &capturing, err, err_len)) return rc;
  if (int rc = call_ws(ctx, embed_grad_workspace(a), capturing, err, err_len)) return rc;
  int nl = 0;
  const cudaError_t e = launch_embed_grad(a, ctx->ws, ctx->num_sms, st, &nl);
  ctx->launches += static_cast<uint64_t>(nl);
  if (!capturing) ctx->last_stream = st;
  return e == cudaSuccess ? ORDA_OK : cuda_fail(e, "embedding gradient", err, err_len);
}

int orda_quantize_grad_w_device(OrdaContext* ctx, float* grad_w, size_t v, size_t h, size_t ld, const int64_t* labels,
                                size_t bt, int64_t ignore_index, int stochastic, uint64_t seed, int8_t* q, float* scale,
                                void* stream, char* err, size_t err_len) {
  if (!ctx || !grad_w || (bt > 0 && !labels) || ld < h) {
    set_error(err, err_len, "invalid argument");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // target-row flags live in the context workspace
  ctx->vocab_ready = false;
  if (ensure_ws(ctx, round_up(v, 256)) != cudaSuccess) {
    set_error(err, err_len, "device workspace allocation failed");
    return ORDA_ERR_OOM;
  }
  uint8_t* flags = static_cast<uint8_t*>(ctx->ws);
  cudaError_t e = cudaMemsetAsync(flags, 0, v, st);
  if (e != cudaSuccess) return cuda_fail(e, "memset", err, err_len);
  launch_target_flags(labels, static_cast<long long>(bt), static_cast<long long>(v), ignore_index, flags, st);
  ctx->launches += 2;
  launch_quant(grad_w, static_cast<long long>(v), static_cast<long long>(h), static_cast<long long>(ld), flags,
               stochastic, seed, q, scale, st);
  if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "quantise", err, err_len);
  ctx->last_stream = st;
  return ORDA_OK;
}

int orda_gemm_bf16_device(OrdaContext* ctx, const void* a, size_t lda, int a_kind, const void* b, size_t ldb, int b_kind,
                          float* c, size_t ldc, size_t m, size_t n, size_t k, float alpha, float beta, void* stream,
                          char* err, size_t err_len) {
  if (!ctx || !a || !b || !c || k == 0) {
    set_error(err, err_len, "invalid argument (null pointer or k == 0)");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  GemmDesc gd;
  gd.a_mn_major = a_kind == 1;
  gd.b_mn_major = b_kind == 1;
  gd.a[0] = a_kind == 1 ? MatRef{a, static_cast<long long>(k), static_cast<long long>(m), static_cast<long long>(lda)}
                        : MatRef{a, static_cast<long long>(m), static_cast<long long>(k), static_cast<long long>(lda)};
  gd.b[0] = b_kind == 1 ? MatRef{b, static_cast<long long>(k), static_cast<long long>(n), static_cast<long long>(ldb)}
                        : MatRef{b, static_cast<long long>(n), static_cast<long long>(k), static_cast<long long>(ldb)};
  gd.k_seg[0] = static_cast<long long>(k);
  gd.M = static_cast<long long>(m);
  gd.N = static_cast<long long>(n);
  gd.raster_n_fastest = m > n;
  gd.status = ctx->d_words;
  gd.args.out0 = c;
  gd.args.ld0 = static_cast<long long>(ldc);
  gd.args.alpha = alpha;
  gd.args.beta = beta;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(ctx->d_words, 0, sizeof(int), st);
  if (e != cudaSuccess) return cuda_fail(e, "memset", err, err_len);
  const char* why = nullptr;
  int nl = 0;
  gd.demote_kept = ctx->l2_set;
  gd.launches = &nl;
  e = gemm_launch(gd, ctx->num_sms, st, &why);
  ctx->launches += static_cast<uint64_t>(nl);
  if (e != cudaSuccess) return cuda_fail(e, why ? why : "GEMM", err, err_len);
  ctx->last_stream = st;
  return ORDA_OK;
}

void orda_context_set_concurrency(OrdaContext* ctx, int spare_sms) {
  if (ctx) ctx->spare_sms = std::max(0, std::min(spare_sms, 32));
}

void orda_context_enable_timing(OrdaContext* ctx, int enable) {
  if (ctx) ctx->timing = enable != 0;
}

int orda_context_phase_times(OrdaContext* ctx, double* ms_out, uint64_t* launches_out) {
  if (!ctx) return 0;
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  for (auto& pe : ctx->pending) {
    cudaEventSynchronize(pe.end);
    float ms = 0.0f;
    if (cudaEventElapsedTime(&ms, pe.begin, pe.end) == cudaSuccess) ctx->phase_ms[pe.phase] += ms;
    ctx->phase_launches[pe.phase] += static_cast<uint64_t>(pe.launches);
    ctx->event_pool.push_back(pe.begin);
    ctx->event_pool.push_back(pe.end);
  }
  ctx->pending.clear();
  for (int i = 0; i < ORDA_NUM_PHASES; ++i) {
    if (ms_out) ms_out[i] = ctx->phase_ms[i];
    if (launches_out) launches_out[i] = ctx->phase_launches[i];
  }
  return ORDA_NUM_PHASES;
}

void orda_context_reset_timing(OrdaContext* ctx) {
  if (!ctx) return;
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  for (auto& pe : ctx->pending) {
    cudaEventSynchronize(pe.end);
    ctx->event_pool.push_back(pe.begin);
    ctx->event_pool.push_back(pe.end);
  }
  ctx->pending.clear();
  for (int i = 0; i < ORDA_NUM_PHASES; ++i) {
    ctx->phase_ms[i] = 0.0;
    ctx->phase_launches[i] = 0;
  }
}

uint64_t orda_context_launch_count(const OrdaContext* ctx) { return ctx ? ctx->launches : 0; }

int orda_context_selftest_bounded_wait(OrdaContext* ctx, uint32_t limit_us, void* stream, char* err,
                                       size_t err_len) {
  if (!ctx || limit_us == 0 || limit_us > 1000000) {
    set_error(err, err_len, "invalid argument (limit_us must be in (0, 1e6])");
    return ORDA_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(ctx->d_words, 0, sizeof(int), st);
  if (e == cudaSuccess) e = launch_bounded_wait_selftest(ctx->d_words, static_cast<uint64_t>(limit_us) * 1000, st);
  if (e != cudaSuccess) return cuda_fail(e, "bounded-wait self-test", err, err_len);
  ctx->launches += 1;
  ctx->last_stream = st;
  return ORDA_OK;
}

// ------------------------------------------------------------ host-Mat entry

int orda_distillation_loss(const OrdaMatF32* student_hidden, const OrdaMatF32* weight, const int64_t* labels,
                           size_t n_labels, const OrdaTeacher* teacher, const OrdaLossOptions* opts, OrdaOutput* out,
                           char* err, size_t err_len) {
  if (!student_hidden || !weight || !teacher || !opts || !out) {
    set_error(err, err_len, "null argument");
    return ORDA_ERR_INVALID;
  }
  std::memset(out, 0, sizeof *out);
  size_t v = 0, h = 0, bt = 0;
  if (int rc = orda_validate(student_hidden, weight, labels, n_labels, teacher, opts, &v, &h, &bt, err, err_len))
    return rc;
  if (opts->backend == ORDA_BACKEND_CPU) {
    set_error(err, err_len, "Backend::Cpu is not available: this library is the B200 path and has no CPU backend");
    return ORDA_ERR_BACKEND;
  }
  const float w_t = opts->has_teacher_ce_weight ? opts->teacher_ce_weight : orda_default_teacher_ce_weight(teacher->mode);
  if (w_t < 0.0f) {
    set_error(err, err_len, "teacher_ce_weight must be >= 0, got %s", fmt_f32(w_t).c_str());
    return ORDA_ERR_INVALID;
  }
  if (!orda_is_available()) {
    set_error(err, err_len,
              opts->backend == ORDA_BACKEND_CUDA
                  ? "Backend::Cuda requested but no sm_100 CUDA device is available"
                  : "Backend::Auto found no sm_100 CUDA device (this library has no CPU path)");
    return ORDA_ERR_BACKEND;
  }
  int dev = 0;
  cudaGetDevice(&dev);
  OrdaContext* ctx = nullptr;
  {
    std::lock_guard<std::mutex> lock(g_default_mu);
    if (dev < 0 || dev >= 64) dev = 0;
    if (!g_default_ctx[dev]) {
      if (int rc = orda_context_create(dev, &g_default_ctx[dev], err, err_len)) return rc;
    }
    ctx = g_default_ctx[dev];
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  cudaSetDevice(ctx->device);
  // compute, host->device and device->host streams
  for (cudaStream_t* sp : {&ctx->own_stream, &ctx->copy_in, &ctx->copy_out})
    if (!*sp) cudaStreamCreateWithFlags(sp, cudaStreamNonBlocking);
  cudaStream_t st = ctx->own_stream, cin = ctx->copy_in, cout = ctx->copy_out;

  const OrdaTeacherMode mode = teacher->mode;
  const bool live = mode == ORDA_TEACHER_TIED || mode == ORDA_TEACHER_SEPARATE;
  const bool pre = mode == ORDA_TEACHER_PRECOMPUTED;
  const size_t ht = mode == ORDA_TEACHER_SEPARATE ? teacher->hidden.cols : h;
  const bool tgrad = w_t > 0.0f && live;
  const size_t ldh = round_up(h, 8), ldht = round_up(ht, 8), ldtl = round_up(v, 4);

  // Pipeline groups. Precomputed teacher logits (the largest input) are
  // copied in row slabs of about kTeacherSlab bytes; the device runs the
  // forward and backward work of a slab's rows (whole chunks of the
  // resolver's plan) while the next slab is in flight, and each backward
  // group's grad_hidden rows go back to the host while later slabs arrive.
  const size_t kTeacherSlab = g_host_slab_bytes.load();
  constexpr size_t kRingBytes = size_t{64} << 20;  // f32 staging of the bf16 inputs
  const OrdaChunkPlan plan0 = resolve_chunk_size(bt, opts->chunk_size, true, v, opts->config.has_max_chunks != 0,
                                                 opts->config.max_chunks);
  size_t group_rows = 0;
  if (pre && bt * v * 4 > 2 * kTeacherSlab && plan0.chunk_size > 0) {
    size_t rows = kTeacherSlab / (v * 4) / plan0.chunk_size * plan0.chunk_size;
    rows = std::max(rows, plan0.chunk_size);
    if (rows < bt) group_rows = rows;
  }
  const size_t n_groups = group_rows ? ceil_div(bt, group_rows) : 1;

  // With the INT8 round trip, grad_W comes back compressed: its INT8 codes,
  // row scales and exact target rows (0.66 GB instead of 2.15 GB at c4), and
  // the host forms q * s (host_dequant.cc: the device's own float multiply,
  // so the values are bit-identical). ORDA_HOST_DEQUANT=0 copies the fp32
  // grad_W instead (a diagnostic switch). Target rows: non-ignored labels,
  // the rule of target_flags_kernel.
  // host workers of the conversions and the dequantisation (one per core,
  // at most 16: about 90 GB/s of fp32 converted on a 16-core host); without
  // them the call copies fp32 both ways
  const bool want_deq = opts->config.quantize_grad_weight != 0 && host_dequant_enabled();
  const int conv_mode = host_convert_mode();
  const bool want_conv = conv_mode != 0;
  std::unique_ptr<HostPool> pool;
  if (want_deq || want_conv) {
    try {
      pool = std::make_unique<HostPool>(std::max(1u, std::min(16u, std::thread::hardware_concurrency())));
    } catch (...) {
      pool.reset();
    }
  }
  const bool host_deq = want_deq && pool;
  std::vector<int32_t> exact_pos, exact_idx;
  if (host_deq) {
    std::vector<uint8_t> is_target(v, 0);
    for (size_t i = 0; i < bt; ++i) {
      const int64_t t = labels[i];
      if (t != opts->ignore_index && t >= 0 && static_cast<size_t>(t) < v) is_target[static_cast<size_t>(t)] = 1;
    }
    exact_pos.assign(v, -1);
    for (size_t r = 0; r < v; ++r) {
      if (!is_target[r]) continue;
      exact_pos[r] = static_cast<int32_t>(exact_idx.size());
      exact_idx.push_back(static_cast<int32_t>(r));
    }
  }
  const size_t n_exact = exact_idx.size();

  // device staging layout
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = round_up(off + bytes, 256);
    return o;
  };
  const size_t o_hs = take(bt * ldh * 2), o_w = take(v * ldh * 2);
  const size_t o_ht = take(live ? bt * ldht * 2 : 0), o_wt = take(mode == ORDA_TEACHER_SEPARATE ? v * ldht * 2 : 0);
  const size_t o_tl = take(pre ? bt * ldtl * 4 : 0);
  const size_t o_lab = take(bt * 8);
  const size_t o_ghs = take(bt * h * 4), o_gw = take(v * h * 4);
  const size_t o_ght = take(tgrad ? bt * ht * 4 : 0), o_gwt = take(tgrad && mode == ORDA_TEACHER_SEPARATE ? v * ht * 4 : 0);
  const size_t o_sc = take(4 * sizeof(float));
  // Host conversion: a ring of kRing page-locked bf16 chunks of kChunk
  // elements feeds the copies; bf16 teacher-logit chunks land in a device
  // scratch chunk and are widened into the fp32 teacher rows. A chunk the
  // host does not convert crosses as fp32 (GEMM operands through the device
  // ring and the conversion kernel), so the ring holds a whole chunk.
  const bool host_conv = want_conv && pool;
  constexpr size_t kChunk = size_t{32} << 20;  // elements (64 MiB of bf16)
  constexpr int kRing = 3;
  const size_t ring_bytes = std::max(std::max(kRingBytes, std::max(h, ht) * 4), host_conv ? kChunk * 4 : 0);
  const size_t o_ring = take(ring_bytes);
  const size_t o_q = take(host_deq ? v * h : 0), o_qs = take(host_deq ? v * 4 : 0);
  const size_t o_xidx = take(n_exact * 4), o_xrows = take(n_exact * h * 4);
  const size_t o_tscr = take(host_conv && pre ? std::max(kChunk, v) * 2 : 0);
  if (ctx->stage_bytes < off) {
    cudaFree(ctx->stage);
    ctx->stage = nullptr;
    ctx->stage_bytes = 0;
    cudaError_t e = cudaMalloc(&ctx->stage, off);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_error(err, err_len, "device staging allocation of %zu bytes failed", off);
      return ORDA_ERR_OOM;
    }
    ctx->stage_bytes = off;
  }
  uint8_t* S = static_cast<uint8_t*>(ctx->stage);

  // library-owned page-locked outputs
  auto host_mat = [&](size_t rows, size_t cols, OrdaMatOut& m) -> bool {
    m.rows = rows;
    m.cols = cols;
    m.data = pinned_alloc(std::max<size_t>(rows * cols, 1) * 4);
    return m.data != nullptr;
  };
  float* sc_host = pinned_alloc(4 * sizeof(float));
  bool ok_alloc = sc_host && host_mat(bt, h, out->grad_student_hidden) && host_mat(v, h, out->grad_weight);
  if (ok_alloc && tgrad) ok_alloc = host_mat(bt, ht, out->grad_teacher_hidden);
  if (ok_alloc && tgrad && mode == ORDA_TEACHER_SEPARATE) ok_alloc = host_mat(v, ht, out->grad_teacher_weight);
  // page-locked landing buffers of the compressed grad_W
  int8_t* q_host = nullptr;
  float *qs_host = nullptr, *xrows_host = nullptr;
  if (ok_alloc && host_deq) {
    q_host = reinterpret_cast<int8_t*>(pinned_alloc(v * h));
    qs_host = pinned_alloc(v * 4);
    xrows_host = pinned_alloc(n_exact * h * 4);
    ok_alloc = q_host && qs_host && xrows_host;
  }
  uint16_t* ring_host[kRing] = {nullptr, nullptr, nullptr};
  if (ok_alloc && host_conv) {
    for (int b = 0; b < kRing && ok_alloc; ++b) {
      ring_host[b] = reinterpret_cast<uint16_t*>(pinned_alloc(std::max(kChunk, std::max(std::max(h, ht), v)) * 2));
      ok_alloc = ring_host[b] != nullptr;
    }
  }
  auto release_landing = [&]() {
    pinned_release(q_host);
    pinned_release(qs_host);
    pinned_release(xrows_host);
    for (int b = 0; b < kRing; ++b) pinned_release(ring_host[b]);
  };

  if (!ok_alloc) {
    release_landing();
    pinned_release(sc_host);
    orda_output_free(out);
    set_error(err, err_len, "page-locked host allocation for the outputs failed");
    return ORDA_ERR_OOM;
  }

  // events, destroyed when the call ends
  std::vector<cudaEvent_t> events;
  auto mk_event = [&]() {
    cudaEvent_t e = nullptr;
    cudaEventCreateWithFlags(&e, cudaEventDisableTiming);
    events.push_back(e);
    return e;
  };
  cudaEvent_t ev_inputs = mk_event();
  std::vector<cudaEvent_t> ev_teacher;
  for (size_t k = 0; k < (pre ? n_groups : 0); ++k) ev_teacher.push_back(mk_event());

  // ---- copier thread: every host->device copy on `cin`, in the order the
  // device needs them (labels, the bf16 operands through the f32 ring and a
  // conversion kernel, then the teacher-logit slabs), recording an event
  // after each stage and announcing it. A separate thread keeps pageable
  // sources (whose copies return only when consumed) from delaying the
  // kernel launches of the main thread.
  struct Feed {
    std::mutex mu;
    std::condition_variable cv;
    size_t announced = 0;  // stages whose events are recorded
    cudaError_t error = cudaSuccess;
  } feed;
  auto announce = [&feed](size_t n, cudaError_t e) {
    std::lock_guard<std::mutex> lk(feed.mu);
    feed.announced = n;
    if (e != cudaSuccess && feed.error == cudaSuccess) feed.error = e;
    feed.cv.notify_all();
  };
  float* ring = reinterpret_cast<float*>(S + o_ring);
  cudaEvent_t ev_ring[kRing] = {nullptr, nullptr, nullptr};
  if (host_conv)
    for (int b = 0; b < kRing; ++b) ev_ring[b] = mk_event();
  cudaEvent_t ev_queue = host_conv ? mk_event() : nullptr;  // the copier's last copy
  size_t up_copier = 0;                  // bytes the copier sends (read after it joins)
  size_t up_main = 0, down_main = 0;     // bytes the calling thread copies
  std::thread copier([&]() {
    cudaSetDevice(ctx->device);
    cudaError_t e = cudaMemcpyAsync(S + o_lab, labels, bt * 8, cudaMemcpyHostToDevice, cin);
    up_copier += bt * 8;
    // next page-locked ring chunk, once the copy that last read it is done
    int slot = 0;
    bool used[kRing] = {false, false, false};
    auto next_chunk = [&](int* b) -> uint16_t* {
      *b = slot;
      slot = (slot + 1) % kRing;
      if (used[*b] && e == cudaSuccess) e = cudaEventSynchronize(ev_ring[*b]);
      used[*b] = true;
      return ring_host[*b];
    };
    // f32 host rows -> bf16 on the host -> device rows
    // Host memory bandwidth, not only PCIe, bounds these copies: a chunk
    // converted on the host costs 8 bytes of host memory traffic per element
    // (read fp32, write bf16, the copy reads bf16) against 4 for an fp32
    // copy, which moves twice the bytes over PCIe. So the copier converts
    // while the copy engine is busy and sends the next chunk as fp32 when the
    // engine has run dry: the split follows the host's speed.
    bool queued = false;
    auto engine_idle = [&]() -> bool {
      if (conv_mode == 2) return false;
      if (!queued) return true;
      const cudaError_t q = cudaEventQuery(ev_queue);
      if (q == cudaErrorNotReady) {
        cudaGetLastError();  // not an error: the copy is still running
        return false;
      }
      return true;
    };
    auto mark_queued = [&]() {
      if (e == cudaSuccess) e = cudaEventRecord(ev_queue, cin);
      queued = true;
    };
    auto put_bf16_host = [&](const OrdaMatF32& m, size_t ld, size_t o) {
      const size_t per = std::max<size_t>(1, kChunk / std::max<size_t>(m.cols, 1));
      for (size_t r0 = 0; r0 < m.rows && e == cudaSuccess; r0 += per) {
        const size_t n = std::min(per, m.rows - r0), cnt = n * m.cols;
        const float* src = m.data + r0 * m.cols;
        if (engine_idle()) {
          // fp32 through the device ring and the conversion kernel
          e = cudaMemcpyAsync(ring, src, cnt * 4, cudaMemcpyHostToDevice, cin);
          up_copier += cnt * 4;
          if (e == cudaSuccess) {
            launch_f32_to_bf16(ring, static_cast<long long>(n), static_cast<long long>(m.cols),
                               reinterpret_cast<uint16_t*>(S + o) + r0 * ld, static_cast<long long>(ld), cin);
            e = cudaGetLastError();
          }
          mark_queued();
          continue;
        }
        int b;
        uint16_t* buf = next_chunk(&b);
        if (e != cudaSuccess) break;
        pool->run([&](unsigned w, unsigned nw) {
          size_t a, z;
          split_range(cnt, nw, w, &a, &z);
          f32_to_bf16_host(src + a, z - a, buf + a);
        });
        e = cudaMemcpy2DAsync(S + o + r0 * ld * 2, ld * 2, buf, m.cols * 2, m.cols * 2, n, cudaMemcpyHostToDevice,
                              cin);
        up_copier += cnt * 2;
        if (e == cudaSuccess) e = cudaEventRecord(ev_ring[b], cin);
        mark_queued();
      }
    };
    // f32 host rows -> ring -> bf16 device rows (one stream: each slab's copy
    // follows the conversion of the previous one, so one ring buffer serves)
    auto put_bf16 = [&](const OrdaMatF32& m, size_t ld, size_t o) {
      const size_t per = std::max<size_t>(1, ring_bytes / (m.cols * 4));
      for (size_t r0 = 0; r0 < m.rows && e == cudaSuccess; r0 += per) {
        const size_t n = std::min(per, m.rows - r0);
        e = cudaMemcpyAsync(ring, m.data + r0 * m.cols, n * m.cols * 4, cudaMemcpyHostToDevice, cin);
        up_copier += n * m.cols * 4;
        if (e != cudaSuccess) break;
        launch_f32_to_bf16(ring, static_cast<long long>(n), static_cast<long long>(m.cols),
                           reinterpret_cast<uint16_t*>(S + o) + r0 * ld, static_cast<long long>(ld), cin);
        e = cudaGetLastError();
      }
    };
    auto put = [&](const OrdaMatF32& m, size_t ld, size_t o) {
      if (host_conv) put_bf16_host(m, ld, o);
      else put_bf16(m, ld, o);
    };
    if (e == cudaSuccess) put(*student_hidden, ldh, o_hs);
    if (e == cudaSuccess) put(*weight, ldh, o_w);
    if (e == cudaSuccess && live) put(teacher->hidden, ldht, o_ht);
    if (e == cudaSuccess && mode == ORDA_TEACHER_SEPARATE) put(teacher->weight, ldht, o_wt);
    if (e == cudaSuccess) e = cudaEventRecord(ev_inputs, cin);
    if (e != cudaSuccess) {
      announce(SIZE_MAX, e);
      return;
    }
    announce(1, cudaSuccess);
    // Teacher logits: a chunk whose values are all bf16 values crosses as
    // bf16 and is widened on the device (exact); otherwise as fp32, and
    // after the first such chunk the rest of the call copies fp32 directly.
    bool try_bf16 = host_conv;
    auto put_teacher_rows = [&](size_t r0, size_t n) {
      if (try_bf16) {
        const size_t per = std::max<size_t>(1, kChunk / v);
        for (size_t c0 = r0; c0 < r0 + n && e == cudaSuccess && try_bf16; c0 += per) {
          const size_t m = std::min(per, r0 + n - c0), cnt = m * v;
          if (engine_idle()) {
            e = cudaMemcpy2DAsync(S + o_tl + c0 * ldtl * 4, ldtl * 4, teacher->logits.data + c0 * v, v * 4, v * 4, m,
                                  cudaMemcpyHostToDevice, cin);
            up_copier += m * v * 4;
            mark_queued();
            continue;
          }
          int b;
          uint16_t* buf = next_chunk(&b);
          if (e != cudaSuccess) return;
          const float* src = teacher->logits.data + c0 * v;
          unsigned char exact[64];
          pool->run([&](unsigned w, unsigned nw) {
            size_t a, z;
            split_range(cnt, nw, w, &a, &z);
            exact[w] = f32_to_bf16_if_exact(src + a, z - a, buf + a) ? 1 : 0;
          });
          for (unsigned w = 0; w < pool->size(); ++w) try_bf16 = try_bf16 && exact[w];
          if (!try_bf16) {
            // this chunk and the rest of the rows as fp32
            e = cudaMemcpy2DAsync(S + o_tl + c0 * ldtl * 4, ldtl * 4, teacher->logits.data + c0 * v, v * 4, v * 4,
                                  r0 + n - c0, cudaMemcpyHostToDevice, cin);
            up_copier += (r0 + n - c0) * v * 4;
            mark_queued();
            return;
          }
          e = cudaMemcpyAsync(S + o_tscr, buf, cnt * 2, cudaMemcpyHostToDevice, cin);
          up_copier += cnt * 2;
          if (e == cudaSuccess) e = cudaEventRecord(ev_ring[b], cin);
          if (e == cudaSuccess) {
            launch_bf16_rows_to_f32(reinterpret_cast<const uint16_t*>(S + o_tscr), static_cast<long long>(m),
                                    static_cast<long long>(v), reinterpret_cast<float*>(S + o_tl + c0 * ldtl * 4),
                                    static_cast<long long>(ldtl), cin);
            e = cudaGetLastError();
          }
          mark_queued();
        }
        return;
      }
      e = cudaMemcpy2DAsync(S + o_tl + r0 * ldtl * 4, ldtl * 4, teacher->logits.data + r0 * v, v * 4, v * 4, n,
                            cudaMemcpyHostToDevice, cin);
      up_copier += n * v * 4;
      if (host_conv) mark_queued();
    };
    for (size_t k = 0; k < ev_teacher.size(); ++k) {
      const size_t r0 = k * (group_rows ? group_rows : bt);
      const size_t n = std::min(group_rows ? group_rows : bt, bt - r0);
      put_teacher_rows(r0, n);
      if (e == cudaSuccess) e = cudaEventRecord(ev_teacher[k], cin);
      if (e != cudaSuccess) {
        announce(SIZE_MAX, e);
        return;
      }
      announce(k + 2, cudaSuccess);
    }
  });
  // waits (host) until stage n is announced; then its event may be waited on
  auto wait_stage = [&](size_t n) -> int {
    std::unique_lock<std::mutex> lk(feed.mu);
    feed.cv.wait(lk, [&] { return feed.announced >= n || feed.error != cudaSuccess; });
    if (feed.error != cudaSuccess) return cuda_fail(feed.error, "host->device copy", err, err_len);
    return ORDA_OK;
  };
  auto finish = [&](int rc) {
    if (copier.joinable()) copier.join();
    if (rc == ORDA_OK && feed.error != cudaSuccess) rc = cuda_fail(feed.error, "host->device copy", err, err_len);
    if (rc == ORDA_OK) {
      cudaError_t e = cudaStreamSynchronize(cout);
      if (e != cudaSuccess) rc = cuda_fail(e, "device->host copy", err, err_len);
    }
    if (rc == ORDA_OK) rc = check_status(ctx, err, err_len);
    if (rc != ORDA_OK) {
      // nothing may still write into the outputs when they are released
      cudaStreamSynchronize(cin);
      cudaStreamSynchronize(st);
      cudaStreamSynchronize(cout);
    }
    for (cudaEvent_t e : events) cudaEventDestroy(e);
    if (rc == ORDA_OK) {
      out->loss = sc_host[0];
      out->student_ce = sc_host[1];
      out->teacher_ce = sc_host[2];
      out->kl = sc_host[3];
      g_last_h2d.store(up_copier + up_main);
      g_last_d2h.store(down_main);
    } else {
      orda_output_free(out);
    }
    pinned_release(sc_host);
    release_landing();
    return rc;
  };

  OrdaDeviceOutputs dout{};
  dout.grad_student_hidden = reinterpret_cast<float*>(S + o_ghs);
  dout.ld_grad_student_hidden = h;
  dout.grad_weight = reinterpret_cast<float*>(S + o_gw);
  dout.ld_grad_weight = h;
  if (tgrad) {
    dout.grad_teacher_hidden = reinterpret_cast<float*>(S + o_ght);
    dout.ld_grad_teacher_hidden = ht;
  }
  if (tgrad && mode == ORDA_TEACHER_SEPARATE) {
    dout.grad_teacher_weight = reinterpret_cast<float*>(S + o_gwt);
    dout.ld_grad_teacher_weight = ht;
  }
  dout.scalars = reinterpret_cast<float*>(S + o_sc);
  if (host_deq) {
    dout.grad_weight_q = reinterpret_cast<int8_t*>(S + o_q);
    dout.grad_weight_scale = reinterpret_cast<float*>(S + o_qs);
  }

  DevInputs in;
  in.bt = bt;
  in.h = h;
  in.v = v;
  in.ht_dim = ht;
  in.mode = mode;
  in.labels = reinterpret_cast<const int64_t*>(S + o_lab);
  in.hs = MatRef{S + o_hs, static_cast<long long>(bt), static_cast<long long>(h), static_cast<long long>(ldh)};
  in.w = MatRef{S + o_w, static_cast<long long>(v), static_cast<long long>(h), static_cast<long long>(ldh)};
  if (live) in.ht = MatRef{S + o_ht, static_cast<long long>(bt), static_cast<long long>(ht), static_cast<long long>(ldht)};
  if (mode == ORDA_TEACHER_SEPARATE)
    in.wt = MatRef{S + o_wt, static_cast<long long>(v), static_cast<long long>(ht), static_cast<long long>(ldht)};
  if (pre) {
    in.t_logits = S + o_tl;
    in.ld_t_logits = static_cast<long long>(ldtl);
    in.t_logits_bf16 = false;
  }

  if (int rc = wait_stage(1)) return finish(rc);
  if (cudaError_t e = cudaStreamWaitEvent(st, ev_inputs, 0); e != cudaSuccess) return finish(cuda_fail(e, "event wait", err, err_len));
  if (n_exact > 0) {
    cudaError_t e = cudaMemcpyAsync(S + o_xidx, exact_idx.data(), n_exact * 4, cudaMemcpyHostToDevice, st);
    up_main += n_exact * 4;
    if (e != cudaSuccess) return finish(cuda_fail(e, "host->device copy", err, err_len));
  }
  HostPipe hp;
  hp.group_rows = group_rows;
  if (pre) {
    // the row pass of rows [s, s + n) needs the slabs that hold them (copies
    // on one stream complete in order: the last slab's event covers all)
    hp.before_rows = [&](size_t s0, size_t n) -> int {
      const size_t k = group_rows ? (s0 + n - 1) / group_rows : 0;
      if (int rc = wait_stage(k + 2)) return rc;
      cudaError_t e = cudaStreamWaitEvent(st, ev_teacher[k], 0);
      return e == cudaSuccess ? ORDA_OK : cuda_fail(e, "event wait", err, err_len);
    };
  }
  hp.after_dgrad = [&](size_t g0, size_t g1) -> int {
    cudaEvent_t ev = mk_event();
    cudaError_t e = cudaEventRecord(ev, st);
    if (e == cudaSuccess) e = cudaStreamWaitEvent(cout, ev, 0);
    if (e == cudaSuccess)
      e = cudaMemcpyAsync(out->grad_student_hidden.data + g0 * h, dout.grad_student_hidden + g0 * h,
                          (g1 - g0) * h * 4, cudaMemcpyDeviceToHost, cout);
    down_main += (g1 - g0) * h * 4;
    if (e == cudaSuccess && tgrad) {
      e = cudaMemcpyAsync(out->grad_teacher_hidden.data + g0 * ht, dout.grad_teacher_hidden + g0 * ht,
                          (g1 - g0) * ht * 4, cudaMemcpyDeviceToHost, cout);
      down_main += (g1 - g0) * ht * 4;
    }
    return e == cudaSuccess ? ORDA_OK : cuda_fail(e, "device->host copy", err, err_len);
  };
  OrdaChunkPlan plan{};
  if (int rc = run_device(ctx, in, *opts, dout, nullptr, st, &plan, err, err_len, nullptr, &hp)) return finish(rc);

  // grad_W (after the INT8 round trip, if any) and the scalars
  float* xrows_dev = reinterpret_cast<float*>(S + o_xrows);
  if (n_exact > 0) {
    launch_gather_rows(dout.grad_weight, static_cast<long long>(h), reinterpret_cast<const int32_t*>(S + o_xidx),
                       static_cast<long long>(n_exact), static_cast<long long>(h), xrows_dev, st);
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return finish(cuda_fail(e, "gather rows", err, err_len));
  }
  cudaEvent_t ev_done = mk_event();
  cudaError_t e = cudaEventRecord(ev_done, st);
  if (e == cudaSuccess) e = cudaStreamWaitEvent(cout, ev_done, 0);
  // compressed grad_W: scales and exact rows first, then the codes in row
  // slabs, each announced by an event so the host dequantises slab k while
  // slab k + 1 is in flight
  std::vector<std::pair<size_t, cudaEvent_t>> slabs;  // (end row, event)
  cudaEvent_t ev_meta = nullptr;
  if (host_deq) {
    if (e == cudaSuccess) e = cudaMemcpyAsync(qs_host, dout.grad_weight_scale, v * 4, cudaMemcpyDeviceToHost, cout);
    if (e == cudaSuccess && n_exact > 0)
      e = cudaMemcpyAsync(xrows_host, xrows_dev, n_exact * h * 4, cudaMemcpyDeviceToHost, cout);
    down_main += v * 4 + n_exact * h * 4 + v * h;
    if (e == cudaSuccess) e = cudaEventRecord(ev_meta = mk_event(), cout);
    const size_t slab_rows = std::max<size_t>(1, (size_t{32} << 20) / std::max<size_t>(h, 1));
    for (size_t r0 = 0; r0 < v && e == cudaSuccess; r0 += slab_rows) {
      const size_t r1 = std::min(v, r0 + slab_rows);
      e = cudaMemcpyAsync(q_host + r0 * h, dout.grad_weight_q + r0 * h, (r1 - r0) * h, cudaMemcpyDeviceToHost, cout);
      cudaEvent_t ev = mk_event();
      if (e == cudaSuccess) e = cudaEventRecord(ev, cout);
      slabs.emplace_back(r1, ev);
    }
  } else if (e == cudaSuccess) {
    e = cudaMemcpyAsync(out->grad_weight.data, dout.grad_weight, v * h * 4, cudaMemcpyDeviceToHost, cout);
    down_main += v * h * 4;
  }
  if (e == cudaSuccess && tgrad && mode == ORDA_TEACHER_SEPARATE) {
    e = cudaMemcpyAsync(out->grad_teacher_weight.data, dout.grad_teacher_weight, v * ht * 4, cudaMemcpyDeviceToHost,
                        cout);
    down_main += v * ht * 4;
  }
  if (e == cudaSuccess) e = cudaMemcpyAsync(sc_host, dout.scalars, 4 * sizeof(float), cudaMemcpyDeviceToHost, cout);
  down_main += 4 * sizeof(float);
  if (e != cudaSuccess) return finish(cuda_fail(e, "device->host copy", err, err_len));
  if (host_deq) {
    // the workers split each slab's rows once the slab has landed (the
    // copier, the pool's other user, has finished)
    if (copier.joinable()) copier.join();
    e = cudaEventSynchronize(ev_meta);
    size_t r0 = 0;
    for (size_t k = 0; k < slabs.size() && e == cudaSuccess; ++k) {
      const size_t r1 = slabs[k].first;
      e = cudaEventSynchronize(slabs[k].second);
      if (e != cudaSuccess) break;
      pool->run([&](unsigned w, unsigned nw) {
        size_t a, z;
        split_range(r1 - r0, nw, w, &a, &z);
        if (a < z) dequant_rows_host(q_host, qs_host, exact_pos.data(), xrows_host, r0 + a, r0 + z, h,
                                     out->grad_weight.data);
      });
      r0 = r1;
    }
    if (e != cudaSuccess) return finish(cuda_fail(e, "device->host copy", err, err_len));
  }
  out->chunk_plan = plan;
  return finish(ORDA_OK);
}

void orda_set_host_slab_bytes(size_t bytes) { g_host_slab_bytes.store(bytes ? bytes : (size_t{512} << 20)); }

void orda_last_call_bytes(uint64_t* h2d, uint64_t* d2h) {
  if (h2d) *h2d = g_last_h2d.load();
  if (d2h) *d2h = g_last_d2h.load();
}

void orda_output_free(OrdaOutput* out) {
  if (!out) return;
  pinned_release(out->grad_student_hidden.data);
  pinned_release(out->grad_weight.data);
  pinned_release(out->grad_teacher_hidden.data);
  pinned_release(out->grad_teacher_weight.data);
  out->grad_student_hidden.data = nullptr;
  out->grad_weight.data = nullptr;
  out->grad_teacher_hidden.data = nullptr;
  out->grad_teacher_weight.data = nullptr;
}

}  // extern "C"
