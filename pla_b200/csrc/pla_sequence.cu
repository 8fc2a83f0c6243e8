// C ABI of the sequence operators (declarations and contract:
// include/pla_b200.h): argument checks, the choice of a kernel variant, and
// the launches on the caller's stream.  No allocation, no synchronisation.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <numeric>
#include <type_traits>

#include "../../include/pla_b200.h"
#include "causal_kernel.cuh"
#include "delta_backward.cuh"
#include "delta_prepare.cuh"
#include "delta_step.cuh"
#include "delta_sweep.cuh"
#include "host_shared.h"
#include "qk_norm_kernel.cuh"

namespace pla {

cudaError_t sequence_faults(unsigned int* out, bool clear) {
  const unsigned int zero = 0;
  if (clear) return cudaMemcpyToSymbol(seq::g_sequence_faults, &zero, sizeof(zero));
  return cudaMemcpyFromSymbol(out, seq::g_sequence_faults, sizeof(*out));
}

namespace {

using namespace seq;

#define SEQ_CUDA(call)                                                  \
  do {                                                                  \
    const cudaError_t e_ = (call);                                      \
    if (e_ != cudaSuccess) return record_cuda_error(e_, #call);         \
  } while (0)

constexpr long long kMaxGrid = 0x7fffffff;
constexpr long long kMaxTokens = 1 << 30;  // 32-bit token numbers, with room for a stride past the end

size_t type_size(int dtype) { return dtype == PLA_F32 ? 4 : dtype == PLA_F16 || dtype == PLA_BF16 ? 2 : 0; }
bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
cudaStream_t as_stream(pla_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

struct Bytes {
  uintptr_t lo = 0, hi = 0;
};
Bytes dense(const void* p, long long elements, size_t size) {
  const uintptr_t b = reinterpret_cast<uintptr_t>(p);
  return p && elements > 0 ? Bytes{b, b + static_cast<uintptr_t>(elements) * size} : Bytes{};
}
struct Dim {
  long long extent, stride;
};
Bytes strided(const void* p, size_t size, std::initializer_list<Dim> dims) {
  long long lo = 0, hi = 0;
  for (const Dim& d : dims) {
    if (d.extent <= 0 || !p) return {};
    const long long reach = (d.extent - 1) * d.stride * static_cast<long long>(size);
    (reach < 0 ? lo : hi) += reach;
  }
  const uintptr_t b = reinterpret_cast<uintptr_t>(p);
  return {b + static_cast<uintptr_t>(lo), b + static_cast<uintptr_t>(hi) + size};
}
bool meets(Bytes a, Bytes b) { return a.lo < b.hi && b.lo < a.hi; }

// Shared-memory opt-in of a kernel, once per device.
template <auto Kernel>
int allow_shared(size_t bytes) {
  int dev = 0;
  SEQ_CUDA(cudaGetDevice(&dev));
  static std::atomic<size_t> set[64] = {};
  if (dev < 0 || dev >= 64) return PLA_ERR_NO_DEVICE;
  if (set[dev].load(std::memory_order_acquire) >= bytes) return PLA_OK;
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  if (set[dev].load(std::memory_order_relaxed) < bytes) {
    SEQ_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    set[dev].store(bytes, std::memory_order_release);
  }
  return PLA_OK;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PLA_OK : record_cuda_error(e, what);
}

// Calls f with a value of the element type.
template <typename F>
int with_type(int dtype, F&& f) {
  switch (dtype) {
    case PLA_F32: return f(float{});
    case PLA_BF16: return f(__nv_bfloat16{});
    default: return f(__half{});
  }
}
template <int N>
struct Int {
  static constexpr int value = N;
};

// ---- causal depthwise convolution ------------------------------------------
int check_causal(const pla_causal* a) {
  if (!a) return PLA_ERR_INVALID_ARGUMENT;
  if (a->batch < 0 || a->tokens < 0 || a->channels < 0 || a->sequences < 0) return PLA_ERR_INVALID_ARGUMENT;
  if (a->tokens > kMaxTokens) return PLA_ERR_TOO_LARGE;
  if (!type_size(a->dtype)) return PLA_ERR_UNSUPPORTED;
  if (a->taps < 2 || a->taps > 4) return PLA_ERR_UNSUPPORTED;
  if (a->cu_seqlens ? a->batch != 1 : a->sequences != a->batch) return PLA_ERR_INVALID_ARGUMENT;
  const bool work = a->batch && a->tokens && a->channels;
  if (work && (!a->x || !a->w)) return PLA_ERR_INVALID_ARGUMENT;
  return PLA_OK;
}

CausalParams causal_params(const pla_causal* a) {
  CausalParams p = {};
  p.x = a->x;
  p.x_batch = a->x_batch;
  p.x_token = a->x_token;
  p.w = a->w;
  p.b = a->b;
  p.cu = a->cu_seqlens;
  p.state_in = a->state_in;
  p.state_out = a->state_out;
  p.y = a->y;
  p.batch = a->batch;
  p.tokens = a->tokens;
  p.channels = a->channels;
  p.sequences = a->sequences;
  p.silu = a->silu != 0;
  return p;
}

// Long strips re-read the least; shorter ones while the device's threads would
// stay idle.
void cut_strips(CausalParams* p, int vec, long long threads, int longest) {
  const long long across = p->channels / vec;
  p->strip = longest;
  while (p->strip > 4 && across * p->batch * ((p->tokens + p->strip - 1) / p->strip) < threads) p->strip /= 2;
  p->strips = (p->tokens + p->strip - 1) / p->strip;
}

bool causal_vector(const pla_causal* a, int vec, std::initializer_list<const void*> more) {
  const size_t unit = vec * type_size(a->dtype);
  if (a->channels % vec || a->x_batch % vec || a->x_token % vec) return false;
  for (const void* p : more)
    if (!aligned_to(p, unit)) return false;
  return aligned_to(a->x, unit) && aligned_to(a->state_in, unit) && aligned_to(a->w, unit) && aligned_to(a->b, unit);
}

// f(element type, V, K): 8 bytes of channels a thread (backward, which holds
// five times as much: two channels), or single ones.
template <bool BACK, typename F>
int with_causal(int dtype, int taps, bool wide, F&& f) {
  return with_type(dtype, [&](auto zero) {
    auto with_taps = [&](auto v) {
      switch (taps) {
        case 2: return f(zero, v, Int<2>{});
        case 3: return f(zero, v, Int<3>{});
        default: return f(zero, v, Int<4>{});
      }
    };
    constexpr int W = BACK ? 2 : 8 / sizeof(decltype(zero));
    return wide ? with_taps(Int<W>{}) : with_taps(Int<1>{});
  });
}

// ---- norms -----------------------------------------------------------------
int check_norm(const pla_qk_norm* a, bool backward) {
  if (!a) return PLA_ERR_INVALID_ARGUMENT;
  if (a->batch < 0 || a->tokens < 0 || a->dim < 0 || a->rot < 0 || a->q.heads < 0 || a->k.heads < 0 || a->table_rows < 0 ||
      a->rot > a->dim || a->rot % 2 || !(a->eps >= 0.f))
    return PLA_ERR_INVALID_ARGUMENT;
  if (a->tokens > kMaxTokens) return PLA_ERR_TOO_LARGE;
  if (!type_size(a->dtype)) return PLA_ERR_UNSUPPORTED;
  if (a->dim > 256) return PLA_ERR_UNSUPPORTED;
  if (a->rot && (!a->cos_table || !a->sin_table)) return PLA_ERR_INVALID_ARGUMENT;
  if (a->positions && a->position_bytes != 4 && a->position_bytes != 8) return PLA_ERR_INVALID_ARGUMENT;
  const long long tokens = static_cast<long long>(a->batch) * a->tokens;
  const pla_norm_side* side[2] = {&a->q, &a->k};
  for (const pla_norm_side* s : side) {
    if (!tokens || !s->heads || !a->dim) continue;
    if (!s->x || !s->y || (backward && !s->dy)) return PLA_ERR_INVALID_ARGUMENT;
    const Bytes out = dense(s->y, tokens * s->heads * a->dim, type_size(a->dtype));
    for (const pla_norm_side* o : side) {
      const Dim dim = {a->dim, 1}, heads = {o->heads, o->x_head};
      if (meets(out, strided(o->x, type_size(a->dtype), {dim, heads, {a->tokens, o->x_token}, {a->batch, o->x_batch}})))
        return PLA_ERR_INVALID_ARGUMENT;
      if (backward && meets(out, strided(o->dy, type_size(a->dtype),
                                         {dim, {o->heads, o->dy_head}, {a->tokens, o->dy_token}, {a->batch, o->dy_batch}})))
        return PLA_ERR_INVALID_ARGUMENT;
    }
  }
  return PLA_OK;
}

NormParams norm_params(const pla_qk_norm* a) {
  NormParams p = {};
  const pla_norm_side* side[2] = {&a->q, &a->k};
  for (int i = 0; i < 2; ++i) {
    NormSide& s = p.side[i];
    s.x = side[i]->x;
    s.x_batch = side[i]->x_batch;
    s.x_token = side[i]->x_token;
    s.x_head = side[i]->x_head;
    s.w = side[i]->w;
    s.y = side[i]->y;
    s.dy = side[i]->dy;
    s.dy_batch = side[i]->dy_batch;
    s.dy_token = side[i]->dy_token;
    s.dy_head = side[i]->dy_head;
    s.heads = side[i]->heads;
  }
  p.cos = a->rot ? a->cos_table : nullptr;
  p.sin = a->rot ? a->sin_table : nullptr;
  p.positions = a->positions;
  p.position_batch = a->position_batch;
  p.position_bytes = a->position_bytes;
  p.table_rows = a->table_rows;
  p.batch = a->batch;
  p.tokens = a->tokens;
  p.dim = a->dim;
  p.rot = a->rot;
  p.interleaved = a->interleaved != 0;
  p.l2 = a->l2 != 0;
  p.eps = a->eps;
  return p;
}

bool norm_vector(const pla_qk_norm* a, bool backward) {
  const size_t unit = 4 * type_size(a->dtype);
  if (a->rot / 2 % 4 || (a->dim - a->rot) / 2 % 4 || (a->dim - a->rot) % 2) return false;
  if (a->rot && (!aligned_to(a->cos_table, 16) || !aligned_to(a->sin_table, 16))) return false;
  for (const pla_norm_side* s : {&a->q, &a->k}) {
    if (!aligned_to(s->x, unit) || !aligned_to(s->y, unit) || !aligned_to(s->w, unit)) return false;
    if (s->x_batch % 4 || s->x_token % 4 || s->x_head % 4) return false;
    if (backward && (!aligned_to(s->dy, unit) || s->dy_batch % 4 || s->dy_token % 4 || s->dy_head % 4)) return false;
  }
  return true;
}

// f(element type, lanes of a head, pairs adjacent): the group as small as holds
// a head at 4 pairs a lane.
template <typename F>
int with_norm4(const pla_qk_norm* a, F&& f) {
  return with_type(a->dtype, [&](auto zero) {
    const auto lanes = [&](auto inter) {
      if (a->dim <= 64) return f(zero, Int<8>{}, inter);
      if (a->dim <= 128) return f(zero, Int<16>{}, inter);
      return f(zero, Int<32>{}, inter);
    };
    return a->interleaved && a->rot ? lanes(std::true_type{}) : lanes(std::false_type{});
  });
}
int norm_lanes(const pla_qk_norm* a, bool wide) { return !wide || a->dim > 128 ? 32 : a->dim > 64 ? 16 : 8; }

// Blocks of one side in the backward pass: a number of groups that is a
// multiple of the heads (a group keeps its head), a few turns each so that a
// block's partial sum is small beside what it reads, and both sides together
// no more than run at a time, each by its share of the heads (4094 tokens of 32
// heads of 96, fp16: 36 us; twice as many blocks 37, half as many again 45).
int norm_side_blocks(const pla_qk_norm* a, int heads, int lanes) {
  const long long rows = static_cast<long long>(a->batch) * a->tokens * heads;
  if (!rows) return 0;
  const int groups = kNormThreads / lanes, step = heads / std::gcd(heads, groups);
  const long long most = 148ll * 2 * heads / (static_cast<long long>(a->q.heads) + a->k.heads);
  const long long want = std::min((rows + groups * 4 - 1) / (groups * 4), most);
  return static_cast<int>(std::max<long long>(1, want / step) * step);
}

// ---- gated delta rule ------------------------------------------------------
int check_delta(const pla_delta* a) {
  if (!a) return PLA_ERR_INVALID_ARGUMENT;
  if (a->batch < 0 || a->tokens < 0 || a->sequences < 0 || a->hk < 0 || a->hv < 0 || a->dk < 0 || a->dv < 0)
    return PLA_ERR_INVALID_ARGUMENT;
  if (a->tokens > kMaxTokens) return PLA_ERR_TOO_LARGE;
  if (!type_size(a->dtype)) return PLA_ERR_UNSUPPORTED;
  if (a->cu_seqlens ? a->batch != 1 : a->sequences != a->batch) return PLA_ERR_INVALID_ARGUMENT;
  if (a->hv && (a->hk < 1 || a->hv % a->hk)) return PLA_ERR_INVALID_ARGUMENT;
  if (a->dk < 1 || a->dk > 128 || a->dv > 128) return PLA_ERR_UNSUPPORTED;
  if (a->batch && a->tokens && a->hv && a->dv && (!a->q || !a->k || !a->v || !a->g || !a->beta))
    return PLA_ERR_INVALID_ARGUMENT;
  return PLA_OK;
}

struct DeltaSizes {
  long long chunks = 0;
  size_t plan = 0, tiles = 0, heads = 0, states = 0, us = 0, scales = 0, total = 0;
};
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

template <typename T, int DK>
DeltaSizes delta_sizes_of(const pla_delta* a, bool backward) {
  using L = DeltaLayout<T, DK>;
  DeltaSizes s;
  s.chunks = a->cu_seqlens ? a->tokens / kChunk + static_cast<long long>(a->sequences)
                           : static_cast<long long>(a->batch) * ((a->tokens + kChunk - 1) / kChunk);
  s.plan = a->cu_seqlens ? up256(s.chunks * sizeof(int4)) + up256((4ull * a->sequences + 1) * sizeof(int)) : 0;
  s.tiles = up256(static_cast<size_t>(s.chunks) * a->hk * L::kTiles);
  s.heads = up256(static_cast<size_t>(s.chunks) * a->hv * L::kHead);
  if (backward) {
    const size_t rows = static_cast<size_t>(s.chunks) * a->hv * ((a->dv + 63) / 64) * 64;
    s.states = up256(rows * kPlanes * DK * 2);
    s.us = up256(rows * kPlanes * kChunk * 2);
    s.scales = up256(rows * 4 * sizeof(float));
  }
  s.total = s.plan + s.tiles + s.heads + 2 * s.states + 2 * s.us + s.scales;
  return s;
}

// f(element type, padded Dk)
template <typename F>
int with_delta(const pla_delta* a, F&& f) {
  return with_type(a->dtype, [&](auto zero) { return a->dk <= 64 ? f(zero, Int<64>{}) : f(zero, Int<128>{}); });
}

DeltaParams delta_params(const pla_delta* a, const DeltaSizes& s) {
  DeltaParams p = {};
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.g = a->g;
  p.beta = a->beta;
  p.q_batch = a->q_batch, p.q_token = a->q_token, p.q_head = a->q_head;
  p.k_batch = a->k_batch, p.k_token = a->k_token, p.k_head = a->k_head;
  p.v_batch = a->v_batch, p.v_token = a->v_token, p.v_head = a->v_head;
  p.g_batch = a->g_batch, p.g_token = a->g_token, p.g_head = a->g_head;
  p.beta_batch = a->beta_batch, p.beta_token = a->beta_token, p.beta_head = a->beta_head;
  p.cu = a->cu_seqlens;
  p.state_in = a->state_in;
  p.state_out = a->state_out;
  p.o = a->o;
  p.batch = a->batch;
  p.tokens = a->tokens;
  p.sequences = a->sequences;
  p.hk = a->hk;
  p.hv = a->hv;
  p.dk = a->dk;
  p.dv = a->dv;
  p.gates32 = a->gates32 != 0;
  p.scale = a->scale;
  p.row_chunks = (a->tokens + kChunk - 1) / kChunk;
  p.chunk_bound = static_cast<int>(s.chunks);
  p.slabs = (a->dv + 15) / 16;
  char* w = static_cast<char*>(a->workspace);
  p.table = reinterpret_cast<int4*>(w);
  p.plan = reinterpret_cast<int*>(w + up256(s.chunks * sizeof(int4)));
  w += s.plan;
  p.tiles = w;
  w += s.tiles;
  p.heads = w;
  w += s.heads;
  p.states = w;
  w += s.states;
  p.dstates = w;
  w += s.states;
  p.us = w;
  w += s.us;
  p.dxs = w;
  w += s.us;
  p.scales = reinterpret_cast<float*>(w);
  p.rows = (a->dv + 63) / 64 * 64;
  const size_t es = type_size(a->dtype);
  const int whole = static_cast<int>(16 / es);
  p.vec_qk = a->dk % 4 == 0 && aligned_to(a->q, 4 * es) && aligned_to(a->k, 4 * es) &&
             !((a->q_batch | a->q_token | a->q_head | a->k_batch | a->k_token | a->k_head) % 4);
  p.vec_v = a->dv % whole == 0 && aligned_to(a->v, 16) && !((a->v_batch | a->v_token | a->v_head) % whole);
  p.vec_o = aligned_to(a->o, 16) && a->dv % whole == 0;
  return p;
}

template <typename T, int DK>
int launch_prepare(const DeltaParams& p, cudaStream_t stream) {
  if (p.cu) {
    delta_plan<<<1, 1024, 0, stream>>>(p.cu, p.tokens, p.sequences, p.plan, p.table, p.chunk_bound);
    const int st = launched("delta_plan");
    if (st != PLA_OK) return st;
  }
  if (static_cast<long long>(p.chunk_bound) * p.hk > kMaxGrid) return PLA_ERR_TOO_LARGE;
  if (!p.chunk_bound) return PLA_OK;
  const auto go = [&](auto heads) {
    constexpr int HEADS = decltype(heads)::value;
    const size_t shared = sizeof(PrepShared<T, DK, HEADS>);
    const int st = allow_shared<delta_prepare<T, DK, HEADS>>(shared);
    if (st != PLA_OK) return st;
    delta_prepare<T, DK, HEADS><<<p.chunk_bound * p.hk, 128 * HEADS, shared, stream>>>(p);
    return launched("delta_prepare");
  };
  return p.hv > p.hk ? go(Int<2>{}) : go(Int<1>{});  // two value heads of a key head side by side
}

// Stages of the ring and shared memory of a sweep; PER_SM blocks fit an SM.
template <typename T, int DK, int VB, int PER_SM, bool BACK>
struct SweepShape {
  using L = DeltaLayout<T, DK>;
  static constexpr size_t kHeld = kSweepRing + sizeof(SweepShared<T, DK, VB, BACK>);
  static constexpr size_t kMost = 227 * 1024 / PER_SM - (PER_SM > 1 ? 1024 : 0);  // 1 KB of a block is the system's
  static constexpr size_t kRoom = kHeld < kMost ? (kMost - kHeld) / L::kStage : 0;
  static constexpr int kStages = kRoom < 3 ? kRoom : 3;
  static constexpr size_t kShared = kHeld + kStages * L::kStage;
  static constexpr int kColumns = VB, kPerSm = PER_SM;
  static long long grid(const DeltaParams& p) {
    return static_cast<long long>(p.sequences) * p.hv * ((p.dv + VB - 1) / VB);
  }
};

// Value features of a sweep's block.  A block's time is the latency of its
// chunks' chain, nearly whatever it holds, so while every block has an SM of
// its own: the fewest features that still leave it so (1001 tokens x 16 heads
// of 128, fp16: 28 us with 16, 42 with 32).  With more blocks than SMs: of a
// batch, whose rows are equally long, two blocks of 32 an SM, if they fit (16-bit
// inputs, Dk up to 64), fill each other's waits (8 x 2048 tokens x 32 heads of 64 x
// 128, bf16: 500 us, back 620; one block: 561 and 705); of a ragged batch one
// block of 32, because the longest sequence's blocks, the first to start, decide
// (16383 tokens in three, 32 heads of 128, when outputs had one plane and two
// blocks fit: 631 us against 692).  f(shape)
template <typename T, int DK, bool BACK, typename F>
int with_columns(const DeltaParams& p, int sms, F&& f) {
  using Two = SweepShape<T, DK, 32, 2, BACK>;
  const long long heads = static_cast<long long>(p.sequences) * p.hv;
  if (p.dv <= 16 || heads * ((p.dv + 15) / 16) <= sms) return f(SweepShape<T, DK, 16, 1, BACK>{});
  if constexpr (Two::kStages >= 1)
    if (!p.cu && heads * ((p.dv + 31) / 32) > sms) return f(Two{});
  return f(SweepShape<T, DK, 32, 1, BACK>{});
}

template <typename T, int DK, bool KEEP>
int launch_sweep(const DeltaParams& p, int sms, cudaStream_t stream) {
  return with_columns<T, DK, false>(p, sms, [&](auto shape) {
    using S = decltype(shape);
    constexpr int VB = S::kColumns;
    static_assert(S::kStages >= 1, "no room for a chunk's tiles");
    const long long grid = S::grid(p);
    if (grid > kMaxGrid) return static_cast<int>(PLA_ERR_TOO_LARGE);
    const int st = allow_shared<delta_sweep<T, DK, VB, S::kStages, S::kPerSm, KEEP>>(S::kShared);
    if (st != PLA_OK) return st;
    delta_sweep<T, DK, VB, S::kStages, S::kPerSm, KEEP><<<static_cast<int>(grid), VB * 8, S::kShared, stream>>>(p);
    return launched("delta_sweep");
  });
}

template <typename T, int DK>
int launch_gradient(const DeltaParams& p, int sms, cudaStream_t stream) {
  int st = with_columns<T, DK, true>(p, sms, [&](auto shape) {
    using S = decltype(shape);
    constexpr int VB = S::kColumns;
    static_assert(S::kStages >= 1, "no room for a chunk's tiles");
    const int st = allow_shared<delta_sweep_back<T, DK, VB, S::kStages, S::kPerSm>>(S::kShared);
    if (st != PLA_OK) return st;
    delta_sweep_back<T, DK, VB, S::kStages, S::kPerSm><<<static_cast<int>(S::grid(p)), VB * 8, S::kShared, stream>>>(p);
    return launched("delta_sweep_back");
  });
  if (st != PLA_OK) return st;
  if (p.cu) {
    delta_clear_rows<T><<<std::min(p.tokens + 1, 4 * sms), 256, 0, stream>>>(p);
    if ((st = launched("delta_clear_rows")) != PLA_OK) return st;
  }
  if (!p.chunk_bound) return PLA_OK;
  const size_t shared = sizeof(GradShared<T, DK>);
  if ((st = allow_shared<delta_gradient<T, DK>>(shared)) != PLA_OK) return st;
  delta_gradient<T, DK><<<p.chunk_bound * p.hk, kGradThreads, shared, stream>>>(p);
  return launched("delta_gradient");
}

}  // namespace
}  // namespace pla

using namespace pla;

extern "C" {

int pla_causal_depthwise_forward(const pla_causal* a, pla_stream_t stream) {
  int st = check_causal(a);
  if (st != PLA_OK) return st;
  const size_t es = type_size(a->dtype);
  const bool work = a->batch && a->tokens && a->channels;
  if (work && !a->y) return PLA_ERR_INVALID_ARGUMENT;
  const long long elements = static_cast<long long>(a->batch) * a->tokens * a->channels;
  const long long held = static_cast<long long>(a->sequences) * (a->taps - 1) * a->channels;
  const Bytes x = strided(a->x, es, {{a->channels, 1}, {a->tokens, a->x_token}, {a->batch, a->x_batch}});
  const Bytes y = dense(a->y, elements, es), out = dense(a->state_out, held, es), in = dense(a->state_in, held, es);
  if (meets(y, x) || meets(y, in) || meets(out, x) || meets(out, in) || meets(out, y)) return PLA_ERR_INVALID_ARGUMENT;
  if (!a->channels || (!work && !(a->state_out && a->sequences))) return PLA_OK;
  int sms;
  if ((st = current_sm100(&sms)) != PLA_OK) return st;
  const bool wide = causal_vector(a, static_cast<int>(8 / es), {a->y, a->state_out});
  return with_causal<false>(a->dtype, a->taps, wide, [&](auto zero, auto v, auto k) {
    using T = decltype(zero);
    constexpr int V = decltype(v)::value, K = decltype(k)::value;
    CausalParams p = causal_params(a);
    cut_strips(&p, V, sms * 768ll, 32);
    const long long items = work ? static_cast<long long>(p.batch) * p.strips * (p.channels / V) : 0;
    const long long states = p.state_out ? held / V : 0;
    const long long main_blocks = (items + kCausalThreads - 1) / kCausalThreads;
    const long long blocks = main_blocks + (states + kCausalThreads - 1) / kCausalThreads;
    if (blocks > kMaxGrid) return static_cast<int>(PLA_ERR_TOO_LARGE);
    causal_forward<T, V, K><<<static_cast<int>(blocks), kCausalThreads, 0, as_stream(stream)>>>(
        p, static_cast<int>(main_blocks));
    return launched("causal_forward");
  });
}

namespace {
// Blocks of strips in the backward pass (what the workspace is sized by).
CausalParams causal_backward_params(const pla_causal* a, bool wide, long long* block_rows) {
  CausalParams p = causal_params(a);
  cut_strips(&p, wide ? 2 : 1, 148 * 768, 64);
  *block_rows = (static_cast<long long>(p.batch) * p.strips + kCausalRows - 1) / kCausalRows;
  return p;
}
}  // namespace

size_t pla_causal_depthwise_workspace(const pla_causal* a) {
  if (check_causal(a) != PLA_OK || !a->batch || !a->tokens || !a->channels) return 0;
  long long wide_rows, rows;
  causal_backward_params(a, a->channels % 2 == 0, &wide_rows);
  causal_backward_params(a, false, &rows);
  return static_cast<size_t>(std::max(rows, wide_rows)) * (a->taps + 1) * a->channels * sizeof(float);
}

int pla_causal_depthwise_backward(const pla_causal* a, const pla_causal_gradient* g, pla_stream_t stream) {
  int st = check_causal(a);
  if (st != PLA_OK) return st;
  if (!g) return PLA_ERR_INVALID_ARGUMENT;
  const size_t es = type_size(a->dtype);
  const bool work = a->batch && a->tokens && a->channels;
  if (work && (!g->dy || !g->dx)) return PLA_ERR_INVALID_ARGUMENT;
  const bool sums = g->dw || g->db;
  if (work && sums && (g->workspace_bytes < pla_causal_depthwise_workspace(a) || !g->workspace || !aligned_to(g->workspace, 16)))
    return PLA_ERR_INVALID_ARGUMENT;
  const Bytes dx = dense(g->dx, static_cast<long long>(a->batch) * a->tokens * a->channels, es);
  if (meets(dx, strided(a->x, es, {{a->channels, 1}, {a->tokens, a->x_token}, {a->batch, a->x_batch}})) ||
      meets(dx, strided(g->dy, es, {{a->channels, 1}, {a->tokens, g->dy_token}, {a->batch, g->dy_batch}})))
    return PLA_ERR_INVALID_ARGUMENT;
  if (!a->channels) return PLA_OK;
  int sms;
  if ((st = current_sm100(&sms)) != PLA_OK) return st;
  const bool wide = causal_vector(a, 2, {g->dy, g->dx, g->dstate_out}) && g->dy_batch % 2 == 0 && g->dy_token % 2 == 0;
  return with_causal<true>(a->dtype, a->taps, wide, [&](auto zero, auto v, auto k) {
    using T = decltype(zero);
    constexpr int V = decltype(v)::value, K = decltype(k)::value;
    long long rows;
    CausalParams p = causal_backward_params(a, V > 1, &rows);
    p.dy = g->dy;
    p.dy_batch = g->dy_batch;
    p.dy_token = g->dy_token;
    p.dstate_out = g->dstate_out;
    p.dx = g->dx;
    p.dstate_in = g->dstate_in;
    p.partial = sums ? static_cast<float*>(g->workspace) : nullptr;
    int st = PLA_OK;
    if (!work) rows = 0;
    if (work) {
      const long long blocks = rows * ((p.channels / V + 31) / 32);
      if (blocks > kMaxGrid) return static_cast<int>(PLA_ERR_TOO_LARGE);
      causal_backward<T, V, K><<<static_cast<int>(blocks), kCausalThreads, 0, as_stream(stream)>>>(p);
      if ((st = launched("causal_backward")) != PLA_OK) return st;
    }
    if (sums) {
      const long long count = static_cast<long long>(K + 1) * p.channels;
      causal_reduce<T><<<static_cast<int>((count + 31) / 32), 256, 0, as_stream(stream)>>>(
          p.partial, static_cast<int>(rows), p.channels, K, static_cast<T*>(g->dw), static_cast<T*>(g->db));
      if ((st = launched("causal_reduce")) != PLA_OK) return st;
    }
    if (p.dstate_in && p.sequences) {
      const long long items = static_cast<long long>(p.sequences) * p.channels;
      if ((items + 255) / 256 > kMaxGrid) return static_cast<int>(PLA_ERR_TOO_LARGE);
      causal_state_gradient<T, K><<<static_cast<int>((items + 255) / 256), 256, 0, as_stream(stream)>>>(p);
      st = launched("causal_state_gradient");
    }
    return st;
  });
}

int pla_causal_depthwise_step(const void* x, int64_t x_row, void* state, int64_t state_row, const void* w, const void* b,
                              void* y, int n, int channels, int taps, int silu, int dtype, pla_stream_t stream) {
  const size_t es = type_size(dtype);
  if (n < 0 || channels < 0) return PLA_ERR_INVALID_ARGUMENT;
  if (!es || taps < 2 || taps > 4) return PLA_ERR_UNSUPPORTED;
  if (!n || !channels) return PLA_OK;
  if (!x || !state || !w || !y) return PLA_ERR_INVALID_ARGUMENT;
  const long long held = static_cast<long long>(taps - 1) * channels;
  if (n > 1 && state_row < held) return PLA_ERR_INVALID_ARGUMENT;  // rows that share memory would race
  const Bytes xs = strided(x, es, {{channels, 1}, {n, x_row}}), ss = strided(state, es, {{held, 1}, {n, state_row}});
  const Bytes ys = dense(y, static_cast<long long>(n) * channels, es);
  if (meets(ys, xs) || meets(ys, ss) || meets(xs, ss)) return PLA_ERR_INVALID_ARGUMENT;
  int sms, st;
  if ((st = current_sm100(&sms)) != PLA_OK) return st;
  const int vec = static_cast<int>(8 / es);
  const bool wide = channels % vec == 0 && x_row % vec == 0 && state_row % vec == 0 && aligned_to(x, 8) &&
                    aligned_to(state, 8) && aligned_to(y, 8) && aligned_to(w, 8) && aligned_to(b, 8);
  return with_causal<false>(dtype, taps, wide, [&](auto zero, auto v, auto k) {
    using T = decltype(zero);
    constexpr int V = decltype(v)::value, K = decltype(k)::value;
    CausalParams p = {};
    p.w = w;
    p.b = b;
    p.y = y;
    p.batch = n;
    p.channels = channels;
    p.silu = silu != 0;
    const long long blocks = (static_cast<long long>(n) * (channels / V) + 127) / 128;
    if (blocks > kMaxGrid) return static_cast<int>(PLA_ERR_TOO_LARGE);
    causal_step<T, V, K><<<static_cast<int>(blocks), 128, 0, as_stream(stream)>>>(
        static_cast<const T*>(x), x_row, static_cast<T*>(state), state_row, p);
    return launched("causal_step");
  });
}

int pla_qk_norm_rotate_forward(const pla_qk_norm* a, pla_stream_t stream) {
  int st = check_norm(a, false);
  if (st != PLA_OK) return st;
  const long long tokens = static_cast<long long>(a->batch) * a->tokens;
  if (!tokens || !a->dim || !(a->q.heads + a->k.heads)) return PLA_OK;
  if (a->batch > 65535) return PLA_ERR_TOO_LARGE;
  int sms;
  if ((st = current_sm100(&sms)) != PLA_OK) return st;
  const bool wide = norm_vector(a, false);
  const int lanes = norm_lanes(a, wide), groups = kNormThreads / lanes;
  // several heads a group (64 bytes a lane in flight) once that still leaves every SM a thousand threads
  const int most = !wide ? 1 : a->dtype == PLA_F32 ? 2 : 4;
  const int hb = most > 1 && tokens * (a->q.heads + a->k.heads) / most * lanes >= sms * 1024ll ? most : 1;
  NormParams p = norm_params(a);
  p.units[0] = (a->q.heads + hb - 1) / hb;
  p.units[1] = (a->k.heads + hb - 1) / hb;
  const int units = p.units[0] + p.units[1];
  const long long whole = (static_cast<long long>(a->tokens) * units + groups - 1) / groups;
  // Several heads a group: no more blocks than run at a time, two an SM, each group walking tokens; one block more
  // is a second walk (8192 tokens of 40 heads of 128, bf16: 45 us; 300 blocks on 296 places 68; 1180 blocks 50).
  // Where batch rows leave an eighth of the places empty that way, and with single heads a group, whose blocks are
  // lighter (8192 tokens of 16 heads of 250, fp16: 69 us, with two an SM 82): eight an SM.  Always a number of
  // groups that is a multiple of the units, so that a group keeps its unit.
  const int step = units / std::gcd(units, groups);
  long long blocks = hb > 1 ? sms * 2ll / a->batch / step * step : 0;
  if (blocks * a->batch * 8 < sms * 2ll * 7) blocks = std::max<long long>(1, (sms * 8ll / a->batch + step - 1) / step) * step;
  p.stride = whole <= blocks ? a->tokens : static_cast<int>(blocks * groups / units);
  blocks = std::min(blocks, whole);
  const dim3 grid(static_cast<int>(blocks), a->batch);
  if (!wide)
    return with_type(a->dtype, [&](auto zero) {
      qk_norm_forward1<decltype(zero)><<<grid, kNormThreads, 0, as_stream(stream)>>>(p);
      return launched("qk_norm_forward1");
    });
  return with_norm4(a, [&](auto zero, auto l, auto inter) {
    using T = decltype(zero);
    constexpr int LANES = decltype(l)::value, HB = sizeof(T) == 4 ? 2 : 4;
    constexpr bool INTER = decltype(inter)::value;
    if (hb > 1)
      qk_norm_forward4<T, LANES, HB, INTER><<<grid, kNormThreads, 0, as_stream(stream)>>>(p);
    else
      qk_norm_forward4<T, LANES, 1, INTER><<<grid, kNormThreads, 0, as_stream(stream)>>>(p);
    return launched("qk_norm_forward4");
  });
}

size_t pla_qk_norm_rotate_workspace(const pla_qk_norm* a) {
  if (!a || a->dim < 0 || a->batch < 0 || a->tokens < 0 || a->q.heads < 0 || a->k.heads < 0) return 0;
  int most = 0;
  for (int lanes : {8, 16, 32}) most = std::max(most, norm_side_blocks(a, a->q.heads, lanes) + norm_side_blocks(a, a->k.heads, lanes));
  return static_cast<size_t>(most) * a->dim * sizeof(float);
}

int pla_qk_norm_rotate_backward(const pla_qk_norm* a, void* workspace, size_t workspace_bytes, pla_stream_t stream) {
  int st = check_norm(a, true);
  if (st != PLA_OK) return st;
  const bool sums = a->q.dw || a->k.dw;
  if ((a->q.dw && !a->q.w) || (a->k.dw && !a->k.w)) return PLA_ERR_INVALID_ARGUMENT;
  if (sums && a->dim &&
      (workspace_bytes < pla_qk_norm_rotate_workspace(a) || (!workspace && pla_qk_norm_rotate_workspace(a)) ||
       !aligned_to(workspace, 16)))
    return PLA_ERR_INVALID_ARGUMENT;
  if (!a->dim) return PLA_OK;
  const long long tokens = static_cast<long long>(a->batch) * a->tokens;
  if (tokens * std::max(a->q.heads, a->k.heads) > kMaxTokens) return PLA_ERR_TOO_LARGE;
  int sms;
  if ((st = current_sm100(&sms)) != PLA_OK) return st;
  const bool wide = norm_vector(a, true);
  const int lanes = norm_lanes(a, wide);
  NormParams p = norm_params(a);
  p.partial = sums ? static_cast<float*>(workspace) : nullptr;
  for (int i = 0; i < 2; ++i) {
    const int heads = i ? a->k.heads : a->q.heads;
    p.side_blocks[i] = norm_side_blocks(a, heads, lanes);
    p.side_stride[i] = heads ? p.side_blocks[i] * (kNormThreads / lanes) / heads : 1;
  }
  const int blocks = p.side_blocks[0] + p.side_blocks[1];
  if (blocks > 0) {
    st = !wide ? with_type(a->dtype, [&](auto zero) {
      qk_norm_backward1<decltype(zero)><<<blocks, kNormThreads, 0, as_stream(stream)>>>(p);
      return launched("qk_norm_backward1");
    })
               : with_norm4(a, [&](auto zero, auto l, auto inter) {
      qk_norm_backward4<decltype(zero), decltype(l)::value, decltype(inter)::value>
          <<<blocks, kNormThreads, 0, as_stream(stream)>>>(p);
      return launched("qk_norm_backward4");
    });
    if (st != PLA_OK) return st;
  }
  if (sums)
    st = with_type(a->dtype, [&](auto zero) {
      using T = decltype(zero);
      qk_norm_reduce<T><<<dim3((a->dim + 31) / 32, 2), 1024, 0, as_stream(stream)>>>(
          p.partial, p.side_blocks[0], p.side_blocks[1], a->dim, static_cast<T*>(a->q.dw), static_cast<T*>(a->k.dw));
      return launched("qk_norm_reduce");
    });
  return st;
}

size_t pla_gated_delta_rule_workspace(const pla_delta* a, int backward) {
  if (check_delta(a) != PLA_OK) return 0;
  size_t bytes = 0;
  const auto size = [&](auto zero, auto dk) {
    bytes = delta_sizes_of<decltype(zero), decltype(dk)::value>(a, backward != 0).total;
    return 0;
  };
  with_delta(a, size);
  return bytes;
}

int pla_gated_delta_rule_forward(const pla_delta* a, pla_stream_t stream) {
  int st = check_delta(a);
  if (st != PLA_OK) return st;
  const size_t es = type_size(a->dtype);
  const bool work = a->batch && a->tokens && a->hv && a->dv;
  if (work && !a->o) return PLA_ERR_INVALID_ARGUMENT;
  const long long held = static_cast<long long>(a->sequences) * a->hv * a->dk * a->dv;
  const Bytes o = dense(a->o, static_cast<long long>(a->batch) * a->tokens * a->hv * a->dv, es);
  const Bytes out = dense(a->state_out, held, 4), in = dense(a->state_in, held, 4);
  const Bytes read[3] = {
      strided(a->q, es, {{a->dk, 1}, {a->hk, a->q_head}, {a->tokens, a->q_token}, {a->batch, a->q_batch}}),
      strided(a->k, es, {{a->dk, 1}, {a->hk, a->k_head}, {a->tokens, a->k_token}, {a->batch, a->k_batch}}),
      strided(a->v, es, {{a->dv, 1}, {a->hv, a->v_head}, {a->tokens, a->v_token}, {a->batch, a->v_batch}})};
  for (const Bytes& r : read)
    if (meets(o, r) || meets(out, r)) return PLA_ERR_INVALID_ARGUMENT;
  if (meets(o, in) || meets(out, in) || meets(o, out)) return PLA_ERR_INVALID_ARGUMENT;
  if (!a->hv || !a->dv || !a->sequences) return PLA_OK;
  int sms;
  if ((st = current_sm100(&sms)) != PLA_OK) return st;
  return with_delta(a, [&](auto zero, auto dk) {
    using T = decltype(zero);
    constexpr int DK = decltype(dk)::value;
    const DeltaSizes s = delta_sizes_of<T, DK>(a, false);
    if (s.chunks > kMaxGrid) return static_cast<int>(PLA_ERR_TOO_LARGE);
    if (s.total && (a->workspace_bytes < s.total || !a->workspace || !aligned_to(a->workspace, 256)))
      return static_cast<int>(PLA_ERR_INVALID_ARGUMENT);
    const DeltaParams p = delta_params(a, s);
    const int st = launch_prepare<T, DK>(p, as_stream(stream));
    if (st != PLA_OK) return st;
    return launch_sweep<T, DK, false>(p, sms, as_stream(stream));
  });
}

int pla_gated_delta_rule_backward(const pla_delta* a, const pla_delta_gradient* g, pla_stream_t stream) {
  int st = check_delta(a);
  if (st != PLA_OK) return st;
  if (!g) return PLA_ERR_INVALID_ARGUMENT;
  const size_t es = type_size(a->dtype);
  const bool work = a->batch && a->tokens && a->hv && a->dv;
  if (work && (!g->d_o || !g->dq || !g->dk || !g->dv || !g->dg || !g->dbeta)) return PLA_ERR_INVALID_ARGUMENT;
  const long long tokens = static_cast<long long>(a->batch) * a->tokens;
  const Bytes written[3] = {dense(g->dq, tokens * a->hk * a->dk, es), dense(g->dk, tokens * a->hk * a->dk, es),
                            dense(g->dv, tokens * a->hv * a->dv, es)};
  const Bytes read[4] = {
      strided(a->q, es, {{a->dk, 1}, {a->hk, a->q_head}, {a->tokens, a->q_token}, {a->batch, a->q_batch}}),
      strided(a->k, es, {{a->dk, 1}, {a->hk, a->k_head}, {a->tokens, a->k_token}, {a->batch, a->k_batch}}),
      strided(a->v, es, {{a->dv, 1}, {a->hv, a->v_head}, {a->tokens, a->v_token}, {a->batch, a->v_batch}}),
      strided(g->d_o, es, {{a->dv, 1}, {a->hv, g->do_head}, {a->tokens, g->do_token}, {a->batch, g->do_batch}})};
  for (const Bytes& w : written)
    for (const Bytes& r : read)
      if (meets(w, r)) return PLA_ERR_INVALID_ARGUMENT;
  const long long held = static_cast<long long>(a->sequences) * a->hv * a->dk * a->dv;
  if (meets(dense(g->dstate_in, held, 4), dense(g->dstate_out, held, 4)) ||
      meets(dense(g->dstate_in, held, 4), dense(a->state_in, held, 4)))
    return PLA_ERR_INVALID_ARGUMENT;
  if (!a->hv || !a->dv || !a->sequences) return PLA_OK;
  int sms;
  if ((st = current_sm100(&sms)) != PLA_OK) return st;
  return with_delta(a, [&](auto zero, auto dk) {
    using T = decltype(zero);
    constexpr int DK = decltype(dk)::value;
    const DeltaSizes s = delta_sizes_of<T, DK>(a, true);
    if (s.chunks > kMaxGrid) return static_cast<int>(PLA_ERR_TOO_LARGE);
    if (s.total && (a->workspace_bytes < s.total || !a->workspace || !aligned_to(a->workspace, 256)))
      return static_cast<int>(PLA_ERR_INVALID_ARGUMENT);
    DeltaParams p = delta_params(a, s);
    p.d_o = g->d_o;
    p.do_batch = g->do_batch, p.do_token = g->do_token, p.do_head = g->do_head;
    p.dstate_out = g->dstate_out;
    p.dstate_in = g->dstate_in;
    p.dq = g->dq, p.dk_out = g->dk, p.dv_out = g->dv, p.dg = g->dg, p.dbeta = g->dbeta;
    const int whole = static_cast<int>(16 / es);
    p.vec_do = a->dv % whole == 0 && aligned_to(g->d_o, 16) && !((g->do_batch | g->do_token | g->do_head) % whole);
    p.vec_o = aligned_to(g->dv, 16) && a->dv % whole == 0;
    p.pair_qk = a->dk % 2 == 0 && aligned_to(g->dq, 2 * es) && aligned_to(g->dk, 2 * es);
    p.state_out = nullptr;
    int st = launch_prepare<T, DK>(p, as_stream(stream));
    if (st != PLA_OK) return st;
    if ((st = launch_sweep<T, DK, true>(p, sms, as_stream(stream))) != PLA_OK) return st;
    return launch_gradient<T, DK>(p, sms, as_stream(stream));
  });
}

int pla_gated_delta_rule_step(const pla_delta_step* a, pla_stream_t stream) {
  if (!a || a->n < 0 || a->hk < 0 || a->hv < 0 || a->dk < 0 || a->dv < 0) return PLA_ERR_INVALID_ARGUMENT;
  const size_t es = type_size(a->dtype);
  if (!es) return PLA_ERR_UNSUPPORTED;
  if (a->hv && (a->hk < 1 || a->hv % a->hk)) return PLA_ERR_INVALID_ARGUMENT;
  if (a->dk < 1 || a->dk > 256) return PLA_ERR_UNSUPPORTED;
  if (!a->n || !a->hv || !a->dv) return PLA_OK;
  if (!a->q || !a->k || !a->v || !a->g || !a->beta || !a->state || !a->o) return PLA_ERR_INVALID_ARGUMENT;
  const long long head = static_cast<long long>(a->dk) * a->dv;
  if (a->n > 1 && a->state_row < head * a->hv) return PLA_ERR_INVALID_ARGUMENT;  // states that share memory would race
  const Bytes state = strided(a->state, 4, {{head * a->hv, 1}, {a->n, a->state_row}});
  const Bytes o = dense(a->o, static_cast<long long>(a->n) * a->hv * a->dv, es);
  const Bytes read[3] = {strided(a->q, es, {{a->dk, 1}, {a->hk, a->q_head}, {a->n, a->q_row}}),
                         strided(a->k, es, {{a->dk, 1}, {a->hk, a->k_head}, {a->n, a->k_row}}),
                         strided(a->v, es, {{a->dv, 1}, {a->hv, a->v_head}, {a->n, a->v_row}})};
  for (const Bytes& r : read)
    if (meets(state, r) || meets(o, r)) return PLA_ERR_INVALID_ARGUMENT;
  if (meets(state, o)) return PLA_ERR_INVALID_ARGUMENT;
  int sms, st;
  if ((st = current_sm100(&sms)) != PLA_OK) return st;
  DeltaStepParams p = {};
  p.q = a->q, p.k = a->k, p.v = a->v, p.g = a->g, p.beta = a->beta;
  p.q_row = a->q_row, p.q_head = a->q_head, p.k_row = a->k_row, p.k_head = a->k_head;
  p.v_row = a->v_row, p.v_head = a->v_head, p.g_row = a->g_row, p.g_head = a->g_head;
  p.beta_row = a->beta_row, p.beta_head = a->beta_head;
  p.state = a->state;
  p.state_row = a->state_row;
  p.o = a->o;
  p.n = a->n, p.hk = a->hk, p.hv = a->hv, p.dk = a->dk, p.dv = a->dv;
  p.gates32 = a->gates32 != 0;
  p.scale = a->scale;
  // whole states by bulk copies: rows a warp can share out evenly, 16-byte addresses
  const bool whole = (a->dv == 32 || a->dv == 64 || a->dv == 128) && a->dk <= 128 && head % 4 == 0 && a->state_row % 4 == 0 &&
                     aligned_to(a->state, 16);
  return with_type(a->dtype, [&](auto zero) {
    using T = decltype(zero);
    if (whole) {
      const long long blocks = static_cast<long long>(p.n) * p.hv;
      if (blocks > kMaxGrid) return static_cast<int>(PLA_ERR_TOO_LARGE);
      const size_t shared = static_cast<size_t>(head) * 4;
      const int st = allow_shared<delta_step<T>>(128 * 128 * 4);
      if (st != PLA_OK) return st;
      delta_step<T><<<static_cast<int>(blocks), kStepWarps * 32, shared, as_stream(stream)>>>(p);
      return launched("delta_step");
    }
    const auto go = [&](auto rows) {
      constexpr int ROWS = decltype(rows)::value;
      const long long blocks = static_cast<long long>(p.n) * p.hv * ((p.dv + 31) / 32);
      if (blocks > kMaxGrid) return static_cast<int>(PLA_ERR_TOO_LARGE);
      delta_step_any<T, ROWS><<<static_cast<int>(blocks), kStepAnyWarps * 32, 0, as_stream(stream)>>>(p);
      return launched("delta_step_any");
    };
    if (p.dk <= 64) return go(Int<4>{});
    if (p.dk <= 128) return go(Int<8>{});
    return go(Int<16>{});
  });
}

}  // extern "C"
