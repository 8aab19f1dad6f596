// f8_step.cu — the step of a model with e4m3 weights, and the rules behind the head of any STT model.
//
// Per layer: norm1 of x plus the block before -> e4m3 rows; in_proj; RoPE and the KV-ring write;
// attention; its output as e4m3 rows; out_proj; norm2 of x plus that -> e4m3 rows; linear_in;
// activation -> e4m3 rows; linear_out. A block's output is not added to x by its product but by the
// next norm, which reads x anyway.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "common.cuh"
#include "engine.h"
#include "rules.cuh"
#include "sm100.cuh"

namespace svl {
namespace {

struct QkvParams {
  const float* y;         // [nb][q_dim + 2 kv_dim]
  const float2* rope_cs;  // [nb][head_dim / 2]
  const int* pos;         // [nb]
  int nb, q_dim, kv_dim, head_dim, ring_cap, windowed, kv_bf16;
  float* q;               // [nb][q_dim]
  void* k_ring;
  void* v_ring;
  int64_t ring_stream_stride;
};

// RoPE on q and k (rope_i, nn/transformer.rs:339-340: pairs (2i, 2i+1) rotate by pos * f_i), q to its
// buffer, k and v into the ring slots of the new position. One thread per pair; a few bytes per
// stream, bound by its launch.
__global__ void qkv_kernel(const QkvParams p) {
  const int pairs = (p.q_dim + 2 * p.kv_dim) / 2, half = p.head_dim / 2;
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  const int b = blockIdx.y;
  pdl_launch();
  pdl_wait();
  if (i >= pairs) return;
  const float2 v = reinterpret_cast<const float2*>(p.y + (int64_t)b * 2 * pairs)[i];
  const int row = 2 * i;
  const bool is_q = row < p.q_dim, is_v = row >= p.q_dim + p.kv_dim;
  float2 z = v;
  if (!is_v) {
    const float2 cs = p.rope_cs[(int64_t)b * half + i % half];
    z.x = v.x * cs.x - v.y * cs.y;
    z.y = v.x * cs.y + v.y * cs.x;
  }
  if (is_q) {
    reinterpret_cast<float2*>(p.q + (int64_t)b * p.q_dim)[i] = z;
    return;
  }
  const int rr = is_v ? row - p.q_dim - p.kv_dim : row - p.q_dim;
  const int slot = p.windowed ? p.pos[b] % p.ring_cap : p.pos[b];
  const int64_t at = b * p.ring_stream_stride + ((int64_t)(rr / p.head_dim) * p.ring_cap + slot) * p.head_dim + rr % p.head_dim;
  void* ring = is_v ? p.v_ring : p.k_ring;
  if (p.kv_bf16)
    reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(ring) + at)[0] = __floats2bfloat162_rn(z.x, z.y);
  else
    reinterpret_cast<float2*>(static_cast<float*>(ring) + at)[0] = z;
}

struct ActParams {
  const float* y;  // [nb][y_stride]: gate rows then value rows when gated
  int64_t y_stride;
  int f;           // hidden width
  uint8_t* q;
  int64_t q_stride;
  float* scales;
  int64_t scale_stride;
};

// The feed-forward activation (FeedForwardLayer, nn/transformer.rs:438-464) and its outputs as e4m3
// rows: a warp per block of 128 columns, 4 per lane, like svl_add_norm_f8_device's without a norm.
// The outputs keep 4 significant bits, so the fast exponential is ample. Bound by the f32 reads.
template <int FFN>
__global__ void __launch_bounds__(256) act_f8_kernel(const ActParams p) {
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int block = blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_launch();
  pdl_wait();
  if (block * kF8Block >= p.f) return;
  const float* y = p.y + (int64_t)b * p.y_stride;
  const int c = block * kF8Block + lane * 4;
  float z[4], top = kF8Tiny;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    z[j] = 0.f;
    if (c + j < p.f) {
      const float x = y[c + j];
      if (FFN == SVL_FFN_GATED_SILU)
        z[j] = __fdividef(x, 1.0f + __expf(-x)) * y[p.f + c + j];
      else if (FFN == SVL_FFN_PLAIN_GELU_TANH)
        z[j] = gelu_tanh_ref(x);
      else
        z[j] = gelu_erf_ref(x);
    }
    top = max_nan(top, fabsf(z[j]));
  }
  for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float inv = __fdiv_rn(kF8Max, top);
  uint8_t* q = p.q + (int64_t)b * p.q_stride + c;
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (c + j < p.f) q[j] = to_e4m3(z[j] * inv);
  if (lane == 0) p.scales[(int64_t)block * p.scale_stride + b] = __fdiv_rn(top, kF8Max);
}

// A launch whose setup runs beside the end of the kernel before.
template <class P>
void launch_early(void (*kernel)(const P), dim3 grid, const P& p, cudaStream_t st, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, p), what);
}

int64_t padded(int k) { return (k + 15) / 16 * 16; }

void norm(const State& s, const float* x, int nb, int k, const float* residual, const Norm* n, float* sum, cudaStream_t st) {
  NormF8Params p{};
  p.x = x;
  p.x_stride = k;
  p.residual = residual;
  p.residual_stride = k;
  if (n) {
    p.norm = n->kind;
    p.weight = n->w.as<float>();
    p.bias = n->b.as<float>();
    p.eps = n->eps;
  }
  p.rows = nb;
  p.k = k;
  p.sum = residual ? sum : nullptr;
  p.sum_stride = k;
  p.q = s.f8_q.as<uint8_t>();
  p.q_stride = padded(k);
  p.scales = s.f8_s.as<float>();
  p.scale_stride = s.max_batch;
  launch_norm_f8(p, st);
}

void product(const State& s, const Linear& L, int nb, float* out, cudaStream_t st) {
  F8GemmParams p{};
  p.m = L.f8;
  p.q = s.f8_q.as<uint8_t>();
  p.q_stride = padded(L.k);
  p.scales = s.f8_s.as<float>();
  p.scale_stride = s.max_batch;
  p.rows = nb;
  p.out = out;
  p.out_stride = L.n;
  p.err = s.err.as<int>();
  launch_f8_gemm(p, st);
}

}  // namespace

void create_state_f8(Model& m, State& s) {
  const auto& c = m.cfg;
  const int64_t B = s.max_batch;
  const int qd = c.num_heads * c.head_dim, kvd = c.num_kv_heads * c.head_dim;
  const int kmax = std::max({c.d_model, qd, c.ffn_hidden});
  s.f8_q.alloc(B * padded(kmax));
  s.f8_s.alloc(B * ((kmax + kF8Block - 1) / kF8Block) * 4);
  const int ff = c.ffn_kind == SVL_FFN_GATED_SILU ? 2 * c.ffn_hidden : c.ffn_hidden;
  s.f8_y.alloc(B * std::max(qd + 2 * kvd, ff) * 4);
  s.f8_delta.alloc(B * c.d_model * 4);
  s.rope_cs.alloc(B * (c.head_dim / 2) * 8);
}

void enqueue_layers_f8(Model& m, State& s, int b0, int nb, cudaStream_t st, bool do_lin, bool do_attn) {
  const auto& c = m.cfg;
  const int d = c.d_model, hd = c.head_dim, qd = c.num_heads * hd, kvd = c.num_kv_heads * hd;
  float* x = s.x.as<float>() + (int64_t)b0 * d;
  float* delta = s.f8_delta.as<float>();
  float* y = s.f8_y.as<float>();
  float2* rope_cs = s.rope_cs.as<float2>() + (int64_t)b0 * (hd / 2);
  const int* pos = s.pos.as<int>() + b0;
  if (do_lin) launch_rope_table(pos, nb, m.inv_freq.as<float>(), hd / 2, rope_cs, st);
  for (int l = 0; l < c.num_layers; l++) {
    const Layer& L = m.layers[l];
    const LayerParams lp = layer_params(m, s, l, b0, nb);
    if (do_lin) {
      norm(s, x, nb, d, l ? delta : nullptr, &L.norm1, x, st);
      product(s, L.in_proj, nb, y, st);
      const GemvParams& g = lp.in_proj;
      const QkvParams k{y, rope_cs, pos, nb, qd, kvd, hd, g.ring_cap, g.windowed, g.kv_bf16, g.out, g.k_ring, g.v_ring, g.ring_stream_stride};
      launch_early(qkv_kernel, dim3(((qd + 2 * kvd) / 2 + 255) / 256, nb), k, st, "RoPE launch");
    }
    if (do_attn) launch_attention_decode(lp.attn, st);
    if (!do_lin) continue;
    norm(s, lp.attn.out, nb, qd, nullptr, nullptr, nullptr, st);
    product(s, L.out_proj, nb, delta, st);
    norm(s, x, nb, d, delta, &L.norm2, x, st);
    product(s, L.ff1, nb, y, st);
    const int f = c.ffn_hidden;
    const ActParams a{y, L.ff1.n, f, s.f8_q.as<uint8_t>(), padded(f), s.f8_s.as<float>(), s.max_batch};
    const dim3 grid((f + 8 * kF8Block - 1) / (8 * kF8Block), nb);
    const auto act = c.ffn_kind == SVL_FFN_GATED_SILU      ? act_f8_kernel<SVL_FFN_GATED_SILU>
                     : c.ffn_kind == SVL_FFN_PLAIN_GELU_TANH ? act_f8_kernel<SVL_FFN_PLAIN_GELU_TANH>
                                                             : act_f8_kernel<SVL_FFN_PLAIN_GELU_ERF>;
    launch_early(act, grid, a, st, "activation launch");
    product(s, L.ff2, nb, delta, st);
  }
}

void f8_flush(Model& m, State& s, int b0, int nb, cudaStream_t st) {
  float* x = s.x.as<float>() + (int64_t)b0 * m.cfg.d_model;
  norm(s, x, nb, m.cfg.d_model, s.f8_delta.as<float>(), nullptr, x, st);
}

void f8_head(Model& m, State& s, int nb, bool pending, cudaStream_t st) {
  float* x = s.x.as<float>();
  norm(s, x, nb, m.cfg.d_model, pending ? s.f8_delta.as<float>() : nullptr, &m.out_norm, x, st);
  product(s, m.text_linear, nb, s.logits.as<float>(), st);
}

// ---- rules ---------------------------------------------------------------------------------

void enqueue_rules(Model& m, State& s, int nb, cudaStream_t st) {
  RulesParams p{};
  p.logits = s.logits.p;
  p.logits_stride = m.stt.text_card;
  p.out = s.rules ? s.logits.p : nullptr;
  p.out_stride = m.stt.text_card;
  p.tokens = s.tok_out.as<int32_t>();
  p.rows = nb;
  p.vocab = m.stt.text_card;
  if (s.rules) {
    svl_logits_rules& r = p.rules;
    r.d_history = s.said.as<int32_t>();
    r.history_stride = r.history_cap = SVL_RULES_HISTORY;
    r.d_lengths = s.said_len.as<int32_t>();
    r.first_penalised = s.rules_first;
    r.d_repetition = s.rule_rep.as<float>();
    r.d_frequency = s.rule_freq.as<float>();
    r.d_presence = s.rule_pres.as<float>();
    r.d_bias_ids = s.rule_ids.as<int32_t>();
    r.d_bias_values = s.rule_vals.as<float>();
    r.bias_stride = r.bias_cap = SVL_RULES_BIASES;
    r.d_masks = s.rule_masks.as<uint32_t>();
    r.n_masks = s.max_batch;
    r.mask_stride = (m.stt.text_card + 31) / 32;
    r.d_mask_rows = s.rule_rows.as<int32_t>();
    r.append = 1;
  }
  launch_rules(p, st);
}

void state_set_rules(State& s, int stream, const svl_stt_rules* rules) {
  const int card = s.m->stt.text_card, B = s.max_batch;
  const int64_t words = (card + 31) / 32;
  if (rules) {
    if (!(rules->repetition > 0.f) || !std::isfinite(rules->repetition) || !std::isfinite(rules->frequency) ||
        !std::isfinite(rules->presence))
      throw Error(SVL_ERR_INVALID_INPUT, "penalties must be finite, the repetition penalty positive");
    if (rules->n_bias < 0 || rules->n_bias > SVL_RULES_BIASES || (rules->n_bias && (!rules->bias_ids || !rules->bias_values)))
      throw Error(SVL_ERR_INVALID_INPUT, "n_bias must be 0..256, with ids and values");
    if (rules->first_penalised < 0) throw Error(SVL_ERR_INVALID_INPUT, "first_penalised must be a token id");
    for (int i = 0; i < rules->n_bias; i++)
      if (rules->bias_ids[i] >= (uint32_t)card) throw Error(SVL_ERR_INVALID_INPUT, "biased token out of range");
  }
  if (!rules && !s.rules) return;
  check_cuda(cudaDeviceSynchronize(), "rules");
  cudaStream_t st = s.m->stream;
  if (!s.rules) {
    s.said.alloc((int64_t)B * SVL_RULES_HISTORY * 4);
    s.said_len.alloc((int64_t)B * 4);
    s.rule_rep.alloc((int64_t)B * 4);
    s.rule_freq.alloc((int64_t)B * 4);
    s.rule_pres.alloc((int64_t)B * 4);
    s.rule_ids.alloc((int64_t)B * SVL_RULES_BIASES * 4);
    s.rule_vals.alloc((int64_t)B * SVL_RULES_BIASES * 4);
    s.rule_masks.alloc(B * words * 4);
    s.rule_rows.alloc((int64_t)B * 4);
    check_cuda(cudaMemsetAsync(s.said_len.p, 0, s.said_len.bytes, st), "memset");
    check_cuda(cudaMemsetAsync(s.said.p, 0xff, s.said.bytes, st), "memset");
  }
  // The rules of streams [lo, hi), all of them the first time; without rules: no penalty, no entry, no grammar.
  const bool first_time = !s.rules;
  const int lo = first_time || stream < 0 ? 0 : stream, hi = first_time || stream < 0 ? B : stream + 1, n = hi - lo;
  std::vector<float> rep(n, 1.f), freq(n, 0.f), pres(n, 0.f), vals((size_t)n * SVL_RULES_BIASES, 0.f);
  std::vector<int32_t> ids((size_t)n * SVL_RULES_BIASES, -1), rows(n, -1);
  std::vector<uint32_t> masks(rules && rules->allowed ? (size_t)n * words : 0);
  for (int b = lo; rules && b < hi; b++) {
    if (stream >= 0 && b != stream) continue;
    const int at = b - lo;
    rep[at] = rules->repetition;
    freq[at] = rules->frequency;
    pres[at] = rules->presence;
    for (int i = 0; i < rules->n_bias; i++) {
      ids[(size_t)at * SVL_RULES_BIASES + i] = (int32_t)rules->bias_ids[i];
      vals[(size_t)at * SVL_RULES_BIASES + i] = rules->bias_values[i];
    }
    if (!rules->allowed) continue;
    rows[at] = b;
    std::copy(rules->allowed, rules->allowed + words, masks.begin() + (size_t)at * words);
  }
  auto up = [&](DevBuf& to, const auto& from, int64_t per_stream) {
    if (!from.empty())
      check_cuda(cudaMemcpyAsync(to.as<uint8_t>() + lo * per_stream * 4, from.data(), from.size() * 4, cudaMemcpyHostToDevice, st), "upload");
  };
  up(s.rule_rep, rep, 1);
  up(s.rule_freq, freq, 1);
  up(s.rule_pres, pres, 1);
  up(s.rule_ids, ids, SVL_RULES_BIASES);
  up(s.rule_vals, vals, SVL_RULES_BIASES);
  up(s.rule_rows, rows, 1);
  up(s.rule_masks, masks, words);
  check_cuda(cudaStreamSynchronize(st), "rules");  // the host values above live until here
  // The captured steps read the rules from these buffers, but for first_penalised, a kernel argument: they
  // are captured again only where the rules first come or it changes (a grammar's next set of tokens before
  // each step of an STT-1b stream, update and step: 1,099 us with a capture, 663 without; the step alone 614).
  if (first_time || (rules && rules->first_penalised != s.rules_first)) {
    for (auto& kv : s.graphs) cudaGraphExecDestroy(kv.second);
    s.graphs.clear();
    s.graph_kernels.clear();
  }
  if (rules) s.rules_first = rules->first_penalised;
  s.rules = true;
}

void state_copy_said(State& to, int dst, const State& from, int src, cudaStream_t st) {
  if (!to.rules) return;
  if (!from.rules) {
    check_cuda(cudaMemsetAsync(to.said_len.as<int>() + dst, 0, 4, st), "copy");
    return;
  }
  check_cuda(cudaMemcpyAsync(to.said.as<int32_t>() + (int64_t)dst * SVL_RULES_HISTORY,
                             from.said.as<int32_t>() + (int64_t)src * SVL_RULES_HISTORY, SVL_RULES_HISTORY * 4,
                             cudaMemcpyDeviceToDevice, st), "copy");
  check_cuda(cudaMemcpyAsync(to.said_len.as<int>() + dst, from.said_len.as<int>() + src, 4, cudaMemcpyDeviceToDevice, st), "copy");
}

}  // namespace svl
