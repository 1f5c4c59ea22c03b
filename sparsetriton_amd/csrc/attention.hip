// Attention over segments of packed rows: argument checks and dispatch of the
// entry points (the kernels are in attention.h, built per type).
#include "attention.h"

static int attn_check(const st_attn_args* a) {
  if (!a || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads || a->dim <= 0) return ST_ERR_ARG;
  if (a->dim % 8 || a->dim > ST_ATTN_MAX_DIM) return ST_ERR_UNSUPPORTED;
  if (a->dtype != ST_F32 && a->dtype != ST_F16 && a->dtype != ST_BF16) return ST_ERR_UNSUPPORTED;
  if (a->window < 0 || a->sinks < 0 || (a->sinks && !a->window)) return ST_ERR_ARG;
  if (!(a->scale > 0.f) || !(a->scale < 3.0e38f)) return ST_ERR_ARG;
  for (int tile : {a->q_tile, a->k_tile})
    if (tile != ST_ATTN_TILE && tile != ST_ATTN_SMALL_TILE) return ST_ERR_ARG;
  for (int64_t n : {a->n_q_items, a->n_q_joins, a->n_k_items, a->n_k_joins})
    if (n < 0 || n >= (1ll << 31)) return ST_ERR_ARG;
  return ST_OK;
}

// Rows at 16-byte addresses, and a tile's rows within a 32-bit byte offset of its first.
static bool attn_rows_ok(const st_attn_args* a, const void* p, int64_t row, int64_t head) {
  const int64_t esz = a->dtype == ST_F32 ? 4 : 2, group = a->heads / a->kv_heads;
  if (((uintptr_t)p | (uint64_t)(row * esz) | (uint64_t)(head * esz)) & 15) return false;
  return row >= 0 && head >= 0 && row < (1ll << 29) && head < (1ll << 29) &&
         (row * (ST_ATTN_TILE + 1) + head * (group + 1) + a->dim) * esz < (1ll << 31) - 64;
}

static st::AttnArgs attn_args(const st_attn_args* a) {
  st::AttnArgs g{};
  g.q = a->q, g.k = a->k, g.v = a->v, g.o = a->o, g.dout = a->dout;
  g.o_rest = a->o_rest, g.out = a->o, g.rest = a->o_rest, g.dq = a->dq, g.dk = a->dk, g.dv = a->dv;
  g.lse = a->lse, g.delta = a->delta, g.parts = a->parts;
  g.q_row = a->q_row, g.q_head = a->q_head, g.k_row = a->k_row, g.k_head = a->k_head;
  g.v_row = a->v_row, g.v_head = a->v_head, g.do_row = a->dout_row, g.do_head = a->dout_head;
  g.key_mask = a->key_mask;
  g.by_kv_heads = st::attn_divisor(a->kv_heads), g.by_group = st::attn_divisor(a->heads / a->kv_heads);
  g.heads = a->heads, g.kv_heads = a->kv_heads, g.group = a->heads / a->kv_heads;
  g.D = a->dim, g.causal = a->causal != 0;
  g.window = a->window, g.sinks = a->sinks;
  g.scale = a->scale;
  g.scale_log2 = a->scale * 1.44269504088896341f;
  return g;
}

static int attn_run_any(const st_attn_args* a, st::AttnPass pass, const st::AttnArgs& g, hipStream_t s) {
  if (a->dtype == ST_BF16) return st::attn_run_bf16(pass, g, s);
  if (a->dtype == ST_F16) return st::attn_run_f16(pass, g, s);
  return st::attn_run_f32(pass, g, s);
}

extern "C" int st_attn_workspace(int kv_heads, int dim, int64_t q_parts, int64_t k_parts, int64_t* floats) {
  if (kv_heads <= 0 || dim <= 0 || dim > ST_ATTN_MAX_DIM || q_parts < 0 || k_parts < 0 || !floats) return ST_ERR_ARG;
  const int64_t dp = (dim + 31) / 32 * 32;
  const int64_t q = q_parts * kv_heads * ST_ATTN_TILE * (dp + 4), k = k_parts * kv_heads * ST_ATTN_TILE * 2 * dp;
  *floats = q > k ? q : k;
  return ST_OK;
}

extern "C" int st_attn_forward(const st_attn_args* a, st_stream_t stream) {
  const int rc = attn_check(a);
  if (rc != ST_OK) return rc;
  if (a->n_q_items == 0) return ST_OK;
  if (!a->q || !a->o || !a->q_items || (((uintptr_t)a->o | (uintptr_t)a->o_rest) & 15)) return ST_ERR_ARG;
  if (a->n_q_joins && (!a->q_joins || !a->parts || ((uintptr_t)a->parts & 15))) return ST_ERR_ARG;
  if (!attn_rows_ok(a, a->q, a->q_row, a->q_head) || !attn_rows_ok(a, a->k, a->k_row, a->k_head) ||
      !attn_rows_ok(a, a->v, a->v_row, a->v_head))
    return ST_ERR_ARG;
  st::AttnArgs g = attn_args(a);
  g.items = (const st::AttnItem*)a->q_items, g.n_items = (int)a->n_q_items;
  g.by_items = st::attn_divisor(g.n_items);
  g.joins = (const st::AttnJoin*)a->q_joins, g.n_joins = (int)a->n_q_joins;
  g.tile = a->q_tile, g.item_major = a->q_item_major != 0;
  return attn_run_any(a, st::kAttnForward, g, (hipStream_t)stream);
}

extern "C" int st_attn_backward(const st_attn_args* a, st_stream_t stream) {
  int rc = attn_check(a);
  if (rc != ST_OK) return rc;
  if (a->n_q_items && (!a->q || !a->o || !a->dout || !a->lse || !a->delta || !a->dq || !a->q_items)) return ST_ERR_ARG;
  if (a->n_k_items && (!a->k || !a->v || !a->dk || !a->dv || !a->k_items)) return ST_ERR_ARG;
  if ((a->n_q_joins && !a->q_joins) || (a->n_k_joins && !a->k_joins)) return ST_ERR_ARG;
  if ((a->n_q_joins || a->n_k_joins) && (!a->parts || ((uintptr_t)a->parts & 15))) return ST_ERR_ARG;
  if (((uintptr_t)a->o | (uintptr_t)a->o_rest | (uintptr_t)a->dq | (uintptr_t)a->dk | (uintptr_t)a->dv) & 15) return ST_ERR_ARG;
  if (!attn_rows_ok(a, a->q, a->q_row, a->q_head) || !attn_rows_ok(a, a->k, a->k_row, a->k_head) ||
      !attn_rows_ok(a, a->v, a->v_row, a->v_head) || !attn_rows_ok(a, a->dout, a->dout_row, a->dout_head))
    return ST_ERR_ARG;
  st::AttnArgs g = attn_args(a);
  if (a->n_q_items) {
    g.items = (const st::AttnItem*)a->q_items, g.n_items = (int)a->n_q_items;
    g.by_items = st::attn_divisor(g.n_items);
    g.joins = (const st::AttnJoin*)a->q_joins, g.n_joins = (int)a->n_q_joins;
    g.tile = a->q_tile, g.item_major = a->q_item_major != 0;
    rc = attn_run_any(a, st::kAttnDq, g, (hipStream_t)stream);
    if (rc != ST_OK) return rc;
  }
  if (!a->n_k_items) return ST_OK;
  g.items = (const st::AttnItem*)a->k_items, g.n_items = (int)a->n_k_items;
  g.by_items = st::attn_divisor(g.n_items);
  g.joins = (const st::AttnJoin*)a->k_joins, g.n_joins = (int)a->n_k_joins;
  g.tile = a->k_tile, g.item_major = a->k_item_major != 0;
  return attn_run_any(a, st::kAttnDkv, g, (hipStream_t)stream);
}
