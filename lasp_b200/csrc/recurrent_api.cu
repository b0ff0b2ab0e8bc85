// extern "C" entry points of the recurrences over tokens: what they refuse, before anything is launched.
#include "recurrent.cuh"

namespace {

constexpr int64_t kMostBlocks = 2147483647;
constexpr int kMostTokens = 2147480000, kMostChannels = kMostTokens;   // (a run, chunk or tile beyond is still an int)

bool known(int dtype) { return dtype == LASP_F32 || dtype == LASP_BF16 || dtype == LASP_F16; }
bool params_ok(int dtype, int param_dtype) { return param_dtype == LASP_F32 || param_dtype == dtype; }
bool bits_ok(const void* p, int bits) { return !p || bits == 32 || bits == 64; }
bool missing(const lasp_tokens& t) { return t.data == nullptr; }

int check_conv(const lasp_conv_args* a) {
  if (!a) return LASP_ERR_NULL;
  if (!known(a->dtype) || !params_ok(a->dtype, a->param_dtype)) return LASP_ERR_DTYPE;
  if (a->rows <= 0 || a->tokens < 0 || a->channels <= 0 || a->width < 2 || a->width > 4 || a->sequences < 0) return LASP_ERR_SHAPE;
  if (a->activation != LASP_ACT_NONE && a->activation != LASP_ACT_SILU) return LASP_ERR_SHAPE;
  if (a->sequences && (a->rows != 1 || !bits_ok(a->offsets, a->index_bits))) return LASP_ERR_SHAPE;
  if (a->rows > 65535 || a->sequences > (1 << 17) || a->tokens > kMostTokens || a->channels > kMostChannels) return LASP_ERR_TOO_LARGE;
  if (!a->weight || (a->sequences && !a->offsets) || (a->tokens && missing(a->x))) return LASP_ERR_NULL;
  return LASP_OK;
}

int check_scan(const lasp_scan_args* a) {
  if (!a) return LASP_ERR_NULL;
  if (!known(a->dtype) || !params_ok(a->dtype, a->param_dtype)) return LASP_ERR_DTYPE;
  if (a->rows <= 0 || a->tokens < 0 || a->channels <= 0 || a->states <= 0 || a->states > 64 || a->sequences < 0) return LASP_ERR_SHAPE;
  if (a->groups <= 0 || a->groups > 65535 || a->channels % a->groups) return LASP_ERR_SHAPE;
  if (a->sequences && (a->rows != 1 || !bits_ok(a->offsets, a->index_bits))) return LASP_ERR_SHAPE;
  // (a block for every eight channels of every sequence at most; a thread for every dB and dC of a group)
  const int64_t sequences = a->sequences ? (int64_t)a->sequences + 1 : a->rows;
  if (a->tokens > kMostTokens || a->channels > kMostChannels || sequences * (a->channels / 8 + a->groups) > kMostBlocks ||
      (int64_t)a->rows * a->tokens / 2 > kMostBlocks)
    return LASP_ERR_TOO_LARGE;
  if (!a->A || (a->sequences && !a->offsets)) return LASP_ERR_NULL;
  if (a->tokens && (missing(a->u) || missing(a->dt) || missing(a->B) || missing(a->C))) return LASP_ERR_NULL;
  return LASP_OK;
}

}  // namespace

extern "C" {

size_t lasp_b200_conv_workspace_bytes(const lasp_conv_args* a) {
  return a && known(a->dtype) && a->rows > 0 && a->tokens >= 0 && a->channels > 0 && a->width >= 2 && a->width <= 4 ? lasp::conv_workspace(*a) : 0;
}

int lasp_b200_conv_forward(const lasp_conv_args* a, void* stream) {
  if (const int st = check_conv(a); st != LASP_OK) return st;
  if (a->tokens && missing(a->y)) return LASP_ERR_NULL;
  return lasp::status_of(lasp::conv_forward(*a, static_cast<cudaStream_t>(stream)));
}

int lasp_b200_conv_backward(const lasp_conv_args* a, void* stream) {
  if (const int st = check_conv(a); st != LASP_OK) return st;
  if (a->tokens && (missing(a->dy) || missing(a->dx))) return LASP_ERR_NULL;
  if (a->dweight || a->dbias) {
    const size_t need = lasp::conv_workspace(*a);
    if (need && !a->ws) return LASP_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(a->ws) & 15) return LASP_ERR_ALIGN;
    if (a->ws_bytes < need) return LASP_ERR_WORKSPACE;
  }
  return lasp::status_of(lasp::conv_backward(*a, static_cast<cudaStream_t>(stream)));
}

size_t lasp_b200_scan_kept_bytes(const lasp_scan_args* a) { return check_scan(a) == LASP_OK ? lasp::scan_kept(*a) : 0; }
size_t lasp_b200_scan_forward_workspace_bytes(const lasp_scan_args* a) { return check_scan(a) == LASP_OK ? lasp::scan_forward_workspace(*a) : 0; }
size_t lasp_b200_scan_workspace_bytes(const lasp_scan_args* a) { return check_scan(a) == LASP_OK ? lasp::scan_workspace(*a) : 0; }

int lasp_b200_scan_forward(const lasp_scan_args* a, void* stream) {
  if (const int st = check_scan(a); st != LASP_OK) return st;
  if (a->tokens && missing(a->y)) return LASP_ERR_NULL;
  const size_t need = lasp::scan_forward_workspace(*a);
  if (need && !a->ws) return LASP_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(a->kept) | (need ? reinterpret_cast<uintptr_t>(a->ws) : 0)) & 15) return LASP_ERR_ALIGN;
  if ((a->kept && a->kept_bytes < lasp::scan_kept(*a)) || a->ws_bytes < need) return LASP_ERR_WORKSPACE;
  return lasp::status_of(lasp::scan_forward(*a, static_cast<cudaStream_t>(stream)));
}

int lasp_b200_scan_backward(const lasp_scan_args* a, void* stream) {
  if (const int st = check_scan(a); st != LASP_OK) return st;
  if (a->tokens && (missing(a->dy) || missing(a->du) || missing(a->ddt) || missing(a->dB) || missing(a->dC) || (!missing(a->z) && missing(a->dz))))
    return LASP_ERR_NULL;
  if (!a->ws || (a->tokens && !a->kept)) return LASP_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(a->kept) | reinterpret_cast<uintptr_t>(a->ws)) & 15) return LASP_ERR_ALIGN;
  if (a->kept_bytes < lasp::scan_kept(*a) || a->ws_bytes < lasp::scan_workspace(*a)) return LASP_ERR_WORKSPACE;
  return lasp::status_of(lasp::scan_backward(*a, static_cast<cudaStream_t>(stream)));
}

int lasp_b200_conv_step(const lasp_conv_step_args* a, void* stream) {
  if (!a) return LASP_ERR_NULL;
  if (!known(a->dtype) || !params_ok(a->dtype, a->param_dtype)) return LASP_ERR_DTYPE;
  if (a->rows <= 0 || a->channels <= 0 || a->width < 2 || a->width > 4 || a->slot_count < 0 || !bits_ok(a->slots, a->index_bits)) return LASP_ERR_SHAPE;
  if (a->activation != LASP_ACT_NONE && a->activation != LASP_ACT_SILU) return LASP_ERR_SHAPE;
  if (a->rows > 65535 || a->channels > kMostChannels) return LASP_ERR_TOO_LARGE;
  if (!a->weight || missing(a->x) || missing(a->y) || (a->slot_count && !a->state)) return LASP_ERR_NULL;
  return lasp::status_of(lasp::conv_step(*a, static_cast<cudaStream_t>(stream)));
}

int lasp_b200_scan_step(const lasp_scan_step_args* a, void* stream) {
  if (!a) return LASP_ERR_NULL;
  if (!known(a->dtype) || !params_ok(a->dtype, a->param_dtype)) return LASP_ERR_DTYPE;
  if (a->rows <= 0 || a->channels <= 0 || a->states <= 0 || a->states > 64 || a->slot_count < 0 || !bits_ok(a->slots, a->index_bits)) return LASP_ERR_SHAPE;
  if (a->groups <= 0 || a->channels % a->groups) return LASP_ERR_SHAPE;
  if (a->rows > 65535 || a->channels > kMostChannels) return LASP_ERR_TOO_LARGE;
  if (!a->A || missing(a->u) || missing(a->dt) || missing(a->B) || missing(a->C) || missing(a->y) || (a->slot_count && !a->state)) return LASP_ERR_NULL;
  return lasp::status_of(lasp::scan_step(*a, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
