// extern "C" entry points of the recurrent mixers' operators (ssm.hip, ssm_bwd.hip,
// conv.hip, norm.hip): checks, the layout of workspaces, launches.  Declarations are in
// include/lizard_hip.h.
#include "../../include/lizard_hip.h"
#include "capi.hpp"
#include "conv.hpp"
#include "norm.hpp"
#include "ssm.hpp"

using lz::fail;
using lz::hip_status;

namespace {

constexpr long long ROWS_LIMIT = (1LL << 31) - (1LL << 20);

bool aligned(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }
bool stride_ok(long long s) { return s >= 0 && s <= LZ_MIXER_MAX_STRIDE; }

// --- ssm --------------------------------------------------------------------

int check_ssm_sizes(const char* what, long long batch, long long length, long long channels,
                    long long state, long long groups) {
  if (batch <= 0 || length <= 0 || channels <= 0 || state <= 0 || groups <= 0)
    return fail(1, "%s: sizes must be positive (batch %lld, length %lld, channels %lld, state "
                   "%lld, groups %lld)", what, batch, length, channels, state, groups);
  if (state > LZ_SSM_MAX_STATE)
    return fail(1, "%s: state %lld beyond %d unsupported", what, state, LZ_SSM_MAX_STATE);
  if (channels % groups)
    return fail(1, "%s: groups %lld must divide channels %lld", what, groups, channels);
  if (channels > LZ_MIXER_MAX_STRIDE)
    return fail(1, "%s: %lld channels beyond %d unsupported", what, channels, LZ_MIXER_MAX_STRIDE);
  if (batch * length > ROWS_LIMIT)
    return fail(1, "%s: %lld tokens exceed the 2^31 - 2^20 limit", what, batch * length);
  // workgroups of up to 1024 threads, segments only where there are fewer blocks than CUs
  const long long blocks = groups * ((channels / groups + 63) / 64);
  if (batch * blocks > (1LL << 21) || batch > 65535)
    return fail(1, "%s: batch %lld x %lld blocks of channels exceed the grid", what, batch, blocks);
  return 0;
}

int check_ssm(const char* what, const lz_ssm_args* a, bool step) {
  if (!a) return fail(1, "%s: null arguments", what);
  if (int rc = check_ssm_sizes(what, a->batch, step ? 1 : a->length, a->channels, a->state, a->groups))
    return rc;
  if (!a->x || !a->dt || !a->B || !a->C || !a->A) return fail(1, "%s: null input pointer", what);
  const bool strides = stride_ok(a->x_token) && stride_ok(a->dt_token) &&
                       (!a->z || stride_ok(a->z_token)) && stride_ok(a->B_token) &&
                       stride_ok(a->C_token);
  if (!step && !strides)
    return fail(1, "%s: token strides must be in [0, %d]", what, LZ_MIXER_MAX_STRIDE);
  if (!stride_ok(a->B_group) || !stride_ok(a->C_group))
    return fail(1, "%s: group strides must be in [0, %d]", what, LZ_MIXER_MAX_STRIDE);
  if (a->x_batch < 0 || a->dt_batch < 0 || a->z_batch < 0 || a->B_batch < 0 || a->C_batch < 0)
    return fail(1, "%s: batch strides must not be negative", what);
  return 0;
}

lz::Ssm ssm_of(const lz_ssm_args* a, bool step) {
  lz::Ssm p = {};
  p.x = a->x, p.dt = a->dt, p.z = a->z, p.B = a->B, p.C = a->C;
  p.A = a->A, p.D = a->D, p.bias = a->dt_bias;
  p.x_b = a->x_batch, p.dt_b = a->dt_batch, p.z_b = a->z_batch, p.B_b = a->B_batch;
  p.C_b = a->C_batch;
  if (!step) {
    p.x_t = (int)a->x_token, p.dt_t = (int)a->dt_token, p.z_t = a->z ? (int)a->z_token : 0;
    p.B_t = (int)a->B_token, p.C_t = (int)a->C_token;
  }
  p.B_g = (int)a->B_group, p.C_g = (int)a->C_group;
  p.batch = a->batch, p.L = step ? 1 : a->length, p.E = a->channels, p.N = a->state;
  p.G = a->groups, p.Eg = p.E / p.G, p.gblocks = (p.Eg + lz::SSM_CH - 1) / lz::SSM_CH;
  p.softplus = a->softplus;
  p.tiles = (p.L + lz::SSM_TT - 1) / lz::SSM_TT;
  return p;
}

// S segments of whole tiles
void ssm_split(lz::Ssm& p, int S) {
  p.seg_tiles = (p.tiles + S - 1) / S;
  p.S = (p.tiles + p.seg_tiles - 1) / p.seg_tiles;
}

// Floats of the segments' own states and sums of delta
size_t ssm_records(const lz::Ssm& p) {
  return (size_t)p.batch * (p.S - 1) * p.E * (p.N + 1);
}

// Whether a thread's share of a row (SSM_V channels) is whole and aligned in every row
bool ssm_vec(const lz::Ssm& p, bool bf16, std::initializer_list<const void*> rows) {
  const int V = lz::SSM_V, bytes = V * (bf16 ? 2 : 4);
  if (p.Eg % V) return false;
  for (long long s : {p.x_b, p.dt_b, p.z ? p.z_b : 0LL, (long long)p.x_t, (long long)p.dt_t,
                      (long long)p.z_t})
    if (s % V) return false;
  for (const void* r : rows)
    if (!aligned(r, bytes)) return false;
  return aligned(p.x, bytes) && aligned(p.dt, bytes) && aligned(p.z, bytes);
}

lz::Ssm ssm_sizes(int batch, int length, int channels, int state, int groups, bool backward) {
  lz_ssm_args a = {};
  a.batch = batch, a.length = length, a.channels = channels, a.state = state, a.groups = groups;
  lz::Ssm p = ssm_of(&a, false);
  ssm_split(p, lz::ssm_segments(p.batch, p.G, p.Eg, p.L, backward));
  return p;
}

size_t ssm_part_bc(const lz::Ssm& p) {
  return (size_t)p.G * p.gblocks * p.batch * p.L * 2 * lz::ssm_bwd_padded(p.N);
}

// Sums over n that pass from one launch to the next
size_t ssm_acc(const lz::Ssm& p) {
  return p.N > lz::SSM_BWD_STATES ? 2 * (size_t)p.batch * p.L * p.E : 0;
}

// What the forward keeps for the backward: the rows that z gates, then the tiles' states
void ssm_kept(lz::Ssm& p, float* states) {
  p.mixed = p.z ? states : nullptr;
  p.saved = states && p.z ? states + (size_t)p.batch * p.L * p.E : states;
}

bool ssm_sizes_ok(int batch, int length, int channels, int state, int groups) {
  return check_ssm_sizes("ssm", batch, length, channels, state, groups) == 0;
}

}  // namespace

extern "C" size_t lz_ssm_states_bytes(int batch, int length, int channels, int state, int gated) {
  if (!ssm_sizes_ok(batch, length, channels, state, 1)) return 0;
  const size_t tiles = (length + lz::SSM_TT - 1) / lz::SSM_TT, rows = gated ? length : 0;
  return (size_t)batch * channels * (rows + tiles * state) * 4;
}

extern "C" size_t lz_ssm_fwd_workspace_bytes(int batch, int length, int channels, int state,
                                             int groups) {
  if (!ssm_sizes_ok(batch, length, channels, state, groups)) return 0;
  return ssm_records(ssm_sizes(batch, length, channels, state, groups, false)) * 4;
}

extern "C" int lz_ssm_fwd(const lz_ssm_args* args, const float* state_in, float* state_out,
                          const int* lengths, void* y, float* states, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (int rc = check_ssm("ssm_fwd", args, false)) return rc;
  if (!y) return fail(1, "ssm_fwd: null output pointer");
  lz::Ssm p = ssm_of(args, false);
  ssm_split(p, lz::ssm_segments(p.batch, p.G, p.Eg, p.L, false));
  const size_t need = ssm_records(p) * 4;
  if (need && (!workspace || workspace_bytes < need))
    return fail(1, "ssm_fwd: workspace of %zu bytes given, %zu needed", workspace_bytes, need);
  p.state_in = state_in, p.state_out = state_out, p.lengths = lengths, p.y = y;
  ssm_kept(p, states);
  p.rec = (float*)workspace;
  p.dsum = p.rec + (size_t)p.batch * (p.S - 1) * p.E * p.N;
  return hip_status(lz::launch_ssm_fwd(p, args->bf16 != 0, ssm_vec(p, args->bf16, {y}),
                                       (hipStream_t)stream), "ssm_fwd");
}

extern "C" int lz_ssm_decode_step(const lz_ssm_args* args, float* state, void* y, void* stream) {
  if (int rc = check_ssm("ssm_decode_step", args, true)) return rc;
  if (!state || !y) return fail(1, "ssm_decode_step: null output pointer");
  lz::Ssm p = ssm_of(args, true);
  p.y = y;
  return hip_status(lz::launch_ssm_step(p, state, args->bf16 != 0, (hipStream_t)stream),
                    "ssm_decode_step");
}

extern "C" size_t lz_ssm_bwd_workspace_bytes(int batch, int length, int channels, int state,
                                             int groups) {
  if (!ssm_sizes_ok(batch, length, channels, state, groups)) return 0;
  const lz::Ssm p = ssm_sizes(batch, length, channels, state, groups, true);
  return (ssm_part_bc(p) + (size_t)p.batch * p.S * p.E * (p.N + 2) + ssm_records(p) +
          ssm_acc(p)) * 4;
}

extern "C" int lz_ssm_bwd(const lz_ssm_args* args, const float* states, const void* dy, void* dx,
                          void* ddt, void* dz, void* dB, void* dC, float* dA, float* dD,
                          float* ddt_bias, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_ssm("ssm_bwd", args, false)) return rc;
  if (!states || !dy || !dx || !ddt || !dB || !dC || !dA || (args->z && !dz))
    return fail(1, "ssm_bwd: null pointer");
  lz::Ssm p = ssm_of(args, false);
  ssm_split(p, lz::ssm_segments(p.batch, p.G, p.Eg, p.L, true));
  const size_t need = lz_ssm_bwd_workspace_bytes(p.batch, p.L, p.E, p.N, p.G);
  if (!workspace || workspace_bytes < need)
    return fail(1, "ssm_bwd: workspace of %zu bytes given, %zu needed", workspace_bytes, need);
  ssm_kept(p, const_cast<float*>(states));
  lz::SsmGrad g = {};
  g.dy = dy, g.dx = dx, g.ddt = ddt, g.dz = dz;
  g.acc = (float*)workspace;
  g.part_bc = g.acc + ssm_acc(p);
  g.part_a = g.part_bc + ssm_part_bc(p);
  g.part_d = g.part_a + (size_t)p.batch * p.S * p.E * p.N;
  g.rec = g.part_d + (size_t)p.batch * p.S * p.E * 2;
  g.dsum = g.rec + (size_t)p.batch * (p.S - 1) * p.E * p.N;
  g.acc_step = (long long)p.batch * p.L * p.E;
  g.NQ = lz::ssm_bwd_padded(p.N);
  const bool vec = ssm_vec(p, args->bf16, {dy, dx, ddt, dz});
  return hip_status(lz::launch_ssm_bwd(p, g, dB, dC, dA, dD, ddt_bias, args->bf16 != 0, vec,
                                       (hipStream_t)stream), "ssm_bwd");
}

// --- short_conv ---------------------------------------------------------------

namespace {

int check_conv(const char* what, const void* x, const float* w, long long batch, long long length,
               long long channels, long long taps, long long x_batch, long long x_token) {
  if (batch <= 0 || length <= 0 || channels <= 0 || taps <= 0)
    return fail(1, "%s: sizes must be positive (batch %lld, length %lld, channels %lld, taps %lld)",
                what, batch, length, channels, taps);
  if (taps > LZ_CONV_MAX_TAPS)
    return fail(1, "%s: %lld taps beyond %d unsupported", what, taps, LZ_CONV_MAX_TAPS);
  if (channels > LZ_MIXER_MAX_STRIDE)
    return fail(1, "%s: %lld channels beyond %d unsupported", what, channels, LZ_MIXER_MAX_STRIDE);
  if (batch * length > ROWS_LIMIT)
    return fail(1, "%s: %lld tokens exceed the 2^31 - 2^20 limit", what, batch * length);
  if (batch > (1 << 20) || batch * ((channels + 511) / 512) > (1LL << 23))
    return fail(1, "%s: batch %lld x %lld channels exceed the grid", what, batch, channels);
  if (x_batch < 0 || !stride_ok(x_token))
    return fail(1, "%s: strides of x must be in [0, %d] a token", what, LZ_MIXER_MAX_STRIDE);
  if (x && w) return 0;
  return fail(1, "%s: null input pointer", what);
}

lz::Conv conv_of(int batch, int length, int channels, bool backward = false) {
  lz::Conv p = {};
  p.batch = batch, p.L = length, p.C = channels;
  lz::conv_split(p, backward);
  return p;
}

}  // namespace

extern "C" int lz_short_conv_fwd(const void* x, long long x_batch, long long x_token,
                                 const float* weight, const float* bias, const void* state_in,
                                 void* state_out, const int* lengths, void* y, int batch,
                                 int length, int channels, int taps, int silu, int bf16,
                                 void* stream) {
  if (int rc = check_conv("short_conv_fwd", x, weight, batch, length, channels, taps, x_batch, x_token))
    return rc;
  if (!y) return fail(1, "short_conv_fwd: null output pointer");
  lz::Conv p = conv_of(batch, length, channels);
  p.x = x, p.w = weight, p.bias = bias, p.state_in = state_in, p.state_out = state_out;
  p.lengths = lengths, p.y = y, p.x_b = x_batch, p.x_t = (int)x_token, p.act = silu;
  return hip_status(lz::launch_conv(p, taps, nullptr, nullptr, nullptr, bf16 != 0,
                                    channels >= lz::CONV_FWD_V, (hipStream_t)stream),
                    "short_conv_fwd");
}

extern "C" int lz_short_conv_decode_step(const void* x, long long x_batch, const float* weight,
                                         const float* bias, void* state, void* y, int batch,
                                         int channels, int taps, int silu, int bf16, void* stream) {
  if (int rc = check_conv("short_conv_decode_step", x, weight, batch, 1, channels, taps, x_batch, 0))
    return rc;
  if (!y || (taps > 1 && !state)) return fail(1, "short_conv_decode_step: null output pointer");
  if (batch > 65535) return fail(1, "short_conv_decode_step: batch %d exceeds the grid", batch);
  lz::Conv p = conv_of(batch, 1, channels);
  p.x = x, p.w = weight, p.bias = bias, p.state_out = state, p.y = y, p.x_b = x_batch, p.act = silu;
  return hip_status(lz::launch_conv_step(p, taps, bf16 != 0, (hipStream_t)stream),
                    "short_conv_decode_step");
}

extern "C" size_t lz_short_conv_bwd_workspace_bytes(int batch, int length, int channels, int taps) {
  if (batch <= 0 || length <= 0 || channels <= 0 || taps <= 0) return 0;
  return (size_t)conv_of(batch, length, channels, true).run_blocks * (taps + 1) * channels * 4;
}

extern "C" int lz_short_conv_bwd(const void* x, long long x_batch, long long x_token,
                                 const float* weight, const float* bias, const void* dy, void* dx,
                                 float* dweight, float* dbias, int batch, int length, int channels,
                                 int taps, int silu, int bf16, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (int rc = check_conv("short_conv_bwd", x, weight, batch, length, channels, taps, x_batch, x_token))
    return rc;
  if (!dy || !dx || !dweight) return fail(1, "short_conv_bwd: null pointer");
  lz::Conv p = conv_of(batch, length, channels, true);
  p.x = x, p.w = weight, p.bias = bias, p.x_b = x_batch, p.x_t = (int)x_token, p.act = silu;
  const size_t need = lz_short_conv_bwd_workspace_bytes(batch, length, channels, taps);
  if (!workspace || workspace_bytes < need)
    return fail(1, "short_conv_bwd: workspace of %zu bytes given, %zu needed", workspace_bytes, need);
  hipError_t e = lz::launch_conv(p, taps, dy, dx, (float*)workspace, bf16 != 0,
                                 channels >= lz::CONV_BWD_V, (hipStream_t)stream);
  if (e == hipSuccess)
    e = lz::launch_conv_sums(p, taps, (const float*)workspace, dweight, dbias, (hipStream_t)stream);
  return hip_status(e, "short_conv_bwd");
}

// --- group_norm ----------------------------------------------------------------

namespace {

int check_norm_sizes(const char* what, long long batch, long long length, long long groups,
                     long long width) {
  if (batch <= 0 || length <= 0 || groups <= 0 || width <= 0)
    return fail(1, "%s: sizes must be positive (batch %lld, length %lld, groups %lld, width %lld)",
                what, batch, length, groups, width);
  if (width > LZ_NORM_MAX_WIDTH)
    return fail(1, "%s: groups of %lld channels beyond %d unsupported", what, width,
                LZ_NORM_MAX_WIDTH);
  if (groups * width > LZ_MIXER_MAX_STRIDE || groups > 65535)
    return fail(1, "%s: %lld groups of %lld channels unsupported", what, groups, width);
  if (batch * length > ROWS_LIMIT)
    return fail(1, "%s: %lld tokens exceed the 2^31 - 2^20 limit", what, batch * length);
  return 0;
}

int check_norm(const char* what, const lz_group_norm_args* a) {
  if (!a) return fail(1, "%s: null arguments", what);
  if (int rc = check_norm_sizes(what, a->batch, a->length, a->groups, a->width)) return rc;
  if (!a->x) return fail(1, "%s: null input pointer", what);
  if (a->x_batch < 0 || a->x_token < 0 || a->x_group < 0 || a->gate_batch < 0 ||
      a->gate_token < 0 || a->gate_group < 0)
    return fail(1, "%s: strides must not be negative", what);
  if (!(a->eps >= 0.f)) return fail(1, "%s: eps must not be negative", what);
  return 0;
}

lz::Norm norm_of(const lz_group_norm_args* a, bool backward) {
  lz::Norm p = {};
  p.x = a->x, p.gate = a->gate, p.w = a->weight, p.bias = a->bias;
  p.x_b = a->x_batch, p.x_t = a->x_token, p.x_g = a->x_group;
  p.z_b = a->gate_batch, p.z_t = a->gate_token, p.z_g = a->gate_group;
  p.batch = a->batch, p.L = a->length, p.G = a->groups, p.W = a->width, p.act = a->silu;
  p.eps = a->eps;
  // sequences that follow each other in every tensor are one
  if (p.x_b == p.L * p.x_t && (!p.gate || p.z_b == p.L * p.z_t)) {
    p.L *= p.batch;
    p.batch = 1;
  }
  lz::norm_split(p, backward);
  return p;
}

}  // namespace

extern "C" int lz_group_norm_fwd(const lz_group_norm_args* args, void* y, void* stream) {
  if (int rc = check_norm("group_norm_fwd", args)) return rc;
  if (!y) return fail(1, "group_norm_fwd: null output pointer");
  lz::Norm p = norm_of(args, false);
  p.y = y;
  return hip_status(lz::launch_norm_fwd(p, args->bf16 != 0, (hipStream_t)stream),
                    "group_norm_fwd");
}

extern "C" size_t lz_group_norm_bwd_workspace_bytes(int batch, int length, int groups, int width) {
  if (check_norm_sizes("group_norm", batch, length, groups, width)) return 0;
  lz_group_norm_args a = {};
  a.batch = batch, a.length = length, a.groups = groups, a.width = width;
  return (size_t)norm_of(&a, true).row_blocks * 2 * groups * width * 4;
}

extern "C" int lz_group_norm_bwd(const lz_group_norm_args* args, const void* dy, void* dx,
                                 void* dgate, float* dweight, float* dbias, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (int rc = check_norm("group_norm_bwd", args)) return rc;
  if (!dy || !dx || (args->gate && !dgate)) return fail(1, "group_norm_bwd: null pointer");
  const lz::Norm p = norm_of(args, true);
  const size_t need =
      dweight || dbias
          ? lz_group_norm_bwd_workspace_bytes(args->batch, args->length, args->groups, args->width)
          : 0;
  if (need && (!workspace || workspace_bytes < need))
    return fail(1, "group_norm_bwd: workspace of %zu bytes given, %zu needed", workspace_bytes, need);
  return hip_status(lz::launch_norm_bwd(p, dy, dx, dgate, need ? (float*)workspace : nullptr,
                                        dweight, dbias, args->bf16 != 0, (hipStream_t)stream),
                    "group_norm_bwd");
}
