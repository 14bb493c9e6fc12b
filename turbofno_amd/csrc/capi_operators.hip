// C ABI of the operators around the spectral layer: argument validation and dispatch by type. Declarations are in include/turbofno.h.
#include "../../include/turbofno.h"
#include "capi_error.h"
#include "mix_kernel.h"
#include "places.h"
#include <algorithm>
#include <initializer_list>
#include <memory>
#include <new>

using tfno::fail;
using tfno::hip_status;
using tfno::overlap;
using tfno::packed;
using tfno::Place;
using tfno::place;

namespace {

static_assert(TURBOFNO_C64 == tfno::kC64 && TURBOFNO_F32 == tfno::kF32 && TURBOFNO_BF16 == tfno::kBF16, "types");
static_assert(TURBOFNO_ACT_NONE == tfno::kActNone && TURBOFNO_ACT_RELU == tfno::kActRelu && TURBOFNO_ACT_SILU == tfno::kActSilu &&
              TURBOFNO_ACT_GELU_TANH == tfno::kActGeluTanh, "activations");

constexpr long kMaxPositions = 1L << 36;                // 2^37 real columns: strips of 64, and bytes, fit every index

int check_sizes(int type, long P, int N, int K, int act)
{
    if (type < TURBOFNO_C64 || type > TURBOFNO_BF16) return fail(TURBOFNO_ERR_INVALID_ARG, "type %d is none of TURBOFNO_C64, _F32, _BF16", type);
    if (P < 0 || P > kMaxPositions) return fail(TURBOFNO_ERR_INVALID_ARG, "P=%ld positions: 0 to 2^36 are taken", P);
    if (N <= 0 || K <= 0) return fail(TURBOFNO_ERR_INVALID_ARG, "N and K must be positive (N=%d K=%d)", N, K);
    if (N > 65536 || K > 65536) return fail(TURBOFNO_ERR_UNSUPPORTED, "N=%d, K=%d: at most 65536 channels are taken", N, K);
    if (act < TURBOFNO_ACT_NONE || act > TURBOFNO_ACT_GELU_TANH) return fail(TURBOFNO_ERR_INVALID_ARG, "activation %d is none of TURBOFNO_ACT_*", act);
    return TURBOFNO_OK;
}

// an operand of `rows` rows of P elements: there where P > 0, rows that do not overlap
int check_rows(const char* name, const void* p, long P, int rows, long ld, bool optional = false)
{
    if (!p) return optional || P == 0 ? TURBOFNO_OK : fail(TURBOFNO_ERR_INVALID_ARG, "%s is null", name);
    if (rows > 1 && ld < P) return fail(TURBOFNO_ERR_INVALID_ARG, "%s: %ld elements between channels, but P=%ld positions", name, ld, P);
    if (ld < 0 || ld > kMaxPositions) return fail(TURBOFNO_ERR_INVALID_ARG, "%s: channel stride %ld", name, ld);
    return TURBOFNO_OK;
}
int check_there(const char* name, const void* p) { return p ? TURBOFNO_OK : fail(TURBOFNO_ERR_INVALID_ARG, "%s is null", name); }

bool overlap(const void* a, long rows_a, long ld_a, size_t size_a, const void* b, long rows_b, long ld_b, size_t size_b, long P)
{
    return overlap(place(a, rows_a, ld_a, size_a, P), place(b, rows_b, ld_b, size_b, P));
}

// a result may be an operand, element for element, and overlaps none otherwise
bool clash(const void* out, long ldo, const void* in, long ldi, int rows, size_t size, long P)
{
    return overlap(out, rows, ldo, size, in, rows, ldi, size, P) && !(out == in && (ldo == ldi || rows == 1));
}

// a result against operands that every block may read until the end of the call
bool among(const Place& result, std::initializer_list<Place> operands)
{
    for (const Place& operand : operands)
        if (overlap(result, operand)) return true;
    return false;
}

// Where the results of the clipping lie: apart from one another, from every gradient but their own, and from the norm and the workspace
struct Span {
    const char *from, *to;
    int of;
};
int check_clip_places(Span* spans, int count, const void* const* grads, void* const* out, const long* sizes, const int* types, const Place& norm, const Place& workspace)
{
    auto span = [&](const void* p, int i) { return Span{ static_cast<const char*>(p), static_cast<const char*>(p) + sizes[i] * (long)tfno::size_of(types[i]), i }; };
    auto before = [](const Span& a, const Span& b) { return a.from < b.from; };
    int n = 0;
    for (int i = 0; i < count; ++i) {
        if (!sizes[i]) continue;
        const Span o = span(out[i], i), g = span(grads[i], i);
        for (const Place* p : { &norm, &workspace })
            if (p->at && ((o.from < p->at + p->width && p->at < o.to) || (g.from < p->at + p->width && p->at < g.to)))
                return fail(TURBOFNO_ERR_INVALID_ARG, "tensor %d overlaps the norm or the workspace", i);
        spans[n++] = o;
    }
    if (!std::is_sorted(spans, spans + n, before)) std::sort(spans, spans + n, before);
    for (int k = 1; k < n; ++k)
        if (spans[k].from < spans[k - 1].to) {
            const int a = spans[k - 1].of, b = spans[k].of;
            return fail(TURBOFNO_ERR_INVALID_ARG, "results %d and %d overlap: each would be scaled for both", a < b ? a : b, a < b ? b : a);
        }
    for (int i = 0; i < count; ++i) {
        if (!sizes[i] || out[i] == grads[i]) continue;
        const Span g = span(grads[i], i);
        if (g.to <= spans[0].from || g.from >= spans[n - 1].to) continue;       // beside all of them, as a list of its own mostly is
        const Span* o = std::lower_bound(spans, spans + n, g, [](const Span& a, const Span& b) { return a.to <= b.from; });
        if (o < spans + n && o->from < g.to) return fail(TURBOFNO_ERR_INVALID_ARG, "result %d overlaps gradient %d", o->of, i);
    }
    return TURBOFNO_OK;
}

#define CHECK(call) if (int rc_ = (call)) return rc_

}  // namespace

extern "C" {

int turbofno_mix(int type, long P, int N, int K, const void* x, long ldx, const void* W, const void* bias, const void* residual, long ldr, int act,
                 void* z, long ldz, void* y, long ldy, void* stream)
{
    CHECK(check_sizes(type, P, N, K, act));
    CHECK(check_rows("x", x, P, K, ldx));
    CHECK(check_there("W", W));
    CHECK(check_rows("residual", residual, P, N, ldr, true));
    CHECK(check_rows("z", z, P, N, ldz, true));
    CHECK(check_rows("y", y, P, N, ldy));
    const size_t e = tfno::size_of(type);
    if (overlap(x, K, ldx, e, y, N, ldy, e, P) || overlap(x, K, ldx, e, z, N, ldz, e, P)) return fail(TURBOFNO_ERR_INVALID_ARG, "a result overlaps x");
    if (overlap(y, N, ldy, e, z, N, ldz, e, P)) return fail(TURBOFNO_ERR_INVALID_ARG, "y and z overlap");
    if (clash(y, ldy, residual, ldr, N, e, P) || clash(z, ldz, residual, ldr, N, e, P)) return fail(TURBOFNO_ERR_INVALID_ARG, "a result overlaps residual without being it");
    const Place small[2] = { packed(W, (long)(e * N * K)), packed(bias, (long)(e * N)) };
    if (among(place(y, N, ldy, e, P), { small[0], small[1] }) || among(place(z, N, ldz, e, P), { small[0], small[1] })) return fail(TURBOFNO_ERR_INVALID_ARG, "a result overlaps W or bias");
    const int v = tfno::values_of(type);
    const tfno::MixParams q = { x, nullptr, W, bias, residual, nullptr, nullptr, y, z, P * v, ldx * v, 0, ldr * v, ldy * v, ldz * v, N, K, K, act };
    const hipStream_t st = (hipStream_t)stream;
    return hip_status(type == TURBOFNO_C64 ? tfno::launch_mix_c64(q, false, st) : type == TURBOFNO_F32 ? tfno::launch_mix_f32(q, false, st)
                                           : tfno::launch_mix_bf16(q, false, st), "mix launch");
}

int turbofno_mix_8bit(int type, long P, int N, int K, const void* xq, long ldx, const float* xscale, const void* Wq, const float* wscale, const void* bias,
                      const void* residual, long ldr, int act, void* y, long ldy, void* stream)
{
    CHECK(check_sizes(type, P, N, K, act));
    CHECK(check_rows("xq", xq, P, K, ldx));
    CHECK(check_there("Wq", Wq));
    CHECK(check_there("wscale", wscale));
    if (P) CHECK(check_there("xscale", xscale));
    CHECK(check_rows("residual", residual, P, N, ldr, true));
    CHECK(check_rows("y", y, P, N, ldy));
    const int v = tfno::values_of(type);
    if (overlap(xq, K, ldx, v, y, N, ldy, tfno::size_of(type), P)) return fail(TURBOFNO_ERR_INVALID_ARG, "y overlaps xq");
    if (clash(y, ldy, residual, ldr, N, tfno::size_of(type), P)) return fail(TURBOFNO_ERR_INVALID_ARG, "y overlaps residual without being it");
    if (among(place(y, N, ldy, tfno::size_of(type), P), { packed(Wq, (long)N * K * v), packed(bias, N * (long)tfno::size_of(type)), packed(xscale, 4 * P), packed(wscale, 4l * N) }))
        return fail(TURBOFNO_ERR_INVALID_ARG, "y overlaps Wq, bias or a scale");
    const tfno::MixParams q = { xq, nullptr, Wq, bias, residual, xscale, wscale, y, nullptr, P * v, ldx * v, 0, ldr * v, ldy * v, 0, N, K, K, act };
    return hip_status(tfno::launch_mix_8bit(q, type, (hipStream_t)stream), "mix_8bit launch");
}

int turbofno_mix_input_grad(int type, long P, int N, int K, const void* gy, long ldgy, const void* z, long ldz, const void* W, int act, void* gz, long ldgz,
                            void* gx, long ldgx, void* stream)
{
    CHECK(check_sizes(type, P, N, K, act));
    CHECK(check_rows("gy", gy, P, N, ldgy));
    CHECK(check_there("W", W));
    const bool slopes = act != TURBOFNO_ACT_NONE;
    if (slopes) {
        CHECK(check_rows("z", z, P, N, ldz));
        CHECK(check_rows("gz", gz, P, N, ldgz));
    }
    CHECK(check_rows("gx", gx, P, K, ldgx));
    const size_t e = tfno::size_of(type);
    if (overlap(gx, K, ldgx, e, gy, N, ldgy, e, P) || (slopes && (overlap(gx, K, ldgx, e, z, N, ldz, e, P) || overlap(gx, K, ldgx, e, gz, N, ldgz, e, P) ||
                                                                  overlap(gz, N, ldgz, e, gy, N, ldgy, e, P) || overlap(gz, N, ldgz, e, z, N, ldz, e, P))))
        return fail(TURBOFNO_ERR_INVALID_ARG, "a result overlaps gy, z or the other result");
    const Place weights = packed(W, (long)(e * N * K));
    if (overlap(place(gx, K, ldgx, e, P), weights) || (slopes && overlap(place(gz, N, ldgz, e, P), weights))) return fail(TURBOFNO_ERR_INVALID_ARG, "a result overlaps W");
    const int v = tfno::values_of(type);
    const tfno::MixParams q = { gy, slopes ? z : nullptr, W, nullptr, nullptr, nullptr, nullptr, gx, slopes ? gz : nullptr, P * v, ldgy * v, ldz * v, 0, ldgx * v,
                                ldgz * v, K, N, K, act };
    const hipStream_t st = (hipStream_t)stream;
    return hip_status(type == TURBOFNO_C64 ? tfno::launch_mix_c64(q, true, st) : type == TURBOFNO_F32 ? tfno::launch_mix_f32(q, true, st)
                                           : tfno::launch_mix_bf16(q, true, st), "mix_input_grad launch");
}

size_t turbofno_mix_weight_grad_workspace_bytes(int type, long P, int N, int K)
{
    if (check_sizes(type, P, N, K, TURBOFNO_ACT_NONE)) return 0;
    return tfno::mix_weight_grad_workspace(type, P, N, K);
}

int turbofno_mix_weight_grad(int type, long P, int N, int K, const void* gz, long ldgz, const void* x, long ldx, void* gW, void* gbias, void* workspace,
                             size_t workspace_bytes, void* stream)
{
    CHECK(check_sizes(type, P, N, K, TURBOFNO_ACT_NONE));
    CHECK(check_rows("gz", gz, P, N, ldgz));
    CHECK(check_rows("x", x, P, K, ldx));
    CHECK(check_there("gW", gW));
    const size_t e = tfno::size_of(type), need = tfno::mix_weight_grad_workspace(type, P, N, K);
    // blocks read gz and x while others write their sums or, without a second kernel, the results
    const Place results[3] = { packed(gW, (long)(e * N * K)), packed(gbias, (long)(e * N)), packed(workspace, (long)need) };
    for (int i = 0; i < 3; ++i) {
        if (overlap(results[i], place(gz, N, ldgz, e, P)) || overlap(results[i], place(x, K, ldx, e, P)))
            return fail(TURBOFNO_ERR_INVALID_ARG, "gW, gbias or the workspace overlaps gz or x");
        if (overlap(results[i], results[(i + 1) % 3])) return fail(TURBOFNO_ERR_INVALID_ARG, "gW, gbias and the workspace overlap one another");
    }
    if (!workspace || workspace_bytes < need) return fail(TURBOFNO_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : (size_t)0, need);
    return hip_status(tfno::launch_mix_weight_grad(type, P, N, K, gz, ldgz, x, ldx, gW, gbias, workspace, (hipStream_t)stream), "mix_weight_grad launch");
}

static int norm_on(bool eight, int type, long P, int K, const void* x, long ldx, const void* residual, long ldr, const float* gain, float eps, void* s, long lds,
                   void* y, long ldy, float* rstd, void* stream)
{
    CHECK(check_sizes(type, P, 1, K, TURBOFNO_ACT_NONE));
    CHECK(check_rows("x", x, P, K, ldx));
    CHECK(check_rows("residual", residual, P, K, ldr, true));
    CHECK(check_there("gain", gain));
    CHECK(check_rows("s", s, P, K, lds, true));
    CHECK(check_rows(eight ? "q" : "y", y, P, K, ldy));
    if (eight && P) CHECK(check_there("scale", rstd));
    if (!(eps >= 0.f)) return fail(TURBOFNO_ERR_INVALID_ARG, "eps=%g must not be negative", (double)eps);
    const int v = tfno::values_of(type);
    const size_t e = tfno::size_of(type), ey = eight ? (size_t)v : e;
    auto taken = [&](const void* in, long ldi) {
        return clash(s, lds, in, ldi, K, e, P) || (eight ? overlap(y, K, ldy, ey, in, K, ldi, e, P) : clash(y, ldy, in, ldi, K, e, P));
    };
    if (taken(x, ldx) || taken(residual, ldr))
        return fail(TURBOFNO_ERR_INVALID_ARG, "a result overlaps an operand without being it");
    if (overlap(y, K, ldy, ey, s, K, lds, e, P)) return fail(TURBOFNO_ERR_INVALID_ARG, "the results overlap");
    const Place px = place(x, K, ldx, e, P), pr = place(residual, K, ldr, e, P), ps = place(s, K, lds, e, P), py = place(y, K, ldy, ey, P);
    if (among(packed(gain, 4l * K), { ps, py }) || among(packed(rstd, 4 * P), { px, pr, ps, py, packed(gain, 4l * K) }))
        return fail(TURBOFNO_ERR_INVALID_ARG, "a result overlaps gain, or %s another operand", eight ? "scale" : "rstd");
    const tfno::NormParams q = { x, residual, gain, s, y, rstd, P * v, ldx * v, ldr * v, lds * v, ldy * v, K, eps };
    return hip_status(tfno::launch_rms_norm(q, type, eight, (hipStream_t)stream), eight ? "rms_norm_8bit launch" : "rms_norm launch");
}

int turbofno_rms_norm(int type, long P, int K, const void* x, long ldx, const void* residual, long ldr, const float* gain, float eps, void* s, long lds, void* y,
                      long ldy, float* rstd, void* stream)
{
    return norm_on(false, type, P, K, x, ldx, residual, ldr, gain, eps, s, lds, y, ldy, rstd, stream);
}

int turbofno_rms_norm_8bit(int type, long P, int K, const void* x, long ldx, const void* residual, long ldr, const float* gain, float eps, void* s, long lds,
                           void* q, long ldq, float* scale, void* stream)
{
    return norm_on(true, type, P, K, x, ldx, residual, ldr, gain, eps, s, lds, q, ldq, scale, stream);
}

size_t turbofno_rms_norm_backward_workspace_bytes(int type, long P, int K)
{
    if (check_sizes(type, P, 1, K, TURBOFNO_ACT_NONE)) return 0;
    return tfno::rms_norm_backward_workspace(type, P, K);
}

int turbofno_rms_norm_backward(int type, long P, int K, const void* gy, long ldgy, const void* s, long lds, const float* gain, const float* rstd, const void* gs,
                               long ldgs, void* gx, long ldgx, float* ggain, void* workspace, size_t workspace_bytes, void* stream)
{
    CHECK(check_sizes(type, P, 1, K, TURBOFNO_ACT_NONE));
    CHECK(check_rows("gy", gy, P, K, ldgy));
    CHECK(check_rows("s", s, P, K, lds));
    CHECK(check_there("gain", gain));
    if (P) CHECK(check_there("rstd", rstd));
    CHECK(check_rows("gs", gs, P, K, ldgs, true));
    CHECK(check_rows("gx", gx, P, K, ldgx));
    CHECK(check_there("ggain", ggain));
    const size_t e = tfno::size_of(type), need = tfno::rms_norm_backward_workspace(type, P, K);
    if (clash(gx, ldgx, gy, ldgy, K, e, P) || clash(gx, ldgx, s, lds, K, e, P) || clash(gx, ldgx, gs, ldgs, K, e, P)) return fail(TURBOFNO_ERR_INVALID_ARG, "gx overlaps an operand without being it");
    const Place px = place(gx, K, ldgx, e, P), pg = packed(gain, 4l * K), pr = packed(rstd, 4 * P), po = packed(ggain, 4l * K);
    if (among(px, { pg, pr, po })) return fail(TURBOFNO_ERR_INVALID_ARG, "gx overlaps gain, rstd or ggain");
    if (among(packed(workspace, (long)need), { place(gy, K, ldgy, e, P), place(s, K, lds, e, P), place(gs, K, ldgs, e, P), px, pg, pr, po }))
        return fail(TURBOFNO_ERR_INVALID_ARG, "the workspace overlaps an operand");
    if (!workspace || workspace_bytes < need) return fail(TURBOFNO_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : (size_t)0, need);
    const int v = tfno::values_of(type);
    const tfno::NormGradParams q = { gy, s, gs, gain, rstd, gx, ggain, static_cast<float*>(workspace), P * v, ldgy * v, lds * v, ldgs * v, ldgx * v, K };
    return hip_status(tfno::launch_rms_norm_backward(q, type, (hipStream_t)stream), "rms_norm_backward launch");
}

size_t turbofno_clip_grad_norm_workspace_bytes(int count) { return count < 0 ? 0 : tfno::clip_workspace(count); }

int turbofno_clip_grad_norm(int count, const void* const* grads, void* const* out, const long* sizes, const int* types, float max_norm, float* norm, void* workspace,
                            size_t workspace_bytes, void* stream)
{
    if (count < 0) return fail(TURBOFNO_ERR_INVALID_ARG, "count=%d", count);
    if (count && (!grads || !out || !sizes || !types)) return fail(TURBOFNO_ERR_INVALID_ARG, "a list is null");
    CHECK(check_there("norm", norm));
    if (!(max_norm >= 0.f)) return fail(TURBOFNO_ERR_INVALID_ARG, "max_norm=%g must not be negative", (double)max_norm);
    for (int i = 0; i < count; ++i) {
        if (types[i] < TURBOFNO_C64 || types[i] > TURBOFNO_BF16) return fail(TURBOFNO_ERR_INVALID_ARG, "types[%d]=%d is none of TURBOFNO_C64, _F32, _BF16", i, types[i]);
        if (sizes[i] < 0 || sizes[i] > kMaxPositions) return fail(TURBOFNO_ERR_INVALID_ARG, "sizes[%d]=%ld", i, sizes[i]);
        if (sizes[i] && (!grads[i] || !out[i])) return fail(TURBOFNO_ERR_INVALID_ARG, "tensor %d is null", i);
    }
    const size_t need = tfno::clip_workspace(count);
    Span few[128];
    const std::unique_ptr<Span[]> many(count > 128 ? new (std::nothrow) Span[count] : nullptr);
    if (count > 128 && !many) return fail(TURBOFNO_ERR_INVALID_ARG, "no host memory for the places of %d tensors", count);
    const Place at_norm = packed(norm, sizeof(float)), at_workspace = packed(workspace, (long)need);
    if (overlap(at_norm, at_workspace)) return fail(TURBOFNO_ERR_INVALID_ARG, "norm overlaps the workspace");
    CHECK(check_clip_places(count > 128 ? many.get() : few, count, grads, out, sizes, types, at_norm, at_workspace));
    if (!workspace || workspace_bytes < need) return fail(TURBOFNO_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : (size_t)0, need);
    return hip_status(tfno::launch_clip(count, grads, out, sizes, types, max_norm, norm, workspace, (hipStream_t)stream), "clip_grad_norm launch");
}

}  // extern "C"
