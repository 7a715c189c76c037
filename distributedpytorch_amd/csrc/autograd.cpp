// Autograd nodes in C++ of group norm, dropout and cross attention.
//
// Their kernels take microseconds on the maps of one image.  A backward pass runs in autograd's own thread, where every
// Python object that the forward thread touched last is a cache miss: as Python nodes, a forward and backward pass of
// dropout on 1 x 256 x 33 x 33 took 77 us and of an fp32 group norm on 3 x 48 x 65 x 97 (46 us of kernels) 136 us of host
// time, where a node that only returns its gradient takes 38 us, nearly all of it the change of threads.  Here they take
// 27 to 54 and 60 to 99, by where the two threads run: dropout's backward 38 us where torch.relu's takes 38, group norm's 46
// with the gradient of x alone and 58 with those of weight and bias.
//
// Arguments are checked in Python (ops/group_norm.py, ops/dropout.py, ops/cross_attention.py).  What is here: layouts that
// the kernels read, outputs, workspaces, launches on the tensors' GPU and its current stream.  The operators are reachable as
// torch.ops.dpamd too, and hooks may put other tensors in a saved one's place: what a kernel would follow out of a tensor's
// memory (another device, type or size) is refused here as well.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <climits>

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The launchers of the kernel library, in the order of bind()'s addresses.
struct Launchers {
    long (*gn_workspace)(long, long, int, int, int);
    int (*gn_fwd)(const void*, const void*, const void*, const void*, void*, void*, void*, long, long, int, int, long, long,
                  float, int, int, void*);
    int (*gn_bwd)(const void*, const void*, const void*, const void*, const void*, const void*, void*, void*, void*, void*,
                  void*, long, long, int, int, long, long, long, int, int, void*);
    int (*dropout)(const void*, const void*, void*, long, unsigned, unsigned long long, const void*, int, int, void*);
    long (*xa_workspace)(int, int, int, int, int, int, int);
    int (*xa_fwd)(const void*, const void*, const void*, void*, void*, const void*, const void*, long, void*, const long*,
                  int, int, int, int, int, int, float, int, void*);
    int (*xa_bwd)(const void*, const void*, const void*, const void*, const void*, const void*, void*, void*, void*, void*,
                  const void*, const void*, long, void*, const long*, int, int, int, int, int, int, float, int, void*);
} dp;

void bind(at::IntArrayRef at) {
    TORCH_CHECK(at.size() == sizeof(dp) / sizeof(void*), "bind: an address for each launcher");
    for (size_t i = 0; i < at.size(); ++i) reinterpret_cast<void**>(&dp)[i] = reinterpret_cast<void*>(at[i]);
}

const void* in(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor some(const optional<Tensor>& t) { return t ? *t : Tensor(); }
bool wanted(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool beside(const Tensor& t, const Tensor& x) { return !t.defined() || t.device() == x.device(); }
bool like(const Tensor& t, const Tensor& x) {
    return !t.defined() || (t.device() == x.device() && t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes());
}

void* stream(const Tensor& t) {
    TORCH_CHECK(dp.gn_fwd != nullptr && t.is_cuda(), "dpamd operators take GPU tensors, after ops._backend.native()");
    return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

int type_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return 0;
        case at::kHalf: return 1;
        case at::kFloat: return 2;
        default: TORCH_CHECK_TYPE(false, "bf16, fp16 or fp32, got ", t.scalar_type());
    }
}

void check(int status, const char* what) {
    TORCH_CHECK(status == 0, "HIP launcher '", what, "' failed with status ", status);
}

// The kernels are closed to autograd: their results carry no history of their own.
void first_order(const char* what) {
    TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), what, ": no gradients of gradients (create_graph=True)");
}

// Nor do they carry a tangent along: one that came in would be missing from the result, without an error.
void no_tangent(const char* what, std::initializer_list<Tensor> inputs) {
    for (const Tensor& t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what, ": no forward-mode derivatives; set_backend('torch') "
                                    "runs the plain formulation, which has them");
}

Tensor workspace(long floats, const Tensor& like) {
    return floats > 0 ? at::empty({floats}, like.options().dtype(at::kFloat)) : Tensor();
}

// ------------------------------------------------------------------------------------------------ group norm
bool channels(const Tensor& t, const Tensor& map) {
    return !t.defined() || (t.device() == map.device() && t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == map.size(1));
}

// `t` where its memory is NHWC rows `ld` elements apart (a channels-last map or a channel slice of one), a channels-last
// copy otherwise.
Tensor rows(const Tensor& t, int64_t& ld) {
    const int64_t n = t.size(0), c = t.size(1), h = t.size(2), w = t.size(3);
    ld = c;
    if (t.is_contiguous(at::MemoryFormat::ChannelsLast)) return t;
    const int64_t s = w > 1 ? t.stride(3) : h > 1 ? t.stride(2) : t.stride(0);
    if ((t.stride(1) == 1 || c == 1) && s >= c && (h == 1 || t.stride(2) == w * s) && (n == 1 || t.stride(0) == h * w * s)) {
        ld = s;
        return t;
    }
    return t.contiguous(at::MemoryFormat::ChannelsLast);
}

Tensor map_like(const Tensor& x) { return at::empty_like(x, x.options(), at::MemoryFormat::ChannelsLast); }

Tensor vector32(const Tensor& t) { return t.defined() ? t.to(at::kFloat).contiguous() : t; }

Tensor norm_forward(const Tensor& map, const Tensor& w, const Tensor& b, const Tensor& residual, int64_t groups, double eps,
                    int64_t act, Tensor& stats) {
    TORCH_CHECK(map.dim() == 4 && groups > 0 && map.size(1) <= INT_MAX && channels(w, map) && channels(b, map) && like(residual, map),
                "group_norm_act: a [N, C, H, W] map, weight and bias [C], a residual like the map, all on one GPU");
    const c10::DeviceGuard guard(map.device());
    const Tensor y = map_like(map);
    stats = at::empty({map.size(0), groups, 2}, map.options().dtype(at::kDouble));
    if (map.numel() == 0) return y;
    int64_t ldx, ldr = map.size(1);
    const Tensor x = rows(map, ldx), r = residual.defined() ? rows(residual, ldr) : residual;
    const long n = x.size(0), hw = x.size(2) * x.size(3);
    const int c = (int)x.size(1), g = (int)groups;
    const Tensor ws = workspace(dp.gn_workspace(n, hw, c, g, (int)x.element_size()), x);
    check(dp.gn_fwd(in(x), in(r), in(w), in(b), out(y), out(stats), out(ws), n, hw, c, g, ldx, ldr, (float)eps, (int)act,
                    type_code(x), stream(x)), "gn_fwd");
    return y;
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                          const optional<Tensor>& residual, int64_t groups, double eps, int64_t act) {
        const Tensor w = some(weight), b = some(bias), r = some(residual), w32 = vector32(w), b32 = vector32(b);
        Tensor stats;
        const Tensor y = norm_forward(x, w32, b32, r, groups, eps, act, stats);
        // an activation's derivative needs z: the residual is kept for it (without one its gradient is dy itself)
        ctx->save_for_backward({x, act ? r : Tensor(), w32, b32, stats});
        const auto type = [](const Tensor& t) { return wanted(t) ? (int64_t)t.scalar_type() : int64_t(-1); };
        ctx->saved_data["plan"] = std::vector<int64_t>{groups, act, type(w), type(b), wanted(r)};
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_order("group_norm_act");
        const auto saved = ctx->get_saved_variables();
        const auto plan = ctx->saved_data["plan"].toIntVector();
        const Tensor &map = saved[0], &residual = saved[1], &dy = grads[0];
        const Tensor w = vector32(saved[2]), b = vector32(saved[3]), stats = saved[4].contiguous();
        TORCH_CHECK(like(dy, map) && like(residual, map) && channels(w, map) && channels(b, map) && beside(stats, map),
                    "group_norm_act: saved tensors and gradient belong on the map's GPU");
        const c10::DeviceGuard guard(map.device());
        const Tensor dx = map_like(map);
        Tensor dres = residual.defined() ? map_like(map) : Tensor(), dw, db;
        if (plan[2] >= 0) dw = at::empty_like(w);
        if (plan[3] >= 0) db = at::empty_like(b);
        if (map.numel()) {
            int64_t ldx, ldd, ldr = map.size(1);
            const Tensor x = rows(map, ldx), g = rows(dy, ldd), r = residual.defined() ? rows(residual, ldr) : residual;
            const long n = x.size(0), hw = x.size(2) * x.size(3);
            const int c = (int)x.size(1), groups = (int)plan[0];
            const Tensor ws = workspace(dp.gn_workspace(n, hw, c, groups, (int)x.element_size()), x);
            check(dp.gn_bwd(in(g), in(x), in(r), in(w), in(b), in(stats), out(dx), out(dres), out(dw), out(db), out(ws), n, hw, c,
                            groups, ldx, ldr, ldd, (int)plan[1], type_code(x), stream(x)), "gn_bwd");
        } else {
            if (dw.defined()) dw.zero_();
            if (db.defined()) db.zero_();
        }
        if (!dres.defined() && plan[4]) dres = dy;
        if (dw.defined()) dw = dw.to((at::ScalarType)plan[2]);
        if (db.defined()) db = db.to((at::ScalarType)plan[3]);
        return {dx, dw, db, dres, Tensor(), Tensor(), Tensor()};
    }
};

Tensor group_norm_act(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                      const optional<Tensor>& residual, int64_t groups, double eps, int64_t act) {
    const Tensor w = some(weight), b = some(bias), r = some(residual);
    no_tangent("group_norm_act", {x, w, b, r});
    if (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(b) || wanted(r)))
        return GroupNormAct::apply(x, weight, bias, residual, groups, eps, act);
    Tensor stats;
    return norm_forward(x, vector32(w), vector32(b), r, groups, eps, act, stats);
}

// ------------------------------------------------------------------------------------------------ dropout
// `t` where its elements fill their memory without gaps in one of torch's two layouts, else a copy
Tensor dense(const Tensor& t) {
    if (t.is_contiguous() || (t.dim() == 4 && t.is_contiguous(at::MemoryFormat::ChannelsLast))) return t;
    return t.contiguous();
}

// `t` in the memory order of strides
Tensor ordered(const Tensor& t, at::IntArrayRef strides) {
    if (!t.defined() || t.strides() == strides) return t;
    return at::empty_strided(t.sizes(), strides, t.options()).copy_(t);
}

Tensor drop(const Tensor& x, const Tensor& residual, int64_t threshold, int64_t seed, const Tensor& device_seed, bool word) {
    TORCH_CHECK(like(residual, x) && beside(device_seed, x) &&
                    (!device_seed.defined() || (device_seed.scalar_type() == at::kLong && device_seed.numel() == 1)),
                "dropout: a residual like x, a seed of one int64 on x's GPU");
    const c10::DeviceGuard guard(x.device());
    const Tensor y = at::empty_strided(x.sizes(), x.strides(), x.options());
    if (x.numel())
        check(dp.dropout(in(x), in(residual), out(y), x.numel(), (unsigned)threshold, (unsigned long long)seed, in(device_seed),
                         word, type_code(x), stream(x)), "dropout");
    return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& input, const optional<Tensor>& residual, int64_t threshold,
                          int64_t seed, const optional<Tensor>& device_seed, bool word) {
        const Tensor x = dense(input), r = some(residual), s = some(device_seed);
        ctx->save_for_backward({s});
        std::vector<int64_t> plan{threshold, seed, word, wanted(input), wanted(r)};
        plan.insert(plan.end(), x.strides().begin(), x.strides().end());
        ctx->saved_data["plan"] = std::move(plan);
        return drop(x, ordered(r, x.strides()), threshold, seed, s, word);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_order("dropout");
        const auto saved = ctx->get_saved_variables();
        const auto plan = ctx->saved_data["plan"].toIntVector();
        Tensor dx;
        if (plan[3])                   // the mask follows the memory order of the forward's input
            dx = drop(ordered(grads[0], at::IntArrayRef(plan).slice(5)), Tensor(), plan[0], plan[1], saved[0], plan[2]);
        return {dx, plan[4] ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor dropout(const Tensor& x, const optional<Tensor>& residual, int64_t threshold, int64_t seed,
               const optional<Tensor>& device_seed, bool word) {
    const Tensor r = some(residual);
    no_tangent("dropout", {x, r});
    if (at::GradMode::is_enabled() && (wanted(x) || wanted(r)))
        return Dropout::apply(x, residual, threshold, seed, device_seed, word);
    const Tensor d = dense(x);
    return drop(d, ordered(r, d.strides()), threshold, seed, some(device_seed), word);
}

// ------------------------------------------------------------------------------------------------ cross attention
// `t` [B, L, H, D] where the kernels can read its heads as 16-byte pieces, a dense copy otherwise
Tensor heads(const Tensor& t) {
    bool ok = t.stride(3) == 1 && ((uintptr_t)t.const_data_ptr() & 15) == 0;
    for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) == 1 || t.stride(i) % 8 == 0);
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

void add_strides(long*& at, const Tensor& t) {
    for (int i = 0; i < 3; ++i) *at++ = t.size(i) == 1 ? 0 : t.stride(i);
}

struct Shape {
    int B, Lq, Lk, Hk, share, D;
    Shape(const Tensor& q, const Tensor& k)
        : B((int)q.size(0)), Lq((int)q.size(1)), Lk((int)k.size(1)), Hk((int)k.size(2)), share((int)(q.size(2) / k.size(2))),
          D((int)q.size(3)) {}
};

// sizes that fit the launchers' ints, lengths and mask as the kernels read them
void fits(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Tensor& mask) {
    bool ok = q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3) &&
              k.size(2) > 0 && q.size(2) % k.size(2) == 0 && k.scalar_type() == q.scalar_type() &&
              v.scalar_type() == q.scalar_type() && beside(k, q) && beside(v, q) && beside(lengths, q) && beside(mask, q);
    for (int i = 0; ok && i < 4; ++i) ok = q.size(i) <= 1 << 29 && k.size(i) <= 1 << 29;
    if (ok && lengths.defined())
        ok = lengths.scalar_type() == at::kInt && lengths.dim() == 1 && lengths.size(0) == q.size(0) && lengths.is_contiguous();
    if (ok && mask.defined())
        ok = mask.scalar_type() == at::kBool && mask.dim() == 2 && mask.size(0) == q.size(0) && mask.size(1) == k.size(1) &&
             (mask.stride(1) == 1 || mask.size(1) == 1);
    TORCH_CHECK(ok, "cross_attention: q [B, Lq, Hq, D], k and v [B, Lk, Hk, D], int32 lengths [B], a bool mask [B, Lk], on one GPU");
}

long mask_stride(const Tensor& mask) { return mask.defined() ? mask.stride(0) : 0; }

Tensor attend(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Tensor& mask, double scale,
              Tensor* lse) {
    fits(q, k, v, lengths, mask);
    const c10::DeviceGuard guard(q.device());
    const Shape s(q, k);
    const Tensor o = at::empty(q.sizes(), q.options());
    if (lse) *lse = at::empty({s.B, s.Hk, (int64_t)s.Lq * s.share}, q.options().dtype(at::kFloat));
    const Tensor ws = workspace(dp.xa_workspace(s.B, s.Lq, s.Lk, s.Hk, s.share, s.D, 0), q);
    long strides[9], *at = strides;
    for (const Tensor* t : {&q, &k, &v}) add_strides(at, *t);
    check(dp.xa_fwd(in(q), in(k), in(v), out(o), lse ? out(*lse) : nullptr, in(lengths), in(mask), mask_stride(mask), out(ws),
                    strides, s.B, s.Lq, s.Lk, s.Hk, s.share, s.D, (float)scale, type_code(q), stream(q)), "xa_fwd");
    return o;
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& query, const Tensor& key, const Tensor& value,
                          const optional<Tensor>& lengths, const optional<Tensor>& mask, double scale) {
        const Tensor q = heads(query), k = heads(key), v = heads(value), n = some(lengths), m = some(mask);
        Tensor lse;
        const Tensor o = attend(q, k, v, n, m, scale, &lse);
        ctx->save_for_backward({q, k, v, o, lse, n, m});
        ctx->saved_data["scale"] = scale;
        return o;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_order("cross_attention");
        const auto saved = ctx->get_saved_variables();
        const Tensor q = heads(saved[0]), k = heads(saved[1]), v = heads(saved[2]), o = heads(saved[3].contiguous()),
                     lse = saved[4].contiguous(), &n = saved[5];
        const Tensor m = saved[6].defined() && saved[6].stride(-1) != 1 ? saved[6].contiguous() : saved[6];
        fits(q, k, v, n, m);
        TORCH_CHECK(like(o, q) && like(grads[0], q) && beside(lse, q), "cross_attention: saved tensors and gradient belong on q's GPU");
        const c10::DeviceGuard guard(q.device());
        const Shape s(q, k);
        const Tensor d = heads(grads[0]);
        const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
                     dv = at::empty(v.sizes(), v.options()), delta = at::empty_like(lse);
        const Tensor ws = workspace(dp.xa_workspace(s.B, s.Lq, s.Lk, s.Hk, s.share, s.D, 1), q);
        long strides[12], *at = strides;
        for (const Tensor* t : {&q, &k, &v, &d}) add_strides(at, *t);
        check(dp.xa_bwd(in(q), in(k), in(v), in(o), in(d), in(lse), out(delta), out(dq), out(dk), out(dv), in(n), in(m),
                        mask_stride(m), out(ws), strides, s.B, s.Lq, s.Lk, s.Hk, s.share, s.D,
                        (float)ctx->saved_data["scale"].toDouble(), type_code(q), stream(q)), "xa_bwd");
        return {dq, dk, dv, Tensor(), Tensor(), Tensor()};
    }
};

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const optional<Tensor>& lengths,
                       const optional<Tensor>& mask, double scale) {
    no_tangent("cross_attention", {q, k, v});
    if (at::GradMode::is_enabled() && (wanted(q) || wanted(k) || wanted(v)))
        return CrossAttention::apply(q, k, v, lengths, mask, scale);
    return attend(heads(q), heads(k), heads(v), some(lengths), some(mask), scale, nullptr);
}

}  // namespace

TORCH_LIBRARY(dpamd, m) {
    m.def("bind(int[] addresses) -> ()", &bind);
    m.def("group_norm_act(Tensor x, Tensor? weight, Tensor? bias, Tensor? residual, int groups, float eps, int act) -> Tensor",
          &group_norm_act);
    m.def("dropout(Tensor x, Tensor? residual, int threshold, int seed, Tensor? device_seed, bool word) -> Tensor", &dropout);
    m.def("cross_attention(Tensor q, Tensor k, Tensor v, Tensor? lengths, Tensor? mask, float scale) -> Tensor",
          &cross_attention);
}
