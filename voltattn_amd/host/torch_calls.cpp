// torch_calls.cpp — the plain calls of torch.ops.voltattn.append_rope and attend_paged, from the
// dispatcher to the C ABI without Python: what such a call does on the host is most of a small
// call's time. A call that is not plain (wrong shapes, types or devices, inputs that require grad,
// an error of the library) goes on to the op of the same name with _checked, which
// voltattn_amd/torch_ops.py registers and which does the whole of it, errors included.
//
// Compiled against PyTorch's headers; the C ABI's functions come by address (_bind), from the
// library that the package has loaded.
#include "voltattn.h"

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>
#include <torch/version.h>

#include <optional>
#include <tuple>

// What the package looks for before it loads this library: it goes with one PyTorch.
extern "C" __attribute__((used, visibility("default"))) const char va_torch_calls_for[] =
    "voltattn calls for PyTorch " C10_STRINGIZE(TORCH_VERSION_MAJOR) "." C10_STRINGIZE(TORCH_VERSION_MINOR) "." C10_STRINGIZE(TORCH_VERSION_PATCH);

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

decltype(&va_append_rope)     p_append_rope = nullptr;
decltype(&va_attend_paged)    p_attend_paged = nullptr;
decltype(&va_attend_ws_bytes) p_attend_ws_bytes = nullptr;

void bind(at::IntArrayRef f) {
    TORCH_CHECK(f.size() == 3, "three functions");
    p_append_rope = reinterpret_cast<decltype(p_append_rope)>(f[0]);
    p_attend_paged = reinterpret_cast<decltype(p_attend_paged)>(f[1]);
    p_attend_ws_bytes = reinterpret_cast<decltype(p_attend_ws_bytes)>(f[2]);
}

// A dense tensor on GPU `dev` with this type and shape.
bool is(const Tensor& t, int dev, at::ScalarType type, at::IntArrayRef shape, bool dense = true) {
    return t.is_cuda() && t.get_device() == dev && t.scalar_type() == type && t.sizes() == shape && (!dense || t.is_contiguous());
}
bool is(const OptTensor& t, int dev, at::ScalarType type, at::IntArrayRef shape) { return t.has_value() && is(*t, dev, type, shape); }

// The row and head strides of t [T, H, D], of which the last dimension is dense; those of a dimension of
// one are never stepped: any that the library takes.
bool strides(const Tensor& t, int64_t* row, int64_t* head) {
    if (t.stride(2) != 1) return false;
    *row = t.size(0) <= 1 ? t.size(2) : t.stride(0);
    *head = t.size(1) == 1 ? 0 : t.stride(1);
    return true;
}

const void* ptr(const OptTensor& t) { return t.has_value() ? t->const_data_ptr() : nullptr; }
template <class T> T* as(const void* p) { return static_cast<T*>(const_cast<void*>(p)); }

// The format of that name and the bits of a value (0: b8+, whose scales lie otherwise).
int format(std::string_view name, int* bits) {
    static const struct { const char* name; va_fmt fmt; int bits; } FORMATS[] = {
        {"b8+", VA_B8P, 0},  {"f16+", VA_F16P, 16}, {"q8+", VA_Q8P, 8}, {"q4+", VA_Q4P, 4},
        {"q3+", VA_Q3P, 3},  {"f16", VA_F16, 16},   {"q8", VA_Q8, 8},   {"q4", VA_Q4, 4}};
    for (const auto& f : FORMATS)
        if (name == f.name) return *bits = f.bits, (int)f.fmt;
    return -1;
}

// torch counts changes in place, so that backward() does not take them for what was saved.
void changed(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

using Rope = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const Tensor&, const OptTensor&,
                                        const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, std::string_view, int64_t,
                                        bool, bool, double);
using Attend = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const Tensor&,
                      std::string_view, c10::SymInt, int64_t);

template <class F> c10::TypedOperatorHandle<F> find(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

std::tuple<Tensor, Tensor> append_rope_checked(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& freq, const OptTensor& cu,
                                               const Tensor& start, const OptTensor& positions, const Tensor& table, const Tensor& kp, const Tensor& vp,
                                               const OptTensor& ks, const OptTensor& vs, std::string_view fmt, int64_t group, bool interleaved,
                                               bool rotated_k, double scaling) {
    static const auto op = find<Rope>("voltattn::append_rope_checked");
    return op.call(q, k, v, freq, cu, start, positions, table, kp, vp, ks, vs, fmt, group, interleaved, rotated_k, scaling);
}

std::tuple<Tensor, Tensor> append_rope(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& freq, const OptTensor& cu, const Tensor& start,
                                       const OptTensor& positions, const Tensor& table, const Tensor& kp, const Tensor& vp, const OptTensor& ks,
                                       const OptTensor& vs, std::string_view fmt, int64_t group, bool interleaved, bool rotated_k, double scaling) {
    int bits = 0;
    const int f = format(fmt, &bits);
    const int dev = q.is_cuda() ? (int)q.get_device() : -1;
    auto plain = [&](va_rope_shape& s) {
        if (f < 0 || dev < 0 || dev != c10::hip::current_device() || q.dim() != 3 || k.dim() != 3 || v.dim() != 3 || start.dim() != 1 || table.dim() != 2 ||
            freq.dim() != 1 || kp.dim() != 4 || (group != 32 && group != 64))
            return false;
        const int64_t T = q.size(0), H = q.size(1), D = q.size(2), Hk = k.size(1), B = start.size(0), half = freq.size(0);
        const int64_t pages = kp.size(0), rows = kp.size(2);
        if ((D != 64 && D != 128) || T < 1 || H < 1 || Hk < 1 || B < 1 || half < 8 || half % 8 || 2 * half > D) return false;
        if (!is(q, dev, at::kHalf, {T, H, D}, false) || !is(k, dev, at::kHalf, {T, Hk, D}, false) || !is(v, dev, at::kHalf, {T, Hk, D}, false) ||
            !is(freq, dev, at::kFloat, {half}) || !is(start, dev, at::kInt, {B}) || !is(table, dev, at::kInt, {B, table.size(1)}))
            return false;
        if (cu.has_value() ? !is(cu, dev, at::kInt, {B + 1}) : T != B) return false;
        if (positions.has_value() && !is(positions, dev, at::kInt, {T})) return false;
        const auto type = bits == 0 ? at::kFloat8_e4m3fn : bits == 16 ? at::kHalf : at::kByte;
        const int64_t row = bits == 0 || bits == 16 ? D : D * bits / 8;
        if (!is(kp, dev, type, {pages, Hk, rows, row}) || !is(vp, dev, type, {pages, Hk, rows, row})) return false;
        if (bits == 0) {
            if (rows % group || !is(ks, dev, at::kHalf, {pages, Hk, rows / group}) || !is(vs, dev, at::kHalf, {pages, Hk, rows / group})) return false;
        } else if (bits != 16) {
            if (group > D || !is(ks, dev, at::kHalf, {pages, Hk, rows, D / group}) || !is(vs, dev, at::kHalf, {pages, Hk, rows, D / group})) return false;
        }
        if (std::max({T, H, Hk, B, rows, pages, table.size(1)}) > INT32_MAX) return false;
        s = va_rope_shape{(int)B, (int)T, (int)H, (int)Hk, (int)D, (int)group, (int)rows, (int)table.size(1), (int)pages, (int)(2 * half), interleaved,
                          (float)scaling, 0, 0, 0, 0, 0, 0};
        return strides(q, &s.q_row, &s.q_head) && strides(k, &s.k_row, &s.k_head) && strides(v, &s.v_row, &s.v_head);
    };
    va_rope_shape s;
    if (!plain(s)) return append_rope_checked(q, k, v, freq, cu, start, positions, table, kp, vp, ks, vs, fmt, group, interleaved, rotated_k, scaling);
    Tensor q_out = at::empty({s.total, s.Hq, s.D}, q.options()), k_out = at::empty({rotated_k ? s.total : 0, s.Hkv, s.D}, q.options());
    va_rope_bufs b{as<uint16_t>(q.const_data_ptr()), as<uint16_t>(k.const_data_ptr()), as<uint16_t>(v.const_data_ptr()), as<int32_t>(ptr(cu)),
                   as<int32_t>(start.const_data_ptr()), as<int32_t>(ptr(positions)), as<int32_t>(table.const_data_ptr()), as<float>(freq.const_data_ptr()),
                   as<uint16_t>(q_out.mutable_data_ptr()), rotated_k ? as<uint16_t>(k_out.mutable_data_ptr()) : nullptr, kp.mutable_data_ptr(),
                   vp.mutable_data_ptr(), bits == 16 ? nullptr : as<uint16_t>(ks->mutable_data_ptr()), bits == 16 ? nullptr : as<uint16_t>(vs->mutable_data_ptr())};
    if (p_append_rope((va_fmt)f, &b, &s, c10::hip::getCurrentHIPStream(dev).stream()) != VA_OK)
        return append_rope_checked(q, k, v, freq, cu, start, positions, table, kp, vp, ks, vs, fmt, group, interleaved, rotated_k, scaling);
    changed(kp);
    changed(vp);
    if (ks.has_value()) changed(*ks);
    if (vs.has_value()) changed(*vs);
    return {q_out, k_out};
}

Tensor attend_paged_checked(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs, const Tensor& table, const OptTensor& cu,
                            const Tensor& lens, std::string_view fmt, c10::SymInt cap, int64_t group) {
    static const auto op = find<Attend>("voltattn::attend_paged_checked");
    return op.call(q, kp, vp, ks, vs, table, cu, lens, fmt, std::move(cap), group);
}

Tensor attend_paged(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs, const Tensor& table, const OptTensor& cu,
                    const Tensor& lens, std::string_view fmt, c10::SymInt cap, int64_t group) {
    const int dev = q.is_cuda() ? (int)q.get_device() : -1;
    auto plain = [&](va_paged_shape& s) {
        if (fmt != "b8+" || dev < 0 || dev != c10::hip::current_device() || q.dim() != 3 || table.dim() != 2 || kp.dim() != 4 || (group != 32 && group != 64) ||
            cap.is_symbolic())
            return false;
        const int64_t T = q.size(0), H = q.size(1), D = q.size(2), B = table.size(0), pages = kp.size(0), Hk = kp.size(1), rows = kp.size(2);
        const int64_t most = cap.as_int_unchecked();
        if ((D != 64 && D != 128) || T < 1 || H < 1 || Hk < 1 || H % Hk || rows % group || std::max({T, H, Hk, B, rows, pages, table.size(1), most}) > INT32_MAX ||
            most < 0)
            return false;
        if (!is(q, dev, at::kHalf, {T, H, D}) || !is(table, dev, at::kInt, {B, table.size(1)}) || !is(lens, dev, at::kInt, {B}) ||
            !is(kp, dev, at::kFloat8_e4m3fn, {pages, Hk, rows, D}) || !is(vp, dev, at::kFloat8_e4m3fn, {pages, Hk, rows, D}) ||
            !is(ks, dev, at::kHalf, {pages, Hk, rows / group}) || !is(vs, dev, at::kHalf, {pages, Hk, rows / group}))
            return false;
        if (cu.has_value() ? !is(cu, dev, at::kInt, {B + 1}) : T != B) return false;
        s = va_paged_shape{(int)B, (int)H, (int)Hk, (int)D, (int)group, (int)rows, (int)table.size(1), (int)pages, (int)most};
        return true;
    };
    va_paged_shape s;
    size_t bytes = 0;
    if (!plain(s) || (bytes = p_attend_ws_bytes(VA_B8P, &s, (int)q.size(0))) == 0)
        return attend_paged_checked(q, kp, vp, ks, vs, table, cu, lens, fmt, std::move(cap), group);
    Tensor out = at::empty(q.sizes(), q.options()), ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    va_attend_bufs b{kp.const_data_ptr(), vp.const_data_ptr(), as<uint16_t>(ks.const_data_ptr()), as<uint16_t>(vs.const_data_ptr()),
                     as<int32_t>(table.const_data_ptr()), as<int32_t>(ptr(cu)), as<int32_t>(lens.const_data_ptr()), as<uint16_t>(q.const_data_ptr()),
                     as<uint16_t>(out.mutable_data_ptr()), as<float>(ws.mutable_data_ptr())};
    if (p_attend_paged(VA_B8P, &b, &s, (int)q.size(0), c10::hip::getCurrentHIPStream(dev).stream()) != VA_OK)
        return attend_paged_checked(q, kp, vp, ks, vs, table, cu, lens, fmt, std::move(cap), group);
    return out;
}

// Above the ops: inputs that require grad take the checked op, whose output's backward() raises, as do those with
// a tangent (forward mode, which no_grad() leaves on), for which it raises itself.
bool requires_grad(std::initializer_list<const Tensor*> ts) {
    const bool backward = at::GradMode::is_enabled();
    for (const Tensor* t : ts) {
        if (!t || !t->unsafeGetTensorImpl()->autograd_meta()) continue;   // neither, as most are
        if ((backward && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined()) return true;
    }
    return false;
}
const Tensor* of(const OptTensor& t) { return t.has_value() ? &*t : nullptr; }

std::tuple<Tensor, Tensor> append_rope_autograd(c10::DispatchKeySet keys, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& freq,
                                                const OptTensor& cu, const Tensor& start, const OptTensor& positions, const Tensor& table, const Tensor& kp,
                                                const Tensor& vp, const OptTensor& ks, const OptTensor& vs, std::string_view fmt, int64_t group,
                                                bool interleaved, bool rotated_k, double scaling) {
    if (requires_grad({&q, &k, &v, &freq, &kp, &vp, of(ks), of(vs)}))
        return append_rope_checked(q, k, v, freq, cu, start, positions, table, kp, vp, ks, vs, fmt, group, interleaved, rotated_k, scaling);
    static const auto op = find<Rope>("voltattn::append_rope");
    at::AutoDispatchBelowAutograd below;
    return op.redispatch(keys & c10::after_autograd_keyset, q, k, v, freq, cu, start, positions, table, kp, vp, ks, vs, fmt, group, interleaved, rotated_k,
                         scaling);
}
Tensor attend_paged_autograd(c10::DispatchKeySet keys, const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs,
                             const Tensor& table, const OptTensor& cu, const Tensor& lens, std::string_view fmt, c10::SymInt cap, int64_t group) {
    if (requires_grad({&q, &kp, &vp, &ks, &vs})) return attend_paged_checked(q, kp, vp, ks, vs, table, cu, lens, fmt, std::move(cap), group);
    static const auto op = find<Attend>("voltattn::attend_paged");
    at::AutoDispatchBelowAutograd below;
    return op.redispatch(keys & c10::after_autograd_keyset, q, kp, vp, ks, vs, table, cu, lens, fmt, std::move(cap), group);
}

} // namespace

TORCH_LIBRARY_FRAGMENT(voltattn, m) {
    m.def("_bind(int[] functions) -> ()", &bind);
}
// For tensors on a GPU; every other key has what Python registers.
TORCH_LIBRARY_IMPL(voltattn, CUDA, m) {
    m.impl("append_rope", &append_rope);
    m.impl("attend_paged", &attend_paged);
}
TORCH_LIBRARY_IMPL(voltattn, AutogradCUDA, m) {
    m.impl("append_rope", &append_rope_autograd);
    m.impl("attend_paged", &attend_paged_autograd);
}
