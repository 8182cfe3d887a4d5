// The generation operators' calls as torch sees them: argument checks, output
// and workspace tensors and the current stream, then one call of the C ABI.
//
// A decode step makes several small calls a layer, each a few microseconds on
// the GPU; through ctypes and Python-level checks one costs 12 to 16 us of host
// time, here 4 to 7. The library's entry points are bound by address (bind), so
// this module follows whichever libquailb200 is loaded.
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>

#include <map>
#include <mutex>
#include <string>
#include <tuple>

#include "../../include/quail_b200.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using Optional = std::optional<Tensor>;

struct Entries {
    decltype(&qb_kv_quant_write) kv_quant_write;
    decltype(&qb_kv_quant_read) kv_quant_read;
    decltype(&qb_decode_attention_workspace) decode_attention_workspace;
    decltype(&qb_decode_attention) decode_attention;
    decltype(&qb_beam_select_workspace) beam_select_workspace;
    decltype(&qb_beam_select) beam_select;
    decltype(&qb_beam_reorder) beam_reorder;
} lib;

void bind(const py::dict& addresses) {
    auto set = [&](const char* name, auto& entry) {
        entry = reinterpret_cast<std::decay_t<decltype(entry)>>(
            addresses[name].cast<uintptr_t>());
    };
    set("qb_kv_quant_write", lib.kv_quant_write);
    set("qb_kv_quant_read", lib.kv_quant_read);
    set("qb_decode_attention_workspace", lib.decode_attention_workspace);
    set("qb_decode_attention", lib.decode_attention);
    set("qb_beam_select_workspace", lib.beam_select_workspace);
    set("qb_beam_select", lib.beam_select);
    set("qb_beam_reorder", lib.beam_reorder);
}

// A status as the binding's own check raises it.
void check(int status, const char* name) {
    if (status != QB_OK) py::module_::import("quail_b200._native").attr("check")(status, name);
}

void need(bool ok, const char* who, const char* what) {
    if (!ok) throw py::value_error(std::string(who) + ": " + what);
}

void* ptr(const Optional& t) { return t ? t->data_ptr() : nullptr; }
template <typename T>
T* ptr_as(const Tensor& t) {
    return static_cast<T*>(t.data_ptr());
}
template <typename T>
T* ptr_as(const Optional& t) {
    return static_cast<T*>(ptr(t));
}

// Every tensor on the first one's CUDA device.
c10::Device device_of(const char* who, std::initializer_list<const Tensor*> tensors) {
    const c10::Device device = (*tensors.begin())->device();
    need(device.is_cuda(), who, "CUDA tensors are needed");
    for (const Tensor* t : tensors)
        need(t == nullptr || t->device() == device, who, "tensors on different devices");
    return device;
}
const Tensor* maybe(const Optional& t) { return t ? &*t : nullptr; }

void* stream_of(c10::Device device) {
    return c10::cuda::getCurrentCUDAStream(device.index()).stream();
}

bool is_vector(const Tensor& t, at::ScalarType type, int64_t n) {
    return t.dim() == 1 && t.size(0) == n && t.scalar_type() == type && t.is_contiguous();
}

// bf16 rows of heads [rows, n, d], each row's heads contiguous.
struct Heads {
    int64_t rows, n, d, ld;
    Heads(const char* who, const char* name, const Tensor& x) {
        if (x.dim() != 3 || x.scalar_type() != at::kBFloat16)
            need(false, who, (std::string(name) + " must be bf16 [rows, n, d]").c_str());
        rows = x.size(0);
        n = x.size(1);
        d = x.size(2);
        if (x.stride(2) != 1 || (n > 1 && x.stride(1) != d))
            need(false, who,
                 ("the heads of a row of " + std::string(name) + " must be contiguous").c_str());
        // a single row's stride may be anything; the library wants one that
        // covers it
        ld = rows > 1 ? x.stride(0) : (n * d + 7) / 8 * 8;
    }
};

struct Cache {   // an 8-bit layer
    int64_t rows, n_kv, d;
    Cache(const char* who, const Tensor& k, const Tensor& v, const Tensor& ks,
          const Tensor& vs) {
        const bool ok =
            k.dim() == 3 && v.sizes() == k.sizes() && ks.dim() == 2 &&
            ks.size(0) == k.size(0) && ks.size(1) == k.size(1) && vs.sizes() == ks.sizes() &&
            k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn &&
            ks.scalar_type() == at::kByte && vs.scalar_type() == at::kByte &&
            k.is_contiguous() && v.is_contiguous() && ks.is_contiguous() && vs.is_contiguous();
        need(ok, who,
             "the cache needs contiguous e4m3 codes [rows, n_kv, d] and uint8 scales "
             "[rows, n_kv]");
        rows = k.size(0);
        n_kv = k.size(1);
        d = k.size(2);
    }
};

int64_t rows_like(const char* who, const Heads& k, const Heads& v, const Cache& cache) {
    need(k.n == cache.n_kv && v.n == cache.n_kv && k.d == cache.d && v.d == cache.d, who,
         "the heads of k and v are not the cache's");
    need(k.rows == v.rows, who, "k and v differ in rows");
    return k.rows;
}

void kv_quant_write(const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc,
                    const Tensor& ks, const Tensor& vs, const Tensor& dst, const Optional& src) {
    const char* who = "kv_quant_write";
    const Cache cache(who, kc, vc, ks, vs);
    const Heads hk(who, "k", k), hv(who, "v", v);
    const int64_t rows = rows_like(who, hk, hv, cache);
    const int64_t n = src && src->dim() == 1 ? src->size(0) : rows;
    need(!src || is_vector(*src, at::kLong, n), who,
         "src must be a contiguous int64 vector as long as the rows");
    need(is_vector(dst, at::kLong, n), who,
         "dst must be a contiguous int64 vector as long as the rows");
    const c10::Device device = device_of(who, {&k, &v, &kc, &vc, &ks, &vs, &dst, maybe(src)});
    const c10::DeviceGuard guard(device);
    check(lib.kv_quant_write(k.data_ptr(), v.data_ptr(), hk.ld, hv.ld, ptr_as<int64_t>(src),
                             ptr_as<int64_t>(dst), n, rows, (int)cache.n_kv, (int)cache.d,
                             kc.data_ptr(), vc.data_ptr(), ptr_as<uint8_t>(ks),
                             ptr_as<uint8_t>(vs), cache.rows, stream_of(device)),
          "qb_kv_quant_write");
}

std::tuple<Tensor, Tensor> kv_quant_read(const Tensor& kc, const Tensor& vc, const Tensor& ks,
                                         const Tensor& vs, const Tensor& src,
                                         const Optional& dst, const Optional& out_k,
                                         const Optional& out_v) {
    const char* who = "kv_quant_read";
    const Cache cache(who, kc, vc, ks, vs);
    need(src.dim() == 1 && is_vector(src, at::kLong, src.size(0)), who,
         "src must be a contiguous int64 vector as long as the rows");
    const int64_t n = src.size(0);
    need(out_k || !dst, who, "dst needs out");
    need(out_k.has_value() == out_v.has_value(), who, "out is a pair of tensors");
    Tensor k, v;
    if (out_k) {
        k = *out_k;
        v = *out_v;
    } else {
        need(kc.is_cuda(), who, "CUDA tensors are needed");
        k = at::empty({n, cache.n_kv, cache.d}, kc.options().dtype(at::kBFloat16));
        v = at::empty_like(k);
    }
    const Heads hk(who, "k", k), hv(who, "v", v);
    const int64_t rows = rows_like(who, hk, hv, cache);
    need(!dst || is_vector(*dst, at::kLong, n), who,
         "dst must be a contiguous int64 vector as long as the rows");
    const c10::Device device =
        device_of(who, {&kc, &vc, &ks, &vs, &k, &v, &src, maybe(dst)});
    const c10::DeviceGuard guard(device);
    check(lib.kv_quant_read(kc.data_ptr(), vc.data_ptr(), ptr_as<uint8_t>(ks),
                            ptr_as<uint8_t>(vs), cache.rows, ptr_as<int64_t>(src),
                            ptr_as<int64_t>(dst), n, (int)cache.n_kv, (int)cache.d,
                            k.data_ptr(), v.data_ptr(), hk.ld, hv.ld, rows, stream_of(device)),
          "qb_kv_quant_read");
    return {k, v};
}

// The current stream's own zeroed workspace of `bytes` or more, kept: each call
// leaves its counters zero. A graph that is being captured must not share it
// (the graph may be replayed beside the stream), so there a call gets a fresh
// one, whose zeroing the graph repeats; workspace= spares that.
Tensor stream_workspace(int use, c10::Device device, int64_t bytes) {
    static std::mutex mutex;
    static auto* held = new std::map<std::tuple<int, int, void*>, Tensor>;   // outlives the GPU
    const auto options = at::TensorOptions().dtype(at::kByte).device(device);
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
        return at::zeros({bytes}, options);
    const std::lock_guard<std::mutex> lock(mutex);
    Tensor& t = (*held)[{use, (int)device.index(), stream_of(device)}];
    if (!t.defined() || t.size(0) < bytes) t = at::zeros({bytes}, options);
    return t;
}

Tensor workspace_for(const char* who, const Optional& given, int use, c10::Device device,
                     int64_t bytes) {
    if (!given) return stream_workspace(use, device, bytes);
    need(given->scalar_type() == at::kByte && given->is_contiguous(), who,
         "workspace must be contiguous uint8");
    return *given;
}

int64_t decode_bytes() {
    int64_t bytes = 0;
    check(lib.decode_attention_workspace(&bytes), "qb_decode_attention_workspace");
    return bytes;
}

int64_t select_bytes(int64_t groups, int64_t beams, int64_t vocab, int64_t n_out) {
    int64_t bytes = 0;
    check(lib.beam_select_workspace(groups, (int)beams, vocab, (int)n_out, &bytes),
          "qb_beam_select_workspace");
    return bytes;
}

Tensor decode_workspace(c10::Device device) {
    const c10::DeviceGuard guard(device);
    return at::zeros({decode_bytes()}, at::TensorOptions().dtype(at::kByte).device(device));
}

Tensor beam_workspace(int64_t groups, int64_t beams, int64_t vocab, int64_t n_out,
                      c10::Device device) {
    need(beams >= 1 && beams <= 32 && n_out >= 1 && n_out <= 32, "beam_workspace",
         "1 to 32 beams and 1 to 32 outputs a group");
    return at::zeros({select_bytes(groups, beams, vocab, n_out)},
                     at::TensorOptions().dtype(at::kByte).device(device));
}

std::tuple<Optional, Optional> decode_attention(
    const Tensor& q, const Tensor& k, const Tensor& v, const Optional& ks, const Optional& vs,
    const Tensor& table, const Tensor& used, int64_t page_tokens, double softmax_scale,
    const Optional& given_out, bool with_lse, const Optional& q8, const Optional& q8_scale,
    int64_t q8_ld, bool ue8m0, const Optional& given_workspace) {
    const char* who = "decode_attention";
    const Heads hq(who, "q", q);
    const int64_t rows = hq.rows;
    int64_t pool_rows, n_kv, d;
    if (ks) {
        need(vs.has_value(), who, "the scales go together");
        const Cache cache(who, k, v, *ks, *vs);
        pool_rows = cache.rows;
        n_kv = cache.n_kv;
        d = cache.d;
    } else {
        need(k.dim() == 3 && v.sizes() == k.sizes() && k.scalar_type() == at::kBFloat16 &&
                 v.scalar_type() == at::kBFloat16 && k.is_contiguous() && v.is_contiguous(),
             who, "bf16 pools must be contiguous [rows, n_kv, d]");
        pool_rows = k.size(0);
        n_kv = k.size(1);
        d = k.size(2);
    }
    need(hq.d == d, who, "q's head size is not the cache's");
    need(page_tokens > 0 && page_tokens <= 1024 && pool_rows % page_tokens == 0, who,
         "the pools are not whole pages");
    need(table.dim() == 2 && table.size(0) == rows && table.scalar_type() == at::kInt &&
             table.stride(1) == 1,
         who, "table must be int32 [rows, pages]");
    need(is_vector(used, at::kInt, rows), who, "used must be int32 [rows]");
    if (q8)
        need(q8->dim() == 2 && q8->size(0) == rows && q8->size(1) == hq.n * d &&
                 q8->element_size() == 1 && q8->is_contiguous() && q8_scale &&
                 q8_scale->dim() == 2 && q8_scale->size(0) == hq.n &&
                 q8_scale->size(1) >= q8_ld && q8_scale->scalar_type() == at::kFloat &&
                 q8_scale->is_contiguous() && q8_scale->size(1) == q8_ld,
             who, "quantised must hold [rows, n_q * d] codes and [n_q, ld] scales");
    Optional out = given_out;
    int64_t out_ld = 0;
    if (out) {
        need(out->sizes() == q.sizes(), who, "out must have q's shape");
        out_ld = Heads(who, "out", *out).ld;
    }
    const c10::Device device =
        device_of(who, {&q, &k, &v, maybe(ks), maybe(vs), &table, &used, maybe(out), maybe(q8),
                        maybe(q8_scale), maybe(given_workspace)});
    const c10::DeviceGuard guard(device);
    if (!out && !q8) {
        out = at::empty({rows, hq.n, d}, q.options());
        out_ld = hq.n * d;
    }
    Optional lse;
    if (with_lse) lse = at::empty({rows, hq.n}, q.options().dtype(at::kFloat));
    const Tensor workspace = workspace_for(who, given_workspace, 0, device, decode_bytes());
    check(lib.decode_attention(
              q.data_ptr(), hq.ld, rows, (int)hq.n, (int)n_kv, (int)d, k.data_ptr(),
              v.data_ptr(), ptr_as<uint8_t>(ks), ptr_as<uint8_t>(vs), pool_rows / page_tokens,
              (int)page_tokens, ptr_as<int32_t>(table), table.size(1),
              rows > 1 ? table.stride(0) : table.size(1), ptr_as<int32_t>(used),
              (float)softmax_scale, workspace.data_ptr(), workspace.size(0), ptr(out), out_ld,
              ptr(q8), ptr_as<float>(q8_scale), q8_ld, ue8m0, ptr_as<float>(lse),
              stream_of(device)),
          "qb_decode_attention");
    return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> beam_select(const Tensor& logits, const Tensor& scores,
                                               const Optional& finished, int64_t pad,
                                               std::optional<int64_t> outputs,
                                               const Optional& given_workspace) {
    const char* who = "beam_select";
    need(scores.dim() == 2 && scores.scalar_type() == at::kFloat && scores.is_contiguous(), who,
         "scores must be contiguous f32 [groups, beams]");
    const int64_t groups = scores.size(0), beams = scores.size(1);
    const int64_t n_out = outputs.value_or(beams);
    need(beams >= 1 && beams <= 32 && n_out >= 1 && n_out <= 32, who,
         "1 to 32 beams and 1 to 32 outputs a group");
    const bool bf16 = logits.scalar_type() == at::kBFloat16;
    need(logits.dim() == 2 && logits.size(0) == groups * beams && logits.stride(1) == 1 &&
             (bf16 || logits.scalar_type() == at::kFloat),
         who, "logits must be f32 or bf16 [groups * beams, vocab]");
    need(!finished || (finished->sizes() == scores.sizes() && finished->is_contiguous() &&
                       (finished->scalar_type() == at::kBool ||
                        finished->scalar_type() == at::kByte)),
         who, "finished must be contiguous bool or uint8 [groups, beams]");
    const c10::Device device =
        device_of(who, {&logits, &scores, maybe(finished), maybe(given_workspace)});
    const c10::DeviceGuard guard(device);
    const int64_t vocab = logits.size(1);
    const Tensor workspace = workspace_for(who, given_workspace, 1, device,
                                           select_bytes(groups, beams, vocab, n_out));
    const Tensor score = at::empty({groups, n_out}, scores.options());
    const Tensor parent = at::empty({groups, n_out}, scores.options().dtype(at::kInt));
    const Tensor token = at::empty({groups, n_out}, scores.options().dtype(at::kLong));
    check(lib.beam_select(logits.data_ptr(), bf16,
                          groups * beams > 1 ? logits.stride(0) : vocab, groups, (int)beams,
                          vocab, ptr_as<float>(scores), ptr_as<uint8_t>(finished), pad,
                          (int)n_out, workspace.data_ptr(), workspace.size(0),
                          ptr_as<float>(score), ptr_as<int32_t>(parent), ptr_as<int64_t>(token),
                          stream_of(device)),
          "qb_beam_select");
    return {score, parent, token};
}

std::tuple<Tensor, Tensor> beam_reorder(const Tensor& pool, const Optional& second,
                                        const Tensor& parents, const Tensor& used,
                                        const Tensor& table, int64_t page_tokens) {
    const char* who = "beam_reorder";
    need(parents.dim() == 2 && parents.scalar_type() == at::kInt && parents.is_contiguous(), who,
         "parents must be contiguous int32 [groups, beams]");
    const int64_t groups = parents.size(0), beams = parents.size(1);
    need(is_vector(used, at::kInt, groups), who, "used must be int32 [groups]");
    need(table.dim() == 2 && table.size(0) == groups * beams &&
             table.scalar_type() == at::kInt && table.is_contiguous(),
         who, "table must be contiguous int32 [groups * beams, pages]");
    need(pool.dim() >= 4 && pool.is_contiguous() &&
             (!second || (second->dim() >= 4 && second->is_contiguous() &&
                          second->sizes().slice(0, 3) == pool.sizes().slice(0, 3))),
         who, "pools must be contiguous [n_layers, 2, rows, ...]");
    const int64_t rows = pool.size(2);
    need(page_tokens > 0 && page_tokens <= 1024 && rows % page_tokens == 0, who,
         "the pools are not whole pages");
    const c10::Device device =
        device_of(who, {&pool, maybe(second), &parents, &used, &table});
    const c10::DeviceGuard guard(device);
    const Tensor out = at::empty_like(table);
    const Tensor next_row = at::empty({groups * beams}, table.options().dtype(at::kLong));
    check(lib.beam_reorder(
              ptr_as<int32_t>(parents), ptr_as<int32_t>(used), groups, (int)beams,
              ptr_as<int32_t>(table), table.size(1), (int)page_tokens, rows / page_tokens,
              pool.data_ptr(), pool.size(0) * pool.size(1),
              pool.stride(2) * (int64_t)pool.element_size(), ptr(second),
              second ? second->stride(2) * (int64_t)second->element_size() : 0,
              ptr_as<int32_t>(out), ptr_as<int64_t>(next_row), stream_of(device)),
          "qb_beam_reorder");
    return {out, next_row};
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
    m.def("bind", &bind);
    m.def("kv_quant_write", &kv_quant_write);
    m.def("kv_quant_read", &kv_quant_read);
    m.def("decode_workspace", &decode_workspace);
    m.def("beam_workspace", &beam_workspace);
    m.def("decode_attention", &decode_attention);
    m.def("beam_select", &beam_select);
    m.def("beam_reorder", &beam_reorder);
}
