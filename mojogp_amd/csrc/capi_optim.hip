// C ABI: the AdamW step (adamw.h).  Declarations are in include/mojogp_amd.h.
#include <algorithm>
#include <cmath>
#include <memory>
#include <mutex>
#include <unordered_map>

#include "adamw.h"
#include "mojogp_amd.h"

using namespace mgp;

namespace {

constexpr int64_t kMaxChunks = (int64_t)1 << 24;  // workgroups of 256 threads a launch

struct Span {
  const char* begin;
  const char* end;
  const char* name;
};

// A plan and the memory that its steps write, in order of addresses.
struct Handle {
  AdamPlan plan;
  std::vector<Span> written;
};

void add_span(std::vector<Span>& v, const void* p, size_t bytes, const char* name) {
  if (p && bytes) v.push_back({static_cast<const char*>(p), static_cast<const char*>(p) + bytes, name});
}

// What of the plan's written memory an array shares, or null.
const Span* shared(const Handle& h, const void* p, size_t bytes) {
  const char *b = static_cast<const char*>(p), *e = b + bytes;
  auto at = std::upper_bound(h.written.begin(), h.written.end(), b,
                             [](const char* x, const Span& s) { return x < s.end; });
  return bytes && at != h.written.end() && at->begin < e ? &*at : nullptr;
}

std::mutex g_lock;
std::unordered_map<void*, std::shared_ptr<Handle>>& handles() {
  static auto* m = new std::unordered_map<void*, std::shared_ptr<Handle>>;
  return *m;
}

std::shared_ptr<Handle> handle_of(void* p) {
  std::lock_guard<std::mutex> hold(g_lock);
  const auto at = handles().find(p);
  MGP_REQUIRE(at != handles().end(), "unknown or destroyed optimizer handle");
  return at->second;
}

AdamPlan plan_of(const mgp_adamw_t* a) {
  MGP_REQUIRE(a != nullptr, "null arguments");
  MGP_REQUIRE(valid_elem(a->type), "unknown element type");
  MGP_REQUIRE(a->bits == 32 || a->bits == 8, "the states have 32 or 8 bits");
  MGP_REQUIRE(!a->master_copies || a->type != ELEM_F32,
              "master copies are of bfloat16 and float16 parameters");
  MGP_REQUIRE(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0,
              "the decay rates of the means must be in [0, 1)");
  MGP_REQUIRE(a->eps >= 1e-30 && a->eps <= 1e30, "eps must be in [1e-30, 1e30]");
  MGP_REQUIRE(a->count >= 1 && a->count < ((int64_t)1 << 24), "count must be in [1, 2^24)");
  MGP_REQUIRE(a->tensors != nullptr, "null tensors");
  AdamPlan p;
  p.type = a->type;
  p.bits = a->bits;
  p.master_copies = a->master_copies != 0;
  p.beta1 = a->beta1;
  p.beta2 = a->beta2;
  p.eps = a->eps;
  p.seed = a->seed;
  p.exp_avg = a->exp_avg;
  p.exp_avg_sq = a->exp_avg_sq;
  p.exp_avg_scale = a->exp_avg_scale;
  p.exp_avg_sq_scale = a->exp_avg_sq_scale;
  p.master = a->master;
  p.table = a->table;
  int64_t chunks = 0;
  for (int64_t i = 0; i < a->count; ++i) {
    const mgp_adamw_tensor_t& t = a->tensors[i];
    MGP_REQUIRE(t.size >= 0 && t.size <= kMaxChunks * kAdamChunk, "a parameter is too large");
    MGP_REQUIRE(t.size == 0 || t.param != nullptr, "null parameter");
    MGP_REQUIRE(std::isfinite(t.weight_decay) && t.weight_decay >= 0.0f,
                "weight decay must be finite and >= 0");
    chunks += ceil_div(t.size, kAdamChunk);
    MGP_REQUIRE(chunks < kMaxChunks, "the parameters are too many values for one optimizer");
    p.tensors.push_back({t.param, t.size, t.weight_decay});
  }
  p.lay_out();
  return p;
}

AdamStep step_of(const AdamPlan& p, const mgp_adamw_step_t* a) {
  MGP_REQUIRE(a != nullptr, "null arguments");
  MGP_REQUIRE(a->grads != nullptr, "null gradients");
  MGP_REQUIRE(a->grad_type == p.type || a->grad_type == ELEM_F32,
              "the gradients must be of the parameters' type or float32");
  MGP_REQUIRE(std::isfinite(a->grad_scale) && a->grad_scale > 0.0,
              "the gradients' scale must be finite and > 0");
  MGP_REQUIRE(!a->form_norm || a->max_norm > 0.0, "max_norm must be > 0");
  MGP_REQUIRE(a->step_device != nullptr || (a->step >= 1 && a->step < ((int64_t)1 << 53)),
              "step must be in [1, 2^53)");
  MGP_REQUIRE(a->rate_device != nullptr || (std::isfinite(a->rate) && a->rate >= 0.0f),
              "the rate must be finite and >= 0");
  return {a->grads, a->grad_type,   a->grad_scale, a->form_norm != 0, a->max_norm,
          a->norm,  a->step,        a->step_device, a->rate,          a->rate_device};
}

}  // namespace

extern "C" {

int mgp_adamw_layout(const mgp_adamw_t* args, int64_t* values, int64_t* table_bytes) {
  return guarded([&] {
    const AdamPlan p = plan_of(args);
    MGP_REQUIRE(values != nullptr && table_bytes != nullptr, "null result");
    *values = p.values;
    *table_bytes = (int64_t)p.table_bytes();
  });
}

int mgp_adamw_create(const mgp_adamw_t* args, void* host_table, int64_t bytes, void** plan) {
  return guarded([&] {
    auto h = std::make_shared<Handle>();
    h->plan = plan_of(args);
    const AdamPlan& p = h->plan;
    MGP_REQUIRE(plan != nullptr && host_table != nullptr, "null result");
    MGP_REQUIRE(bytes >= (int64_t)p.table_bytes(), "the table is too small");
    MGP_REQUIRE(p.table != nullptr && (reinterpret_cast<uintptr_t>(p.table) & 15) == 0,
                "the table must be a 16-byte aligned device array");
    const size_t n = (size_t)p.values, scales = (size_t)(p.values / kAdamBlock) * sizeof(float);
    if (n > 0) {
      MGP_REQUIRE(p.exp_avg && p.exp_avg_sq, "null states");
      MGP_REQUIRE(aligned16(p.exp_avg) && aligned16(p.exp_avg_sq) && aligned16(p.master),
                  "the states must be 16-byte aligned");
      MGP_REQUIRE(p.bits == 32 || (p.exp_avg_scale && p.exp_avg_sq_scale), "null scales");
      MGP_REQUIRE(!p.master_copies || p.master, "null master copies");
    }
    std::vector<Span>& w = h->written;
    for (const AdamTensor& t : p.tensors)
      add_span(w, t.param, (size_t)t.size * elem_bytes(p.type), "a parameter");
    const size_t state = n * (p.bits == 8 ? 1 : sizeof(float));
    add_span(w, p.exp_avg, state, "the states");
    add_span(w, p.exp_avg_sq, state, "the states");
    if (p.bits == 8) {
      add_span(w, p.exp_avg_scale, scales, "the states");
      add_span(w, p.exp_avg_sq_scale, scales, "the states");
    }
    if (p.master_copies) add_span(w, p.master, n * sizeof(float), "the master copies");
    add_span(w, p.table, p.table_bytes(), "the table");
    std::sort(w.begin(), w.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    for (size_t i = 1; i < w.size(); ++i)
      MGP_REQUIRE(w[i - 1].end <= w[i].begin, std::string(w[i].name) + " shares memory with " +
                                                  (w[i - 1].name == w[i].name ? std::string("another")
                                                                              : w[i - 1].name));
    p.write_table(host_table);
    std::lock_guard<std::mutex> hold(g_lock);
    handles()[h.get()] = h;
    *plan = h.get();
  });
}

int mgp_adamw_destroy(void* plan) {
  return guarded([&] {
    std::lock_guard<std::mutex> hold(g_lock);
    MGP_REQUIRE(handles().erase(plan) == 1, "unknown or destroyed optimizer handle");
  });
}

int mgp_adamw_workspace(void* plan, const mgp_adamw_step_t* args, int64_t* bytes) {
  return guarded([&] {
    MGP_REQUIRE(bytes != nullptr, "null result");
    const auto h = handle_of(plan);
    *bytes = (int64_t)adamw_bytes(h->plan, step_of(h->plan, args));
  });
}

int mgp_adamw_step_device(void* plan, const mgp_adamw_step_t* args, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  return guarded([&] {
    const auto h = handle_of(plan);
    const AdamPlan& p = h->plan;
    const AdamStep s = step_of(p, args);
    const size_t need = adamw_bytes(p, s), elem = elem_bytes(s.grad_type);
    MGP_REQUIRE(workspace_bytes >= 0 && (size_t)workspace_bytes >= need,
                "workspace of " + std::to_string(workspace_bytes) + " bytes, " +
                    std::to_string(need) + " are needed");
    MGP_REQUIRE(need == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0),
                "the workspace must be 256-byte aligned");
    auto apart = [&](const char* name, const void* q, size_t bytes) {
      const Span* w = q ? shared(*h, q, bytes) : nullptr;
      MGP_REQUIRE(w == nullptr, std::string(name) + " shares memory with " + w->name);
    };
    // what a step writes besides the plan's memory
    const Span results[2] = {{static_cast<const char*>(workspace),
                              static_cast<const char*>(workspace) + need, "the workspace"},
                             {reinterpret_cast<const char*>(s.norm_out),
                              reinterpret_cast<const char*>(s.norm_out) + sizeof(float), "norm"}};
    auto outside = [&](const char* name, const void* q, size_t bytes, int from, int to) {
      const char *b = static_cast<const char*>(q), *e = b + bytes;
      for (int k = from; k < to; ++k)
        MGP_REQUIRE(!q || !results[k].begin || e <= results[k].begin || results[k].end <= b,
                    std::string(name) + " shares memory with " + results[k].name);
    };
    for (size_t i = 0; i < p.tensors.size(); ++i) {
      const size_t bytes = (size_t)p.tensors[i].size * elem;
      apart("a gradient", s.grads[i], bytes);
      if (bytes) outside("a gradient", s.grads[i], bytes, 0, 2);
    }
    outside("norm", s.norm_out, sizeof(float), 0, 1);
    outside("step", s.step_device, sizeof(int64_t), 0, 2);
    outside("rate", s.rate_device, sizeof(float), 0, 2);
    apart("norm", s.norm_out, sizeof(float));
    apart("step", s.step_device, sizeof(int64_t));
    apart("rate", s.rate_device, sizeof(float));
    apart("the workspace", workspace, need);
    adamw_step(p, s, workspace, static_cast<hipStream_t>(stream));
  });
}

int mgp_adamw_values_device(void* plan, float* exp_avg, float* exp_avg_sq, void* stream) {
  return guarded([&] {
    const auto h = handle_of(plan);
    MGP_REQUIRE(h->plan.bits == 8, "32-bit states are values themselves");
    MGP_REQUIRE(h->plan.values == 0 || (exp_avg && exp_avg_sq), "null result");
    const size_t bytes = (size_t)h->plan.values * sizeof(float);
    for (const float* q : {exp_avg, exp_avg_sq}) {
      const Span* w = shared(*h, q, bytes);
      MGP_REQUIRE(w == nullptr, std::string("a result shares memory with ") + w->name);
    }
    MGP_REQUIRE(bytes == 0 || exp_avg + h->plan.values <= exp_avg_sq ||
                    exp_avg_sq + h->plan.values <= exp_avg,
                "the results share memory");
    adamw_values(h->plan, exp_avg, exp_avg_sq, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
