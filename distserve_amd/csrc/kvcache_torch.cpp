// kvcache_torch.cpp -- torch op shim of the cache operators.
//
// Registers kvcache_ops: the class StepPlan and the ops that take one.  Tensors are checked
// and reduced to pointers, sizes and strides; the current HIP stream of their device is handed to the
// C ABI.  A nonzero return code becomes a RuntimeError carrying kvm_last_error().
//
// The plan's words are copied to the device on the current stream, and nobody waits for them on the host: that stream is
// behind whatever the program has given it, a stream of its own for the copies often behind another one (small copies are
// kernels, on a hardware queue that several streams share).  Calls on other streams wait there for the copy's event.
// Only a call that is captured waits on the host, once, because the graph may run anywhere; and the graph keeps the words.
// The host looks at a word that the stream writes behind the copy: an event counts as captured while the stream it was recorded
// on captures, however long ago that was, and to ask for it breaks the capture.
#include "kvmove.h"

#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/custom_class.h>
#include <torch/library.h>

#include <hip/hip_runtime.h>

#include <algorithm>
#include <chrono>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <mutex>
#include <set>
#include <thread>
#include <vector>

namespace {

void check(int rc, const char *op)
{
    TORCH_CHECK(rc == KVM_OK, op, ": ", kvm_last_error(), " (kvmove error ", rc, ")");
}

int32_t type_code(at::ScalarType t)
{
    switch (t) {
    case at::kHalf: return KVM_F16;
    case at::kBFloat16: return KVM_BF16;
    case at::kFloat: return KVM_F32;
    default: TORCH_CHECK(false, "the cache operators work on float16, bfloat16 and float32, not ", t);
    }
}

// While another thread captures a graph, the calls that a plan's copy needs are allowed to this one (and while this thread
// does, those that tie the words to the graph).
struct BesideCaptures {
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    BesideCaptures() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
    ~BesideCaptures() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
};

// A word of pinned memory that a stream writes a number of its own to.  It goes from plan to plan once that has happened.  (Nothing
// here is ever destroyed: plans may be dropped after everything else.)
class Mark {
    struct Words {
        std::mutex mu;
        std::vector<uint32_t *> free;        // written, so nobody's
        std::vector<Mark> dropped;           // of plans that were gone before the stream came to it
        uint32_t last = 0;
    };
    static Words &words()
    {
        static Words *all = new Words;
        return *all;
    }
    uint32_t *at = nullptr, number = 0;

public:
    bool reached() const { return __atomic_load_n(at, __ATOMIC_ACQUIRE) == number; }

    // Behind what `stream` has now.
    bool set(hipStream_t stream)
    {
        Words &w = words();
        std::lock_guard<std::mutex> lock(w.mu);
        for (size_t i = 0; i < w.dropped.size();) {
            if (w.dropped[i].reached()) {
                w.free.push_back(w.dropped[i].at);
                w.dropped[i] = w.dropped.back();
                w.dropped.pop_back();
            } else {
                ++i;
            }
        }
        if (w.free.empty()) {
            constexpr int kWords = 64, kApart = 16;     // a cache line each
            uint32_t *more = nullptr;
            if (hipHostMalloc((void **)&more, kWords * kApart * sizeof(uint32_t), hipHostMallocPortable | hipHostMallocCoherent) != hipSuccess) return false;
            std::memset(more, 0, kWords * kApart * sizeof(uint32_t));
            for (int i = 0; i < kWords; ++i) w.free.push_back(more + i * kApart);
        }
        if (++w.last == 0) ++w.last;                    // not what fresh words hold
        if (hipStreamWriteValue32(stream, w.free.back(), w.last, 0) != hipSuccess) return false;
        at = w.free.back();
        number = w.last;
        w.free.pop_back();
        return true;
    }
    void drop()
    {
        if (!at) return;
        std::lock_guard<std::mutex> lock(words().mu);
        words().dropped.push_back(*this);
        at = nullptr;
    }
};

// Plans' words that a graph kept and has let go.  A graph tells that from wherever it is taken apart, where no call of the runtime
// is allowed: the memory goes back when the next plan is made or dropped.  (Never destroyed: graphs may outlive everything.)
struct LetGo {
    std::mutex mu;
    std::vector<at::Tensor *> words;
    static LetGo &list()
    {
        static LetGo *all = new LetGo;
        return *all;
    }
    static void by_graph(void *kept)
    {
        LetGo &all = list();
        std::lock_guard<std::mutex> lock(all.mu);
        all.words.push_back((at::Tensor *)kept);
    }
    static void give_back()
    {
        std::vector<at::Tensor *> gone;
        {
            std::lock_guard<std::mutex> lock(list().mu);
            gone.swap(list().words);
        }
        for (at::Tensor *t : gone) delete t;
    }
};

struct StepPlan : torch::CustomClassHolder {
    KvmStep step;
    at::Tensor words;
    c10::ScalarType dtype;
    std::mutex mu;
    std::set<hipStream_t> seen;   // streams the allocator has been told of, and made to wait for the words
    hipStream_t made_on = nullptr;
    hipEvent_t copied = nullptr;  // behind the copy on made_on, as the mark
    Mark mark;
    bool complete = false;        // the copy is known to have ended
    unsigned long long captured_by = 0;   // the last capture that keeps the words

    StepPlan(std::vector<int64_t> first_token, std::vector<int64_t> new_tokens, std::vector<int64_t> table,
             std::vector<int64_t> table_len, int64_t num_blocks, int64_t block_size, int64_t num_heads,
             int64_t num_kv_heads, int64_t head_dim, int64_t type, bool quantized, int64_t device)
        : dtype((c10::ScalarType)type)
    {
        TORCH_CHECK(first_token.size() == new_tokens.size(), "StepPlan: ", first_token.size(), " first tokens but ",
                    new_tokens.size(), " lengths");
        TORCH_CHECK(num_blocks == 0 || table_len.size() == new_tokens.size(), "StepPlan: ", table_len.size(),
                    " block tables for ", new_tokens.size(), " sequences");
        int64_t in_tables = 0, tokens = 0;
        for (int64_t n : table_len) {
            TORCH_CHECK(n >= 0 && n <= (int64_t)table.size(), "StepPlan: bad block table length ", n);
            in_tables += n;
        }
        for (int64_t n : new_tokens) {
            TORCH_CHECK(n >= 0 && n <= INT32_MAX, "StepPlan: a sequence brings ", n, " tokens");
            tokens += n;
        }
        TORCH_CHECK(num_blocks == 0 || in_tables == (int64_t)table.size(), "StepPlan: block tables of ", in_tables,
                    " blocks but ", table.size(), " entries");
        TORCH_CHECK(tokens <= INT32_MAX && num_heads >= 1 && num_heads <= (1 << 20) && num_kv_heads >= 1,
                    "StepPlan: ", tokens, " tokens of ", num_heads, " heads, ", num_kv_heads, " KV heads");
        TORCH_CHECK(tokens * num_heads <= ((int64_t)1 << 40), "StepPlan: too many rows");
        const int64_t most = kvm_plan_words((int64_t)new_tokens.size(), tokens, (int64_t)table.size(), num_heads, num_kv_heads);
        if (most < 0) check((int)most, "StepPlan");
        std::vector<int32_t> host((size_t)most);
        check(kvm_plan_step(first_token.data(), new_tokens.data(), (int64_t)new_tokens.size(), table.data(),
                            table_len.data(), num_blocks, block_size, num_heads, num_kv_heads, head_dim, type_code(dtype),
                            quantized ? KVM_CACHE_E4M3 : KVM_CACHE_PLAIN, host.data(), (int64_t)host.size(), &step),
              "StepPlan");
        if (device < 0) return;   // a plan to look at, without a GPU
        LetGo::give_back();
        const c10::hip::HIPGuard guard((c10::DeviceIndex)device);
        made_on = c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream();
        TORCH_CHECK(!captures(made_on), "StepPlan: make the plan before the graph capture that uses it");
        const BesideCaptures allowed;
        words = at::empty({std::max<int64_t>(step.words, 4)}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device));
        // (from pageable memory: it has been read when the call returns)
        bool ok = hipMemcpyAsync(words.data_ptr(), host.data(), (size_t)step.words * 4, hipMemcpyHostToDevice, made_on) == hipSuccess;
        ok = ok && hipEventCreateWithFlags(&copied, hipEventDisableTiming) == hipSuccess && hipEventRecord(copied, made_on) == hipSuccess;
        if (!ok || !mark.set(made_on)) {
            if (copied) (void)hipEventDestroy(copied);
            TORCH_CHECK(false, "StepPlan: copying the plan to the device failed");
        }
        step.device = device;    // the ops below check where their tensors are and how far they reach
    }

    ~StepPlan() override
    {
        mark.drop();
        if (copied) (void)hipEventDestroy(copied);
        if (words.defined()) LetGo::give_back();
    }

    static bool captures(hipStream_t stream)
    {
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        return hipStreamIsCapturing(stream, &status) != hipSuccess || status != hipStreamCaptureStatusNone;
    }

    // On the host, for what made_on was given before the copy.
    void wait_for_words(const char *op)
    {
        const auto start = std::chrono::steady_clock::now();
        while (!(complete = complete || mark.reached())) {
            std::this_thread::sleep_for(std::chrono::microseconds(20));
            TORCH_CHECK(std::chrono::steady_clock::now() - start < std::chrono::minutes(10), op, ": the plan's copy does not end");
        }
    }

    // A captured call: the graph may run at any time on any stream, so the words have to be there, and stay as long as the graph.
    void keep_for_graph(hipStream_t stream, const char *op)
    {
        wait_for_words(op);
        const BesideCaptures allowed;
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        unsigned long long id = 0;
        hipGraph_t graph = nullptr;
        TORCH_CHECK(hipStreamGetCaptureInfo_v2(stream, &status, &id, &graph, nullptr, nullptr) == hipSuccess && graph, op,
                    ": no graph to capture into");
        if (id == captured_by) return;
        hipUserObject_t object = nullptr;
        at::Tensor *kept = new at::Tensor(words);
        if (hipUserObjectCreate(&object, kept, LetGo::by_graph, 1, hipUserObjectNoDestructorSync) != hipSuccess) {
            delete kept;
            TORCH_CHECK(false, op, ": the graph cannot keep the plan");
        }
        if (hipGraphRetainUserObject(graph, object, 1, hipGraphUserObjectMove) != hipSuccess) {
            (void)hipUserObjectRelease(object, 1);
            TORCH_CHECK(false, op, ": the graph cannot keep the plan");
        }
        captured_by = id;
    }

    // The words for a call on `device`'s current stream, which comes after their copy; the allocator is told of the stream, so
    // that the words' memory is not handed out again before the stream's work is done.
    const int32_t *use(const at::Tensor &like, const char *op, void **stream)
    {
        TORCH_CHECK(words.defined(), op, ": the plan was made without a GPU");
        TORCH_CHECK(like.device() == words.device(), op, ": the plan is on ", words.device(), ", the tensors on ", like.device());
        const c10::DeviceIndex device = words.device().index();
        const c10::hip::HIPStream s = c10::hip::getCurrentHIPStream(device);
        *stream = (void *)s.stream();
        {
            std::lock_guard<std::mutex> lock(mu);
            complete = complete || mark.reached();
            if (captures(s.stream())) keep_for_graph(s.stream(), op);
            if (seen.count(s.stream()) == 0) {
                words.record_stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device).unwrap());
                if (!complete && s.stream() != made_on && hipStreamWaitEvent(s.stream(), copied, 0) != hipSuccess) {
                    (void)hipGetLastError();     // made_on captures in another thread: the event cannot be had now
                    wait_for_words(op);
                }
                seen.insert(s.stream());
            }
        }
        return words.data_ptr<int32_t>();
    }

    int64_t device_index() const { return words.defined() ? words.device().index() : -1; }
};

typedef c10::intrusive_ptr<StepPlan> Plan;

// Nothing that a call reads or writes may be part of a derivative, backward or forward: it would be dropped without a word.
void no_gradients(std::initializer_list<const at::Tensor *> tensors, const char *op)
{
    const bool backward = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const at::Tensor *t : tensors) {
        if (!t) continue;
        TORCH_CHECK(!(backward && t->requires_grad()), op, " has no gradient: call it under torch.no_grad()");
        TORCH_CHECK(!(forward && t->_fw_grad(0).defined()), op, " has no gradient: a tensor has a forward-mode tangent");
    }
}

// A written tensor's version goes up, as after torch's own operators that write in place: a backward pass that has kept
// what was there before is an error then instead of a wrong gradient.  (Tensors made in inference mode have no version.)
void written(std::initializer_list<const at::Tensor *> tensors)
{
    for (const at::Tensor *t : tensors)
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// Bytes from the tensor's first element to the end of its storage.
int64_t extent(const at::Tensor &t) { return (int64_t)t.storage().nbytes() - t.storage_offset() * (int64_t)t.element_size(); }

// [tokens (or more), heads, head_dim] of the plan's type, heads contiguous inside.
KvmRows rows(const Plan &plan, const at::Tensor &t, int64_t tokens, int64_t heads, const char *op, const char *name)
{
    const KvmStep &s = plan->step;
    TORCH_CHECK(t.is_cuda(), op, ": ", name, " must live on the GPU");
    TORCH_CHECK(t.device() == plan->words.device(), op, ": ", name, " is on ", t.device(), ", the plan on ", plan->words.device());
    TORCH_CHECK(t.scalar_type() == plan->dtype, op, ": ", name, " is ", t.scalar_type(), ", the plan is for ", plan->dtype);
    TORCH_CHECK(t.dim() == 3 && t.size(0) >= tokens && t.size(1) == heads && t.size(2) == s.head_dim, op, ": ", name,
                " must be [", tokens, " or more, ", heads, ", ", s.head_dim, "], got ", t.sizes());
    TORCH_CHECK(t.stride(2) == 1, op, ": ", name, " must be contiguous within a head, its last stride is ", t.stride(2));
    // a dimension of one has a stride that means nothing
    return KvmRows{t.data_ptr(), t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0, extent(t)};
}

KvmCache cache(const Plan &plan, int64_t layer, const at::Tensor &k, const at::Tensor &v, const char *op)
{
    const KvmStep &s = plan->step;
    for (const at::Tensor *t : {&k, &v}) {
        TORCH_CHECK(t->is_cuda(), op, ": the pools must live on the GPU");
        TORCH_CHECK(t->dim() == 5 && t->is_contiguous(), op,
                    ": a pool must be a contiguous [num_blocks, layers, kv_heads, block_size, head_dim]");
    }
    TORCH_CHECK(k.device() == plan->words.device(), op, ": the pools are on ", k.device(), ", the plan on ", plan->words.device());
    TORCH_CHECK(k.sizes() == v.sizes() && k.dtype() == v.dtype() && k.device() == v.device(), op,
                ": k_cache and v_cache must agree in shape, dtype and device");
    const bool coded = k.scalar_type() == at::kByte;
    TORCH_CHECK(coded || k.scalar_type() == plan->dtype, op, ": the pools are ", k.scalar_type(), ", the plan is for ", plan->dtype);
    TORCH_CHECK(k.size(4) == s.head_dim + (coded ? 1 : 0), op, ": the pools' last dimension is ", k.size(4), ", ",
                s.head_dim + (coded ? 1 : 0), " expected", coded ? " (head_dim codes and a scale)" : "");
    return KvmCache{k.data_ptr(), v.data_ptr(), k.size(0), k.size(1), layer, k.size(2), k.size(3), s.head_dim,
                    type_code(plan->dtype), coded ? KVM_CACHE_E4M3 : KVM_CACHE_PLAIN, std::min(extent(k), extent(v))};
}

void write_kv(const Plan &plan, int64_t layer, const at::Tensor &k, const at::Tensor &v, const at::Tensor &k_cache,
              const at::Tensor &v_cache)
{
    no_gradients({&k, &v, &k_cache, &v_cache}, "write_kv");
    void *stream;
    const int32_t *words = plan->use(k_cache, "write_kv", &stream);
    const KvmCache c = cache(plan, layer, k_cache, v_cache, "write_kv");
    const KvmStep &s = plan->step;
    const KvmRows kr = rows(plan, k, s.num_tokens, s.num_kv_heads, "write_kv", "k"),
                  vr = rows(plan, v, s.num_tokens, s.num_kv_heads, "write_kv", "v");
    check(kvm_write_kv(&s, words, &c, &kr, &vr, stream), "write_kv");
    written({&k_cache, &v_cache});
}

std::tuple<at::Tensor, at::Tensor> read_kv(const Plan &plan, int64_t layer, const at::Tensor &k_cache, const at::Tensor &v_cache)
{
    no_gradients({&k_cache, &v_cache}, "read_kv");
    void *stream;
    const int32_t *words = plan->use(k_cache, "read_kv", &stream);
    const KvmCache c = cache(plan, layer, k_cache, v_cache, "read_kv");
    const KvmStep &s = plan->step;
    const c10::hip::HIPGuard guard(k_cache.device().index());
    const auto options = k_cache.options().dtype(plan->dtype);
    at::Tensor k = at::empty({s.num_kv_tokens, s.num_kv_heads, s.head_dim}, options), v = at::empty_like(k);
    const KvmRows kr = rows(plan, k, s.num_kv_tokens, s.num_kv_heads, "read_kv", "k"),
                  vr = rows(plan, v, s.num_kv_tokens, s.num_kv_heads, "read_kv", "v");
    check(kvm_read_kv(&s, words, &c, &kr, &vr, stream), "read_kv");
    return {k, v};
}

// The output, and zeros in its rows behind the last sequence's when it is a new one.
at::Tensor output(const Plan &plan, const at::Tensor &q, const std::optional<at::Tensor> &out, const char *op)
{
    if (out.has_value()) {
        TORCH_CHECK(out->sizes() == q.sizes(), op, ": out is ", out->sizes(), ", q is ", q.sizes());
        return *out;
    }
    at::Tensor made = at::empty(q.sizes(), q.options());
    if (q.size(0) > plan->step.num_tokens) made.narrow(0, plan->step.num_tokens, q.size(0) - plan->step.num_tokens).zero_();
    return made;
}

at::Tensor workspace(const Plan &plan, const at::Tensor &q)
{
    if (plan->step.part_rows == 0) return at::Tensor();
    // from the allocator for each call: a captured graph gets memory of its own
    return at::empty({kvm_attention_workspace(&plan->step)}, q.options().dtype(at::kByte));
}

float scale_of(const Plan &plan, std::optional<double> scale)
{
    return scale.has_value() ? (float)*scale : (float)(1.0 / std::sqrt((double)plan->step.head_dim));
}

at::Tensor paged_attention(const Plan &plan, int64_t layer, const at::Tensor &q, const at::Tensor &k_cache,
                           const at::Tensor &v_cache, std::optional<double> scale, const std::optional<at::Tensor> &out)
{
    const char *op = "paged_attention";
    no_gradients({&q, &k_cache, &v_cache, out.has_value() ? &*out : nullptr}, op);
    void *stream;
    const int32_t *words = plan->use(k_cache, op, &stream);
    const KvmCache c = cache(plan, layer, k_cache, v_cache, op);
    const KvmStep &s = plan->step;
    const KvmRows qr = rows(plan, q, s.num_tokens, s.num_heads, op, "q");
    const c10::hip::HIPGuard guard(q.device().index());
    at::Tensor o = output(plan, q, out, op);
    const KvmRows orows = rows(plan, o, s.num_tokens, s.num_heads, op, "out");
    const at::Tensor w = workspace(plan, q);
    check(kvm_paged_attention(&s, words, &c, &qr, &orows, scale_of(plan, scale), w.defined() ? w.data_ptr() : nullptr,
                              w.defined() ? w.numel() : 0, stream),
          op);
    if (out.has_value()) written({&o});
    return o;
}

at::Tensor prompt_attention(const Plan &plan, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                            std::optional<double> scale, const std::optional<at::Tensor> &out)
{
    const char *op = "prompt_attention";
    no_gradients({&q, &k, &v, out.has_value() ? &*out : nullptr}, op);
    void *stream;
    const int32_t *words = plan->use(q, op, &stream);
    const KvmStep &s = plan->step;
    const KvmRows qr = rows(plan, q, s.num_tokens, s.num_heads, op, "q"), kr = rows(plan, k, s.num_tokens, s.num_kv_heads, op, "k"),
                  vr = rows(plan, v, s.num_tokens, s.num_kv_heads, op, "v");
    const c10::hip::HIPGuard guard(q.device().index());
    at::Tensor o = output(plan, q, out, op);
    const KvmRows orows = rows(plan, o, s.num_tokens, s.num_heads, op, "out");
    const at::Tensor w = workspace(plan, q);
    check(kvm_prompt_attention(&s, words, &qr, &kr, &vr, &orows, scale_of(plan, scale), w.defined() ? w.data_ptr() : nullptr,
                               w.defined() ? w.numel() : 0, stream),
          op);
    if (out.has_value()) written({&o});
    return o;
}

}  // namespace

#ifndef KVM_CACHE_NS
#define KVM_CACHE_NS kvcache_ops
#endif
#define KVM_TEXT_(x) #x
#define KVM_TEXT(x) KVM_TEXT_(x)
#define KVM_PLAN "__torch__.torch.classes." KVM_TEXT(KVM_CACHE_NS) ".StepPlan plan"
#define KVM_TORCH_LIBRARY(ns, m) TORCH_LIBRARY(ns, m)

KVM_TORCH_LIBRARY(KVM_CACHE_NS, m)
{
    TORCH_CHECK(kvm_version() / 10000 == KVM_ABI_MAJOR, "libkvmove.so is version ", kvm_version(),
                ", this op library was built for major version ", KVM_ABI_MAJOR);
    m.class_<StepPlan>("StepPlan")
        .def(torch::init<std::vector<int64_t>, std::vector<int64_t>, std::vector<int64_t>, std::vector<int64_t>, int64_t,
                         int64_t, int64_t, int64_t, int64_t, int64_t, bool, int64_t>())
        .def("num_tokens", [](const Plan &p) { return p->step.num_tokens; })
        .def("num_kv_tokens", [](const Plan &p) { return p->step.num_kv_tokens; })
        .def("workspace_bytes", [](const Plan &p) { return kvm_attention_workspace(&p->step); })
        .def("device_index", [](const Plan &p) { return p->device_index(); })
        // the ops below once more: called this way they skip torch's dispatcher, which looks through every
        // argument of an op that takes a class (measured: 13.6 us of host time a call against 5.2)
        .def("write_kv", write_kv)
        .def("read_kv", read_kv)
        .def("paged_attention", paged_attention)
        .def("prompt_attention", prompt_attention);
    m.def("write_kv(" KVM_PLAN ", int layer, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache) -> ()", write_kv);
    m.def("read_kv(" KVM_PLAN ", int layer, Tensor k_cache, Tensor v_cache) -> (Tensor, Tensor)", read_kv);
    m.def("paged_attention(" KVM_PLAN ", int layer, Tensor q, Tensor k_cache, Tensor v_cache, float? scale=None, "
          "Tensor(a!)? out=None) -> Tensor(a!)",
          paged_attention);
    m.def("prompt_attention(" KVM_PLAN ", Tensor q, Tensor k, Tensor v, float? scale=None, Tensor(a!)? out=None) -> "
          "Tensor(a!)",
          prompt_attention);
}
