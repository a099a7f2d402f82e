// dce_api.hip -- implementation of the C ABI declared in include/dce.h.
// Owns device weights/scratch, repacks PyTorch-layout weights into kernel layouts, chunks
// arbitrarily long inputs over the scratch, and sequences the four kernels of the path:
//   conv_stack (z-score+conv1..4)  ->  fc_gemm (fc.0)  ->  fc_gemm (fc.3)  ->  fc3_tail (fc.6+argmax+bits)
// No exception or abort crosses the boundary; every failure is a negative dce_status plus a message.
#include "dce_ctx.h"
#include "block_ops.h"
#include <chrono>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstddef>

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>
#include <dlfcn.h>

using namespace dce;

#if defined(__x86_64__) || defined(__i386__)
#define DCE_CPU_RELAX() __builtin_ia32_pause()
#elif defined(__aarch64__)
#define DCE_CPU_RELAX() asm volatile("yield" ::: "memory")
#else
#define DCE_CPU_RELAX() do {} while (0)
#endif

namespace { int lat_service_stop(dce_ctx* c); }
// guard placement of the context's buffer group `bit` (option guard_mask: a bisecting aid of tools/guard_stress.py; default: every group)
static int guard_of(const dce_ctx* c, int bit) { return ((c->tuning.guard_mask >> bit) & 1) ? c->tuning.guard_alloc : 0; }


namespace {

struct KeyInfo { const char* name; int ndim; int64_t shape[3]; };
const KeyInfo kKeys[14] = {
    {"block1.0.weight", 3, {64, 54, 3}},   {"block1.0.bias", 1, {64, 0, 0}},
    {"block1.2.weight", 3, {64, 64, 3}},   {"block1.2.bias", 1, {64, 0, 0}},
    {"block2.0.weight", 3, {128, 64, 3}},  {"block2.0.bias", 1, {128, 0, 0}},
    {"block2.2.weight", 3, {128, 128, 3}}, {"block2.2.bias", 1, {128, 0, 0}},
    {"fc.0.weight", 2, {2048, 4736, 0}},   {"fc.0.bias", 1, {2048, 0, 0}},
    {"fc.3.weight", 2, {512, 2048, 0}},    {"fc.3.bias", 1, {512, 0, 0}},
    {"fc.6.weight", 2, {16, 512, 0}},      {"fc.6.bias", 1, {16, 0, 0}},
};

}  // namespace

namespace dce {

thread_local std::string g_create_error;
thread_local const Tuning* t_tuning = nullptr;
thread_local std::vector<const char*>* t_plan = nullptr;
thread_local Gate t_gate;

// ---- the ONE table of A/B switches (dce_kernels.h Tuning): key, member, kind.  dce_create_ex's option string / DCE_TUNE name them.
namespace {
struct TuneKey { const char* key; char kind; size_t off; bool experiments; };     // kind: b bool, i int, l long long
#define TK(name, kind) {#name, kind, offsetof(Tuning, name), false}
#define TKX(name, kind) {#name, kind, offsetof(Tuning, name), true}
const TuneKey kTuneKeys[] = {
    TK(gemm_tile, 'b'), TK(phased_min_tiles, 'i'), TK(phased_min_tiles1, 'i'), TK(phased_min, 'i'), TK(phased_cost, 'b'), TK(phased_sn, 'i'),
    TK(fc23, 'i'), TK(gemm_peel, 'b'), TK(conv_peel, 'b'), TK(gemm_small_deep, 'b'), TK(gemv, 'b'),
    TK(split_min, 'l'), TK(split_max, 'l'), TK(chain_min, 'l'), TK(chain_max, 'l'), TK(chain_max3, 'l'), TK(chain_bn16_max, 'l'),
    TK(wino1_max, 'l'), TK(winoh_max, 'l'), TK(winoq_max, 'l'), TK(winoq_chsplit_max, 'i'), TKX(wino1_w8, 'b'),
    TK(bf16_stream, 'b'), TK(x3_bf16_min, 'l'), TKX(x3_bf16_terms, 'i'), TK(bf16_conv_h2, 'b'), TK(bf16_conv_h2_min, 'l'),
    TK(online_graph, 'b'), TK(online_direct, 'b'), TK(latency, 'b'), TK(latency_mb, 'b'), TK(latency_mb_chalf, 'i'), TK(latency_idle_ms, 'i'), TK(latency_fc_delay, 'i'),
    TK(x3_conv, 'b'), TK(x3_conv_min, 'l'), TK(x3_min_tiles, 'i'), TKX(x3_unfused, 'b'), TK(x3_permk, 'b'), TKX(x3_fc3, 'b'), TKX(split_guard, 'b'), TK(h2_fc3, 'b'), TK(h2_min_tiles, 'i'), TK(guard_alloc, 'i'), TK(guard_mask, 'i'),
    TKX(bf16_k32, 'b'), TKX(gemm_lockstep, 'b'), TKX(gemm_pipe, 'b'), TKX(gemm_ki, 'b'), TKX(conv4, 'i'), TKX(x3_persist, 'b'), TKX(x3_pair, 'b'),
    TKX(x3_persist_min, 'l'), TKX(x3_pair_min, 'l'), TKX(conv_direct, 'b'), TKX(h2_ksplit, 'b'), TKX(bf16_fc3_ksplit, 'b'), TKX(one_per_cu, 'b'), TKX(trace_wino1, 'b'),
};
#undef TK
#undef TKX
}  // namespace

bool tuning_parse(const char* spec, Tuning& t, char* err, int err_len)
{
    if (!spec) return true;
    std::string s(spec);
    size_t pos = 0;
    while (pos < s.size()) {
        size_t end = s.find_first_of(",; ", pos);
        if (end == std::string::npos) end = s.size();
        const std::string item = s.substr(pos, end - pos);
        pos = end + 1;
        if (item.empty()) continue;
        const size_t eq = item.find('=');
        const std::string key = item.substr(0, eq), val = eq == std::string::npos ? "1" : item.substr(eq + 1);
        char* stop = nullptr;
        const long long v = strtoll(val.c_str(), &stop, 10);
        if (val.empty() || *stop != '\0') { snprintf(err, (size_t)err_len, "tuning option '%s': '%s' is not an integer", key.c_str(), val.c_str()); return false; }
        const TuneKey* k = nullptr;
        for (const TuneKey& c : kTuneKeys) if (key == c.key) { k = &c; break; }
        if (!k) { snprintf(err, (size_t)err_len, "unknown tuning option '%s' (the table is kTuneKeys in csrc/dce_api.hip; DESIGN.md appendix)", key.c_str()); return false; }
        if (k->experiments && !DCE_EXPERIMENTS) continue;             // a variant this build does not contain: its switch is ignored
        char* m = reinterpret_cast<char*>(&t) + k->off;
        if (k->kind == 'b') *reinterpret_cast<bool*>(m) = v != 0;
        else if (k->kind == 'i') *reinterpret_cast<int*>(m) = (int)v;
        else *reinterpret_cast<long long*>(m) = v;
    }
    if (t.x3_bf16_terms != 2 && t.x3_bf16_terms != 3) { snprintf(err, (size_t)err_len, "x3_bf16_terms must be 2 or 3"); return false; }
    return true;
}

const Tuning& tune()
{
    if (t_tuning) return *t_tuning;
    static const Tuning process_default = [] { Tuning t; char e[8]; (void)tuning_parse(getenv("DCE_TUNE"), t, e, (int)sizeof e); return t; }();   // a launcher reached outside a C-ABI call
    return process_default;
}

}  // namespace dce

namespace {

// roctx ranges around the entry points of the path, so that a profile of a host program (rocprofv3 --marker-trace, or any tool that
// listens to roctx) shows one named range per call next to the kernels it launched.  libdce.so has no link-time dependency on a marker
// library and by default brings none into the process: it binds to one only if something else -- the tool, the application -- has
// ALREADY loaded it (RTLD_NOLOAD), with local scope (its symbols do not enter the global namespace next to a torch wheel's own copy).
// DCE_ROCTX=1 loads it (librocprofiler-sdk-roctx first: what rocprofv3 listens to; the older libroctx64 otherwise), DCE_ROCTX=0 switches
// the ranges off.  Resolved once, at the first dce_create; without a tool attached a push/pop pair costs ~20 ns.
struct Roctx {
    int (*push)(const char*) = nullptr;
    int (*pop)() = nullptr;
    Roctx()
    {
        const char* e = getenv("DCE_ROCTX");
        if (e && atoi(e) == 0) return;
        const int how = RTLD_NOW | RTLD_LOCAL | ((e && atoi(e) != 0) ? 0 : RTLD_NOLOAD);
        for (const char* name : {"librocprofiler-sdk-roctx.so.1", "librocprofiler-sdk-roctx.so", "libroctx64.so.4", "libroctx64.so"}) {
            void* h = dlopen(name, how);
            if (!h) continue;
            push = reinterpret_cast<int (*)(const char*)>(dlsym(h, "roctxRangePushA"));
            pop = reinterpret_cast<int (*)()>(dlsym(h, "roctxRangePop"));
            if (push && pop) return;
            push = nullptr; pop = nullptr;
        }
    }
};
const Roctx& roctx() { static const Roctx r; return r; }
struct RoctxRange {
    bool on;
    explicit RoctxRange(const char* name) : on(roctx().push != nullptr) { if (on) roctx().push(name); }
    ~RoctxRange() { if (on) roctx().pop(); }
    RoctxRange(const RoctxRange&) = delete;
    RoctxRange& operator=(const RoctxRange&) = delete;
};

struct Timer {   // records a [begin,end] event pair around one launch when profiling is on
    dce_ctx* c; int slot; hipEvent_t a = nullptr, b = nullptr;
    Timer(dce_ctx* c_, int slot_) : c(c_), slot(slot_)
    {
        if (!c->prof) return;
        for (hipEvent_t* e : {&a, &b}) {
            if (!c->ev_pool.empty()) { *e = c->ev_pool.back(); c->ev_pool.pop_back(); }
            else if (hipEventCreate(e) != hipSuccess) { *e = nullptr; }
        }
        if (a && b) hipEventRecord(a, c->stream);
    }
    ~Timer()
    {
        if (!c->prof || !a || !b) return;
        hipEventRecord(b, c->stream);
        c->spans.push_back({slot, a, b});
    }
};

int drain_spans(dce_ctx* c)
{
    for (auto& s : c->spans) {
        HIP_TRY(c, hipEventSynchronize(s.b));
        float ms = 0.f;
        HIP_TRY(c, hipEventElapsedTime(&ms, s.a, s.b));
        c->prof_ms[s.slot] += ms;
        c->prof_n[s.slot] += 1;
        c->ev_pool.push_back(s.a);
        c->ev_pool.push_back(s.b);
    }
    c->spans.clear();
    return DCE_OK;
}

#if DCE_EXPERIMENTS
// DCE_FP32_SPLIT's range guard, static half (dce_kernels.h GuardArgs has the why).  For inputs |x| <= X every activation of layer l is
// bounded by  gain[l] X + offs[l]  with  gain[l] = gain[l-1] S_l,  offs[l] = offs[l-1] S_l + max|b_l|,  S_l = max over outputs of the
// sum of |w| (ReLU and MaxPool do not raise a bound).  The operands the kernels split are the input, the four conv layers' outputs
// (the last one = the features), fc.0's output h1 (fc.3 takes three-term operands too) and the weights of conv1..4, fc.0, fc.3: all must stay below LIM = 2^126 (bf16's largest finite number
// is 2^128 - 2^120; the margin covers the accumulators' rounding), so x_hi = min_l (LIM - offs[l]) / gain[l].  A z-scored window
// reaches |z| <= (n-1)/sqrt(n) = 12.166 at n = 150 (one sample against 149 equal ones), so a checkpoint whose x_hi is below that is
// REFUSED: the mode then runs the DCE_FP32 kernels for every call and says so (dce_last_plan, dce_split_guard_info).  The small side:
// a term below 2^-126 may be flushed by the matrix pipe; a layer whose largest |w| is below 2^-40, or a window whose largest |x| is,
// puts whole operands within 2^86 of that floor, where the third terms (2^-16 .. 2^-24 of a value) of the layers behind it can reach it --
// such a checkpoint is refused, such a window takes the fp32 kernels.  (Activation scales inside the net are bounded from below only
// through these two; single tiny weights or samples beside ordinary ones lose nothing that the fp32 sum would keep.)
void compute_split_guard(dce_ctx* c)
{
    dce_ctx::SplitGuard& g = c->guard;
    g = dce_ctx::SplitGuard{};
    g.x_hi = FLT_MAX; g.x_lo = 0.f;
    if (!c->tuning.split_guard) { g.reason = "guard switched off (split_guard=0)"; return; }
    const double LIM = std::ldexp(1.0, 126), SMALL = std::ldexp(1.0, -40), ZMAX = 149.0 / std::sqrt(150.0);
    static const int rows[6] = {64, 64, 128, 128, FC1, FC2}, cols[6] = {54 * 3, 64 * 3, 64 * 3, 128 * 3, FEAT, FC1};
    static const char* names[6] = {"block1.0", "block1.2", "block2.0", "block2.2", "fc.0", "fc.3"};
    double gain = 1.0, offs = 0.0, x_hi = LIM;
    char msg[256];
    for (int l = 0; l < 6; ++l) {
        const float* w = c->host_w[l < 4 ? 2 * l : 8 + 2 * (l - 4)].data();
        const float* b = c->host_w[l < 4 ? 2 * l + 1 : 9 + 2 * (l - 4)].data();
        double smax = 0.0, wmax = 0.0, bmax = 0.0;
        bool finite = true;
        for (int o = 0; o < rows[l]; ++o) {
            double sum = 0.0;
            for (int k = 0; k < cols[l]; ++k) { const double a = std::fabs((double)w[(size_t)o * cols[l] + k]); sum += a; if (a > wmax) wmax = a; }
            finite = finite && std::isfinite(sum) && std::isfinite((double)b[o]);
            if (sum > smax) smax = sum;
            if (std::fabs((double)b[o]) > bmax) bmax = std::fabs((double)b[o]);
        }
        gain *= smax; offs = offs * smax + bmax;
        g.gain[l] = gain; g.offs[l] = offs;
        if (l > 4 && !c->tuning.x3_fc3) continue;                     // fc.3 on fp32 operands (x3_fc3=0): its row is information only
        if (!finite || !std::isfinite(gain) || !std::isfinite(offs)) { snprintf(msg, sizeof msg, "%s holds a non-finite weight or its bound overflows", names[l]); g.refused = true; g.reason = msg; break; }
        if (wmax >= LIM) { snprintf(msg, sizeof msg, "%s: largest |w| %.3g reaches bf16's range limit", names[l], wmax); g.refused = true; g.reason = msg; break; }
        if (wmax < SMALL) { snprintf(msg, sizeof msg, "%s: largest |w| %.3g is below 2^-40 (third terms of the split near the subnormal range)", names[l], wmax); g.refused = true; g.reason = msg; break; }
        if (l == 5 || (l == 4 && !c->tuning.x3_fc3)) continue;        // fc.3's output is never split; fc.0's (h1) only when fc.3 takes three-term operands
        if (offs >= LIM) { snprintf(msg, sizeof msg, "%s: activation bound %.3g reaches bf16's range limit whatever the input", names[l], offs); g.refused = true; g.reason = msg; break; }
        if (gain > 0.0 && (LIM - offs) / gain < x_hi) x_hi = (LIM - offs) / gain;
    }
    if (!g.refused && x_hi < ZMAX * (1.0 + 1e-6)) {
        snprintf(msg, sizeof msg, "a z-scored window (|z| <= %.3f) can drive a layer's activations to %.3g: inputs are safe only up to %.3g", ZMAX, LIM, x_hi);
        g.refused = true; g.reason = msg;
    }
    if (g.refused) { g.x_hi = 0.f; return; }
    float xf = x_hi >= (double)FLT_MAX ? FLT_MAX : (float)x_hi;
    if ((double)xf > x_hi) xf = std::nextafterf(xf, 0.f);
    g.x_hi = xf; g.x_lo = (float)SMALL;
    g.reason = "ok";
}
#endif

// ---- latency mode (latency.hip): kernel arguments, and the resident service behind dce_online_push
// exchange memory (fine-grained): features (4736 floats) | h1, h2 as (value, tag) words | LatSync
constexpr size_t LAT_X_BYTES = FEAT * sizeof(float) + (FC1 + FC2) * sizeof(unsigned long long) + sizeof(LatSync);
LatArgs lat_args(dce_ctx* c)
{
    LatArgs a{};
    a.pk = c->pk;
    a.w1 = c->fc1w; a.b1 = c->fc1b; a.w2 = c->fc2w; a.b2 = c->fc2b; a.w3 = c->fc3w; a.b3 = c->fc3b;
    a.feat = c->lat_x; a.h1 = reinterpret_cast<unsigned long long*>(c->lat_x + FEAT); a.h2 = a.h1 + FC1;
    a.sync = c->lat_sync; a.mbox = c->lat_mbox; a.trace = c->lat_trace;
    a.fc_delay_ticks = (unsigned long long)(c->tuning.latency_fc_delay > 0 ? c->tuning.latency_fc_delay : 0);
    a.deadline_ticks = 5000000ull;                                    // 50 ms of the 100 MHz wall clock: far beyond any hand-over of a healthy launch
    a.idle_ticks = (unsigned long long)(c->tuning.latency_idle_ms > 0 ? c->tuning.latency_idle_ms : 1) * 100000ull;
    a.mb_w1 = c->lat_mb_w1; a.mb_w2 = c->lat_mb_w2;
    a.mb_feat = c->lat_mb_feat; a.mb_h1 = c->lat_mb_h1; a.mb_plt = c->lat_mb_plt; a.mb_flags = c->lat_mb_flags;
    return a;
}

// a wait of the one-shot kernel or of the service ran into its deadline: the arrival counters are out of step -> start over from zero
int lat_check_error(dce_ctx* c)
{
    if (!c->lat_mbox || !__atomic_load_n(&c->lat_mbox->error, __ATOMIC_ACQUIRE)) return DCE_OK;
    (void)hipStreamSynchronize(c->stream);
    if (c->lat_stream) (void)hipStreamSynchronize(c->lat_stream);
    c->lat_running = false;
    c->lat_mbox->error = 0;
    (void)hipMemset(c->lat_x, 0, LAT_X_BYTES);
    c->lat_seq = 0;
    return fail(c, DCE_ERR_HIP, "latency mode: a hand-over between the kernel's workgroups ran into its 50 ms deadline (is another kernel holding CUs? the mode needs all %d)", latency_grid());
}

int lat_service_stop(dce_ctx* c)
{
    if (!c || !c->lat_running) return DCE_OK;
    LatMailbox* mb = c->lat_mbox;
    mb->kind = 2;
    __atomic_store_n(&mb->req, ++c->lat_req, __ATOMIC_RELEASE);
    HIP_TRY(c, hipStreamSynchronize(c->lat_stream));                  // (if it had left by itself already: returns at once)
    c->lat_running = false;
    HIP_TRY(c, hipMemsetAsync(c->lat_x, 0, LAT_X_BYTES, c->lat_stream));          // the one-shot launches count their requests from one again
    HIP_TRY(c, hipStreamSynchronize(c->lat_stream));
    c->lat_seq = 0;
    return DCE_OK;
}

int lat_service_start(dce_ctx* c)
{
    LatMailbox* mb = c->lat_mbox;
    HIP_TRY(c, hipStreamSynchronize(c->stream));                      // the scratch rows and the device must be ours
    HIP_TRY(c, hipStreamSynchronize(c->lat_stream));
    HIP_TRY(c, hipMemsetAsync(c->lat_x, 0, LAT_X_BYTES, c->lat_stream));
    c->lat_seq = 0;
    LatArgs a = lat_args(c);
    a.seq = 1;
    a.hist = c->lat_hist; a.hist_state = c->lat_hist_state;
    a.req_base = c->lat_req; a.done_base = c->online_seq;
    mb->a.tag = mb->b.tag = c->online_seq;
    __atomic_store_n(&mb->alive, 0u, __ATOMIC_RELEASE);
    { TuningScope ts(&c->tuning);
      HIP_TRY(c, launch_latency(2, a, c->lat_stream)); }
    const auto t0 = std::chrono::steady_clock::now();
    while (!__atomic_load_n(&mb->alive, __ATOMIC_ACQUIRE)) {          // the kernel is up (its weights may still be on their way)
        DCE_CPU_RELAX();
        if (std::chrono::steady_clock::now() - t0 > std::chrono::seconds(5))
            return fail(c, DCE_ERR_HIP, "latency mode: the service kernel did not start within 5 s");
    }
    c->lat_running = true;
    return DCE_OK;
}

// every entry point other than dce_online_push: the resident kernel holds every CU's LDS -- it leaves first
int lat_quiesce(dce_ctx* c)
{
    int rc = lat_check_error(c);
    if (rc) return rc;
    return lat_service_stop(c);
}

#if DCE_EXPERIMENTS
// The gated DCE_FP32 fallback behind a guarded DCE_FP32_SPLIT launch (experiments build): binds the gate for the launchers and a tuning without the
// small-batch kernel families and row cuts (the gated kernels: conv_wino2, tile / phased GEMMs, fused fc.3, combine, tail).
struct GateScope {
    dce_ctx* c; TuningScope ts; std::vector<const char*>* plan;
    explicit GateScope(dce_ctx* c_) : c(c_), ts(&c_->gate_tuning), plan(t_plan)
    { c->gate_on = true; t_gate = Gate{c->d_guard, c->guard_gen, c->d_guard + 2}; t_plan = nullptr; }
    ~GateScope() { c->gate_on = false; t_gate = Gate{}; t_plan = plan; }
};
#endif

// ---- The plan of one chunk: which kernel family runs each stage of the path
//          conv stack (z-score + conv1..4)  ->  fc.0  ->  fc.3 (+ fc.6 chunk sums)  ->  fc.6 + argmax + contact bits.
// kPlanRows is the ONE table that turns (precision, windows of the launch) into that choice; choose_plan() looks the row up, applies the few
// overrides a caller's situation forces (taps, the online graph, a refused checkpoint, an option) and lets the FC families resolve by size;
// run_plan() executes it.  Inside a family the launchers pick the kernel by size (launch_conv_wino: quarter / half / one / two windows per
// workgroup; launch_fc_gemm: four-range / chain / tile / phased), all kernels of the fp32 family bit-identical.  tools/gen_options_table.py prints the
// table for DESIGN.md's appendix.
enum class Conv { WinoF32, WinoBf16, X2Bf16, H2, H2F32, H2Bf16,
                  WinoPlanes, X3Planes, X3F32, PairPlanes, PairBf16 };                     // (second line: experiments build)
enum class Fc0 { F32, Gemv, Bf16, H2, F8, X3 };
enum class Fc3 { F32, Gemv, Fused, Bf16, FusedBf16, FusedH2, H2, F8, FusedX3, FusedBf16K };
struct Plan {
    Conv conv; int permk;                 // permk: features (and fc.0's weights) in the K order t' * 128 + c; 2: from persistent workgroups (experiments)
    Fc0 fc0; bool split3;                 // split3 (experiments): fp32 features split by a kernel of their own in front of fc_gemm_x3
    Fc3 fc3; int64_t fused_rows;          // rows the fused fc.3 + fc.6 kernel takes (whole rounds); the rest goes to the chain kernel + tail
    bool guarded;                         // (experiments) DCE_FP32_SPLIT on pre-normalised windows: the conv kernel checks every window's range
    bool latency;                         // latency mode, one window: the whole path in ONE kernel of 256 co-resident workgroups (latency.hip)
    bool latency_mb;                      // latency mode, 2 .. 32 windows: the same on MFMA tiles (latency_mb.hip)
};

enum class Fam { F32, Bf16, H2 };                                         // operand family of an FC stage; the concrete kernel resolves by size
enum Thr { T_ONE, T_CONV16, T_H2FC, T_BF16H2, T_INF };                    // where a row begins: a constant, or the option that moves it
struct PlanRow { int precision; Thr from, below; Conv conv; Fam fc0, fc3; const char* what; };
constexpr PlanRow kPlanRows[] = {
    //  precision       from       below      conv stack      fc.0      fc.3 / fc.6
    {DCE_FP32,       T_ONE,     T_INF,     Conv::WinoF32,  Fam::F32,  Fam::F32,  "exact fp32 on the fp32 matrix pipe"},
    {DCE_BF16_FC,    T_ONE,     T_BF16H2,  Conv::X2Bf16,   Fam::Bf16, Fam::Bf16, "small launches: two bf16 terms per conv operand (results do not depend on the launch size)"},
    {DCE_BF16_FC,    T_BF16H2,  T_INF,     Conv::H2Bf16,   Fam::Bf16, Fam::Bf16, "conv results of fp32 grade (two fp16 terms, per-window scales), bf16 FC: BASELINE configs[4]"},
    {DCE_FP32_F16X2, T_ONE,     T_CONV16,  Conv::WinoF32,  Fam::F32,  Fam::F32,  "= DCE_FP32"},
    {DCE_FP32_F16X2, T_CONV16,  T_H2FC,    Conv::H2F32,    Fam::F32,  Fam::F32,  "mid-size: two-term fp16 conv stack, fp32 features, fp32 FC kernels"},
    {DCE_FP32_F16X2, T_H2FC,    T_INF,     Conv::H2,       Fam::H2,   Fam::H2,   "chip-filling: every GEMM on two fp16 terms per operand"},
};
int64_t plan_threshold(const Tuning& tu, Thr t)
{
    switch (t) {
    case T_ONE:    return 1;
    case T_CONV16: return tu.x3_conv_min;                                                 // 128
    case T_H2FC:   return 256ll * ((tu.h2_min_tiles + FC1 / 128 - 1) / (FC1 / 128) - 1) + 1;      // the first size with h2_min_tiles 256 x 128 tiles of fc.0: 1281
    case T_BF16H2: return tu.bf16_conv_h2_min;                                            // 257
    default:       return INT64_MAX;
    }
}

#if DCE_EXPERIMENTS
Plan choose_plan_experiments(const dce_ctx* c, int zscore, int64_t n);
#endif

// DCE_FP8_FC (both builds): DCE_BF16_FC's conv stack, the features quantized behind it, e4m3 products (their kernels resolve by size: block_gemm.hip)
Plan choose_plan_f8(const dce_ctx* c, int zscore, int64_t n)
{
    const Tuning& tu = tune();
    const bool online = c->src_row_dev != nullptr;
    Plan p{Conv::X2Bf16, 0, Fc0::F8, false, Fc3::F8, n, false, false, false};
    if (n >= plan_threshold(tu, T_BF16H2) && !online && tu.bf16_conv_h2 && tu.x3_conv && c->pkh2.w[0] && c->fc1w_f8p) p.conv = Conv::H2Bf16;
    else if (!tu.x3_conv || n < tu.x3_bf16_min || (online && !zscore)) p.conv = Conv::WinoBf16;
    p.permk = p.conv == Conv::H2Bf16 || (p.conv == Conv::X2Bf16 && tu.x3_permk && c->fc1w_f8p) ? 1 : 0;
    return p;
}

Plan choose_plan(const dce_ctx* c, int zscore, int64_t n)
{
    if (c->precision == DCE_FP8_FC) return choose_plan_f8(c, zscore, n);
    const Tuning& tu = tune();                                        // (bound by run_chunk: the context's switches)
    Plan p{Conv::WinoF32, 0, Fc0::F32, false, Fc3::F32, 0, false, false, false};
    const bool online = c->src_row_dev != nullptr;                    // the online graph: the window start lives in device memory
    // the latency plans serve WHOLE calls only (call_total == n): the last window of a call of k max_batch + 1 windows stays on the batch kernels,
    // so that DCE_FP32's "a window's bits do not depend on the size of the call" holds inside a call also for latency=1 contexts
    const bool lat = tu.latency && c->precision == DCE_FP32 && c->call_total == n && !online && !c->done_flag && !c->want_feat && !c->want_h1 && !c->want_h2 && !c->gate_on;
    if (lat && n == 1) { p.latency = true; return p; }
    if (lat && tu.latency_mb && n >= 2 && n <= LATMB_MAX_N && c->lat_mb_flags && c->lat_mb_w1) { p.latency_mb = true; return p; }
#if DCE_EXPERIMENTS
    return choose_plan_experiments(c, zscore, n);                     // (the lab keeps round 5's predicate tree: every A/B variant and DCE_FP32_SPLIT hang off it)
#else
    // ---- the row
    const int precision = (c->precision == DCE_FP32_F16X2 && c->h2_refused) ? DCE_FP32 : c->precision;      // a non-finite weight: the fp32 kernels
    const PlanRow* row = &kPlanRows[0];
    for (const PlanRow& r : kPlanRows)
        if (r.precision == precision && n >= plan_threshold(tu, r.from) && n < plan_threshold(tu, r.below)) { row = &r; break; }
    Conv conv = row->conv; Fam f0 = row->fc0, f3 = row->fc3;
    // ---- what a caller's situation overrides
    if (conv == Conv::H2 && (online || c->want_feat || !fc_gemm_h2_ok(n, FC1, FEAT, tu.h2_min_tiles))) {                                          // fp32 features for a tap; the online graph's window start; 32-bit offsets
        conv = n >= tu.x3_conv_min && !online ? Conv::H2F32 : Conv::WinoF32; f0 = f3 = Fam::F32;
    }
    if (conv == Conv::H2F32 && online) conv = Conv::WinoF32;
    if (conv == Conv::H2Bf16 && (online || c->want_feat || !tu.bf16_conv_h2 || !tu.x3_conv || !c->pkh2.w[0] || !c->fc1w_bf16p)) conv = Conv::X2Bf16;
    if (conv == Conv::X2Bf16 && (!tu.x3_conv || n < tu.x3_bf16_min || (online && !zscore))) conv = Conv::WinoBf16;                               // option / the online graph on pre-normalised rows
    if (f3 == Fam::H2 && (!tu.h2_fc3 || c->want_h1 || !c->fc2w_h2 || !c->h1h)) f3 = Fam::F32;                                                      // h1 wanted in fp32 (tap), option h2_fc3=0
    p.conv = conv;
    p.permk = conv == Conv::H2Bf16 ? 1 : (conv == Conv::X2Bf16 && tu.x3_permk && !c->want_feat && c->fc1w_bf16p) ? 1 : 0;
    // ---- the FC families resolve by size (what launch_fc_gemm does inside its family, one level up: GEMV, and fc.3 with fc.6's chunk sums in its epilogue)
    const bool gemv = tu.gemv && n <= FC_GEMV_MAX_M && !fc_split_ok(n, FC1, FEAT) && !fc_gemm_chain_ok(n, FC1, FEAT);   // a handful of windows: the weights streamed through all CUs
    p.fc0 = f0 == Fam::H2 ? Fc0::H2 : f0 == Fam::Bf16 ? Fc0::Bf16 : gemv ? Fc0::Gemv : Fc0::F32;
    p.fused_rows = n;
    if (f3 == Fam::Bf16) p.fc3 = fc23_fused_ok(n, 1) ? Fc3::FusedBf16 : Fc3::Bf16;
    else if (f3 == Fam::H2 && fc23_h2_ok(n)) p.fc3 = Fc3::FusedH2;                          // up to one and a half rounds of 128 x 64 tiles (12288 windows)
    else if (f0 != Fam::Bf16 && gemv) p.fc3 = Fc3::Gemv;
    else if (fc23_fused_ok(n, 0) && !fc_gemm_chain_ok(n, FC2, FC1) && !fc_split_ok(n, FC2, FC1)) {
        // chip-filling batch: fc.3's GEMM finishes fc.6's chunk sums in its epilogue (h2 never leaves the CU unless a tap asks for it).  The fused kernel
        // runs whole rounds of 256 tiles = 4096 windows: a batch that ends up to 2048 windows past a round gives that remainder to the chain kernel + tail
        // (same bits, rows are independent) instead of paying a full round for it.
        const int64_t rest = n % 4096;
        const bool cut = tu.gemm_peel && n > 4096 && rest && (rest <= 8 || fc_split_ok(rest, FC2, FC1) || fc_gemm_chain_ok(rest, FC2, FC1));
        p.fc3 = Fc3::Fused; p.fused_rows = cut ? n - rest : n;
    } else if (f3 == Fam::H2 && fc_gemm_h2_ok(n, FC2, FC1, tu.x3_min_tiles)) p.fc3 = Fc3::H2;   // past the fused tile's rounds: fc.3 on fc.0's 256 x 128 kernel (h2 fp32), then the tail
    else p.fc3 = Fc3::F32;
    return p;
#endif
}

#if DCE_EXPERIMENTS
// (experiments build) round 5's predicate tree: DCE_FP32_SPLIT with its range guard and gated fallback, the paired / persistent conv stacks, the K-split and
// lockstep GEMM variants -- everything that was measured slower than what ships, or that another precision dominates, hangs off this function
Plan choose_plan_experiments(const dce_ctx* c, int zscore, int64_t n)
{
    const Tuning& tu = tune();                                        // (bound by run_chunk: the context's switches, or their gated form)
    const bool wino = !(DCE_EXPERIMENTS && tu.conv_direct);
    const bool online = c->src_row_dev != nullptr;                    // the online graph: the window start lives in device memory
    Plan p{Conv::WinoF32, 0, Fc0::F32, false, Fc3::F32, 0, false, false, false};
    if (c->precision == DCE_BF16_FC) {
        const bool x3c = tu.x3_conv && wino && n >= tu.x3_bf16_min && (!online || zscore);
        const bool pair = DCE_EXPERIMENTS && tu.x3_conv && tu.x3_pair && wino && !online && !c->want_feat && n >= tu.x3_pair_min;
        p.conv = pair ? Conv::PairBf16 : x3c ? Conv::X2Bf16 : Conv::WinoBf16;
        p.permk = pair ? 1 : (x3c && tu.x3_permk && !c->want_feat && c->fc1w_bf16p) ? ((DCE_EXPERIMENTS && tu.x3_persist && n >= tu.x3_persist_min) ? 2 : 1) : 0;
        if (tu.bf16_conv_h2 && tu.x3_conv && tu.x3_bf16_terms == 2 && n >= tu.bf16_conv_h2_min && c->pkh2.w[0] && c->fc1w_bf16p && wino && !online && !c->want_feat && !pair) {
            p.conv = Conv::H2Bf16; p.permk = 1;                       // conv results of fp32 grade from two fp16 terms with per-window scales (conv_h2.hip): configs[4] as written
        }
        p.fc0 = Fc0::Bf16;
        p.fc3 = fc23_fused_ok(n, 1) ? (DCE_EXPERIMENTS && tu.bf16_fc3_ksplit && n + 128 <= 2 * c->max_batch ? Fc3::FusedBf16K : Fc3::FusedBf16) : Fc3::Bf16;
        p.fused_rows = n;
        return p;
    }
    const bool h2 = c->precision == DCE_FP32_F16X2 && !c->h2_refused && wino && !online && !c->want_feat && fc_gemm_h2_ok(n, FC1, FEAT, tu.h2_min_tiles);
    if (h2) { p.conv = Conv::H2; p.fc0 = Fc0::H2; }
    else if (c->precision == DCE_FP32_F16X2 && !c->h2_refused && wino && !online && n >= tu.x3_conv_min) p.conv = Conv::H2F32;   // mid-size batch (or a feature tap): two-term fp16 conv stack, fp32 features, fp32 FC kernels
    const bool split = c->precision == DCE_FP32_SPLIT && !c->guard.refused && !c->gate_on;
    // DCE_FP32_SPLIT at a chip-filling batch: the conv stack writes the features straight as three bf16 planes (unless a tap wants
    // them in fp32: then a kernel of its own splits them)
    const bool x3 = split && fc_gemm_x3_ok(n, FC1, FEAT);
    const bool fused = x3 && wino && !c->want_feat && !tu.x3_unfused;
    const bool pair = DCE_EXPERIMENTS && fused && tu.x3_conv && tu.x3_pair && !online && n >= tu.x3_pair_min;
    if (pair) { p.conv = Conv::PairPlanes; p.permk = 1; }
    else if (fused && tu.x3_conv && !online) {
        p.conv = Conv::X3Planes;
        p.permk = (tu.x3_permk && c->fc1w_x3p) ? ((DCE_EXPERIMENTS && tu.x3_persist && n >= tu.x3_persist_min) ? 2 : 1) : 0;
    } else if (fused) p.conv = Conv::WinoPlanes;
    else if (split && !x3 && tu.x3_conv && wino && !online && !c->want_feat && n >= tu.x3_conv_min) p.conv = Conv::X3F32;   // mid-size batch: three-term conv stack, fp32 FC kernels
    p.guarded = tu.split_guard && !zscore && (p.conv == Conv::X3Planes || p.conv == Conv::X3F32);     // (the A/B routes -- Winograd stack + split, taps -- carry the static guard only)
    // a handful of windows (online mode, batch_size 1): the weights streamed through all CUs (from 9 windows up launch_fc_gemm
    // picks the four-range / chain kernels instead); same bits as the GEMMs
    const bool gemv = tu.gemv && !c->gate_on && n <= FC_GEMV_MAX_M && !fc_split_ok(n, FC1, FEAT) && !fc_gemm_chain_ok(n, FC1, FEAT);
    p.fc0 = h2 ? Fc0::H2 : x3 ? Fc0::X3 : gemv ? Fc0::Gemv : Fc0::F32;
    p.split3 = x3 && !fused;
    p.fc3 = gemv ? Fc3::Gemv : Fc3::F32;
    const bool h2f3 = h2 && tu.h2_fc3 && !c->want_h1 && c->fc2w_h2 && c->h1h;                   // DCE_FP32_F16X2: fc.3 on two-term fp16 operands too (h1 leaves fc.0 as two fp16 terms + row scales)
    if (h2f3 && fc23_h2_ok(n)) { p.fc3 = Fc3::FusedH2; p.fused_rows = n; }
    else if (fc23_fused_ok(n, 0) && !fc_gemm_chain_ok(n, FC2, FC1) && !fc_split_ok(n, FC2, FC1)) {
        // chip-filling batch: fc.3's GEMM finishes fc.6's chunk sums in its epilogue (h2 never leaves the CU unless a tap asks for
        // it); one small kernel adds them up.  Same summation tree as the tail kernel.  The fused kernel runs whole rounds of 256
        // tiles = 4096 windows: a batch that ends up to 2048 windows past a round gives that remainder to the chain kernel + tail
        // (same bits, rows are independent) instead of paying a full round for it.
        const int64_t rest = n % 4096;
        p.fc3 = (x3 && !c->want_h1 && c->fc2w_x3 && c->h1p && fc23_x3_ok(n)) ? Fc3::FusedX3 : Fc3::Fused;      // fc.3 on three-term operands too (h1 then leaves fc.0 as three planes)
        const bool cut = p.fc3 == Fc3::Fused && tu.gemm_peel && !c->gate_on && n > 4096 && rest && (rest <= 8 || fc_split_ok(rest, FC2, FC1) || fc_gemm_chain_ok(rest, FC2, FC1));
        p.fused_rows = cut ? n - rest : n;
    } else if (h2f3 && fc_gemm_h2_ok(n, FC2, FC1, tu.x3_min_tiles))
        p.fc3 = Fc3::H2;                                              // a launch past the fused tile's one round: fc.3 on fc.0's 256 x 128 kernel (h2 in fp32), then the tail
    return p;
}

#endif

#if DCE_EXPERIMENTS
// fc.0's three planes in the reference's K order, for the routes that do not take the conv kernels' order t' * 128 + c (feature taps,
// x3_unfused, x3_conv=0, x3_permk=0): 58 MB that the product route never reads, so they are split and uploaded on first use
int ensure_fc1w_x3(dce_ctx* c)
{
    if (c->fc1w_x3) return DCE_OK;
    const auto& v = c->host_w[8];
    std::vector<unsigned short> planes(3 * v.size());
    split3_host(v.data(), FC1, FEAT, planes.data());
    HIP_TRY(c, dev_alloc(&c->fc1w_x3_own, guard_of(c, 0), planes.size() * sizeof(unsigned short)));
    HIP_TRY(c, hipMemcpy(c->fc1w_x3_own, planes.data(), planes.size() * sizeof(unsigned short), hipMemcpyHostToDevice));
    c->fc1w_x3 = c->fc1w_x3_own;
    return DCE_OK;
}
#endif

// DCE_FP8_FC's operands live in the halves of `feat` and `h1` that 16-bit values leave free: features e4m3 behind the bf16 ones, their scales behind those
// (37 bytes a row); h1 e4m3 and its scales (16 bytes a row) in h1.
unsigned char* f8_features(const dce_ctx* c) { return reinterpret_cast<unsigned char*>(c->feat) + (size_t)c->max_batch * FEAT * 2; }
unsigned char* f8_feature_scales(const dce_ctx* c) { return f8_features(c) + (size_t)c->max_batch * FEAT; }
unsigned char* f8_h1_scales(const dce_ctx* c) { return reinterpret_cast<unsigned char*>(c->h1) + (size_t)c->max_batch * FC1; }
static_assert(FEAT % 128 == 0 && FC1 % 128 == 0 && FEAT * 4 >= FEAT * 3 + FEAT / 128 && FC1 * 4 >= FC1 + FC1 / 128, "they fit");

QuantArgs features_f8(const dce_ctx* c, int64_t n)
{
    QuantArgs a{};
    a.x = reinterpret_cast<const char*>(c->feat); a.x_row = FEAT * 2;
    a.q = f8_features(c); a.q_row = FEAT;
    a.s = f8_feature_scales(c); a.s_block = n;
    a.rows = n; a.k = FEAT; a.kblocks = FEAT / BLK; a.units = n * a.kblocks;
    return a;
}
ProductArgs fc0_f8(const dce_ctx* c, int64_t n, int permk)
{
    ProductArgs p{};
    p.a = reinterpret_cast<const char*>(f8_features(c)); p.a_row = FEAT; p.a_rows = n; p.sa = f8_feature_scales(c); p.sa_block = n;
    p.b = reinterpret_cast<const char*>(permk ? c->fc1w_f8p : c->fc1w_f8); p.b_row = FEAT; p.sb = permk ? c->fc1s_f8p : c->fc1s_f8; p.sb_row = FEAT / BLK;
    p.bias = c->fc1b; p.relu = 1;
    p.y = reinterpret_cast<char*>(c->h1); p.y_row = FC1; p.ys = f8_h1_scales(c); p.ys_block = n;
    p.m = (int)n; p.n = FC1; p.kbytes = FEAT; p.groups = 1;
    return p;
}
ProductArgs fc3_f8(const dce_ctx* c, int64_t n)
{
    ProductArgs p{};
    p.a = reinterpret_cast<const char*>(c->h1); p.a_row = FC1; p.a_rows = n; p.sa = f8_h1_scales(c); p.sa_block = n;
    p.b = reinterpret_cast<const char*>(c->fc2w_f8); p.b_row = FC1; p.sb = c->fc2s_f8; p.sb_row = FC1 / BLK;
    p.bias = c->fc2b; p.relu = 1;
    p.y = reinterpret_cast<char*>(c->h2); p.y_row = FC2 * 4;
    p.m = (int)n; p.n = FC2; p.kbytes = FC1; p.groups = 1;
    return p;
}

// ... and its weights, quantized on the device from the fp32 ones (w1p: fc.0 in the feature order t' * 128 + c, on the host; empty: not wanted)
int quantize_weights_f8(dce_ctx* c, const std::vector<float>& w1p)
{
    const size_t n1 = (size_t)FC1 * FEAT, s1 = (size_t)(FC1 / BLK) * (FEAT / BLK), n2 = (size_t)FC2 * FC1, s2 = (size_t)(FC2 / BLK) * (FC1 / BLK);
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t total = 2 * (n1 + up(s1)) + n2 + up(s2);
    if (c->f8) { HIP_TRY(c, dev_free(c->f8)); c->f8 = nullptr; }
    HIP_TRY(c, dev_alloc(&c->f8, guard_of(c, 8), total));
    unsigned char *w1 = c->f8, *w1q = w1 + n1 + up(s1), *w2 = w1q + n1 + up(s1);
    auto run = [&](const float* x, unsigned char* q, int rows, int k) {
        QuantArgs a{};
        a.x = reinterpret_cast<const char*>(x); a.x_row = (long long)k * 4;
        a.q = q; a.q_row = k;
        a.s = q + (size_t)rows * k; a.s_block = k / BLK;
        a.rows = rows; a.k = k; a.kblocks = k / BLK; a.units = (long long)rows * a.kblocks;
        return launch_quantize(a, 0, 1, BLK, 1, c->stream);
    };
    HIP_TRY(c, run(c->fc1w, w1, FC1, FEAT));
    HIP_TRY(c, run(c->fc2w, w2, FC2, FC1));
    c->fc1w_f8 = w1; c->fc1s_f8 = w1 + n1; c->fc2w_f8 = w2; c->fc2s_f8 = w2 + n2;
    if (!w1p.empty()) {
        float* tmp = nullptr;
        HIP_TRY(c, hipMalloc(reinterpret_cast<void**>(&tmp), n1 * sizeof(float)));
        hipError_t e = hipMemcpy(tmp, w1p.data(), n1 * sizeof(float), hipMemcpyHostToDevice);
        if (e == hipSuccess) e = run(tmp, w1q, FC1, FEAT);
        if (e == hipSuccess) e = hipStreamSynchronize(c->stream);
        (void)hipFree(tmp);
        if (e != hipSuccess) return fail(c, DCE_ERR_HIP, "quantizing fc.0's weights failed: %s", hipGetErrorString(e));
        c->fc1w_f8p = w1q; c->fc1s_f8p = w1q + n1;
    }
    HIP_TRY(c, hipStreamSynchronize(c->stream));
    return DCE_OK;
}

// One chunk (n <= max_batch) of the path, everything on device.
//   src: raw sequence rows (zscore=1) or pre-normalised windows (zscore=0)
int run_plan(dce_ctx* c, const Plan& p, const float* src, int zscore, int64_t n,
             float* logits, int32_t* pred, uint8_t* contacts, uint8_t* packed)
{
    const hipStream_t st = c->stream;
    if (p.latency) {
        Timer t(c, 0);
        LatArgs a = lat_args(c);
        a.seq = ++c->lat_seq;
        a.src = src; a.logits = logits; a.pred = pred; a.contacts = contacts; a.packed = packed;
        HIP_TRY(c, launch_latency(zscore ? 1 : 0, a, st));
        return DCE_OK;
    }
    if (p.latency_mb) {
        Timer t(c, 0);
        LatArgs a = lat_args(c);
        a.seq = ++c->lat_mb_seq;
        a.mb_n = (int)n; a.mb_chalf = n <= c->tuning.latency_mb_chalf && n <= LATMB_MAX_N / 2 ? 1 : 0;
        a.src = src; a.logits = logits; a.pred = pred; a.contacts = contacts; a.packed = packed;
        HIP_TRY(c, launch_latency_mb(zscore, a, st));
        return DCE_OK;
    }
    unsigned short* featb = reinterpret_cast<unsigned short*>(c->feat);
    const bool wino = !(DCE_EXPERIMENTS && c->tuning.conv_direct);
    auto conv_f32 = wino ? launch_conv_wino : launch_conv_stack;
#if DCE_EXPERIMENTS
    const GuardArgs ga = p.guarded ? GuardArgs{c->d_guard, c->guard_gen, c->guard.x_hi, c->guard.x_lo} : GuardArgs{};
#endif
    { Timer t(c, 0);
      switch (p.conv) {
      case Conv::WinoF32:    HIP_TRY(c, conv_f32(src, zscore, n, c->pk, c->feat, 0, st, c->src_row_dev)); break;
      case Conv::WinoBf16:   HIP_TRY(c, conv_f32(src, zscore, n, c->pk, c->feat, 1, st, c->src_row_dev)); break;
      case Conv::X2Bf16:     HIP_TRY(c, launch_conv_x3_bf16(src, zscore, n, c->pkx3, featb, st, p.permk, DCE_EXPERIMENTS ? c->tuning.x3_bf16_terms : 2, c->src_row_dev)); break;
#if DCE_EXPERIMENTS
      case Conv::WinoPlanes: HIP_TRY(c, launch_conv_wino(src, zscore, n, c->pk, c->feat3, 2, st, c->src_row_dev)); break;
      case Conv::X3Planes:   HIP_TRY(c, launch_conv_x3(src, zscore, n, c->pkx3, c->feat3, st, p.permk, ga)); break;
      case Conv::X3F32:      HIP_TRY(c, launch_conv_x3_f32(src, zscore, n, c->pkx3, c->feat, st, ga)); break;
      case Conv::PairPlanes: HIP_TRY(c, launch_conv_x3p(src, zscore, n, c->pkx3, c->feat3, st)); break;
      case Conv::PairBf16:   HIP_TRY(c, launch_conv_x3p_bf16(src, zscore, n, c->pkx3, featb, st)); break;
#else
      default: return fail(c, DCE_ERR_STATE, "internal: a conv kernel family of the experiments build in a product plan");
#endif
      case Conv::H2:         HIP_TRY(c, launch_conv_h2(src, zscore, n, c->pkh2, c->feat3, c->feat_scale, st)); break;
      case Conv::H2F32:      HIP_TRY(c, launch_conv_h2_f32(src, zscore, n, c->pkh2, c->feat, st)); break;
      case Conv::H2Bf16:     HIP_TRY(c, launch_conv_h2_bf16(src, zscore, n, c->pkh2, featb, st)); break;
      } }
    { Timer t(c, 1);
      switch (p.fc0) {
      case Fc0::F32:  HIP_TRY(c, launch_fc_gemm(c->feat, c->fc1w, c->fc1b, c->h1, n, FC1, FEAT, 1, st)); break;
      case Fc0::Gemv: HIP_TRY(c, launch_fc_gemv(c->feat, c->fc1w, c->fc1b, c->h1, n, FC1, FEAT, 1, st)); break;
#if DCE_EXPERIMENTS
      case Fc0::X3:   // fc.0 on the bf16 matrix pipe with three-term operands (fc_gemm_x3.hip); everything behind it as in DCE_FP32
          if (!p.permk) { const int rc = ensure_fc1w_x3(c); if (rc) return rc; }
          if (p.split3) HIP_TRY(c, launch_split3(c->feat, c->feat3, n, FEAT, st));
          if (p.fc3 == Fc3::FusedX3) HIP_TRY(c, launch_fc_gemm_x3(c->feat3, p.permk ? c->fc1w_x3p : c->fc1w_x3, c->fc1b, c->h1p, n, FC1, FEAT, 1, st, 1));
          else HIP_TRY(c, launch_fc_gemm_x3(c->feat3, p.permk ? c->fc1w_x3p : c->fc1w_x3, c->fc1b, c->h1, n, FC1, FEAT, 1, st));
          break;
#else
      case Fc0::X3: return fail(c, DCE_ERR_STATE, "internal: fc.0 on three-term operands is an experiments-build kernel");
#endif
      case Fc0::F8:
          HIP_TRY(c, launch_quantize(features_f8(c, n), 1, 1, 1, 1, st));
          HIP_TRY(c, launch_product(fc0_f8(c, n, p.permk), IN_F8_E8, OUT_E4M3, st));
          plan_note("quantize_e4m3"); plan_note("fc0_e4m3");
          break;
      case Fc0::Bf16: HIP_TRY(c, launch_fc_gemm_bf16(c->feat, p.permk ? c->fc1w_bf16p : c->fc1w_bf16, c->fc1b, c->h1, 1, n, FC1, FEAT, 1, st)); break;
      case Fc0::H2:
          if (p.fc3 == Fc3::FusedH2 || p.fc3 == Fc3::H2) HIP_TRY(c, launch_fc_gemm_h2(c->feat3, c->feat_scale, c->fc1w_h2, c->fc1_sw, c->fc1b, c->h1, n, FC1, FEAT, 1, st, c->h1h, c->h1_scale, c->fc1_eW, c->fc1_eB));
          else HIP_TRY(c, launch_fc_gemm_h2(c->feat3, c->feat_scale, c->fc1w_h2, c->fc1_sw, c->fc1b, c->h1, n, FC1, FEAT, 1, st));
          break;
      } }
    const int64_t nf = p.fused_rows;
    { Timer t(c, 2);
      switch (p.fc3) {
      case Fc3::F8: HIP_TRY(c, launch_product(fc3_f8(c, n), IN_F8_E8, OUT_F32, st)); plan_note("fc3_e4m3"); break;
      case Fc3::F32:  HIP_TRY(c, launch_fc_gemm(c->h1, c->fc2w, c->fc2b, c->h2, n, FC2, FC1, 1, st)); break;
      case Fc3::Gemv: HIP_TRY(c, launch_fc_gemv(c->h1, c->fc2w, c->fc2b, c->h2, n, FC2, FC1, 1, st)); break;
      case Fc3::Bf16: HIP_TRY(c, launch_fc_gemm_bf16(c->h1, c->fc2w_bf16, c->fc2b, c->h2, 0, n, FC2, FC1, 1, st)); break;
#if DCE_EXPERIMENTS
      case Fc3::FusedX3: HIP_TRY(c, launch_fc23_fused_x3(c->h1p, c->fc2w_x3, c->fc2b, c->fc3w, c->part, c->max_batch, c->want_h2 ? c->h2 : nullptr, n, st)); break;
#else
      case Fc3::FusedX3: return fail(c, DCE_ERR_STATE, "internal: fc.3 on three-term operands is an experiments-build kernel");
#endif
      case Fc3::H2: HIP_TRY(c, launch_fc_gemm_h2(c->h1h, c->h1_scale, c->fc2w_h2, c->fc2_sw, c->fc2b, c->h2, n, FC2, FC1, 1, st)); break;
      case Fc3::FusedH2: HIP_TRY(c, launch_fc23_fused_h2(c->h1h, c->h1_scale, c->fc2w_h2, c->fc2_sw, c->fc2b, c->fc3w, c->part, c->max_batch, c->want_h2 ? c->h2 : nullptr, n, st)); break;
      case Fc3::FusedBf16K: HIP_TRY(c, launch_fc23_fused_bf16k(c->h1, c->fc2w_bf16, c->fc2b, c->fc3w, c->part, c->max_batch, c->want_h2 ? c->h2 : nullptr, n, st)); break;
      case Fc3::FusedBf16: HIP_TRY(c, launch_fc23_fused(c->h1, c->fc2w_bf16, c->fc2b, c->fc3w, 1, c->part, c->max_batch, c->want_h2 ? c->h2 : nullptr, n, st)); break;
      case Fc3::Fused:
          HIP_TRY(c, launch_fc23_fused(c->h1, c->fc2w, c->fc2b, c->fc3w, 0, c->part, c->max_batch, c->want_h2 ? c->h2 : nullptr, nf, st));
          if (nf < n) HIP_TRY(c, (n - nf <= 8 ? launch_fc_gemv : launch_fc_gemm)(c->h1 + nf * FC1, c->fc2w, c->fc2b, c->h2 + nf * FC2, n - nf, FC2, FC1, 1, st));
          break;
      } }
    { Timer t(c, 3);
      if (p.fc3 == Fc3::Fused || p.fc3 == Fc3::FusedX3 || p.fc3 == Fc3::FusedBf16 || p.fc3 == Fc3::FusedBf16K || p.fc3 == Fc3::FusedH2) {
          HIP_TRY(c, launch_fc6_combine(c->part, c->max_batch, c->fc3b, nf, logits, pred, contacts, st, packed));
          if (nf < n) HIP_TRY(c, launch_fc3_tail(c->h2 + nf * FC2, c->fc3w, c->fc3b, n - nf, logits ? logits + nf * NCLS : nullptr, pred ? pred + nf : nullptr,
                                                 contacts ? contacts + nf * 4 : nullptr, st, nullptr, 0, nullptr, packed ? packed + nf * PACKED_ROW : nullptr));
      } else HIP_TRY(c, launch_fc3_tail(c->h2, c->fc3w, c->fc3b, n, logits, pred, contacts, st, c->done_flag, c->done_seq, c->seq_counter_dev, packed)); }
    return DCE_OK;
}

int run_chunk(dce_ctx* c, const float* src, int zscore, int64_t n,
              float* logits, int32_t* pred, uint8_t* contacts, uint8_t* packed = nullptr)
{
    TuningScope tuning_scope(&c->tuning);
    struct PlanScope { explicit PlanScope(std::vector<const char*>* p) { p->clear(); t_plan = p; } ~PlanScope() { t_plan = nullptr; } } plan_scope(&c->plan);
    c->prof = c->prof_period > 0 && (c->prof_tick++ % c->prof_period) == 0;
    if (c->split_alias) plan_note("fp32_split_is_fp32_f16x2");      // (product library: include/dce.h DCE_FP32_SPLIT)
    if (c->precision == DCE_FP32_SPLIT && c->guard.refused) plan_note("split_guard_refused");
    if (c->precision == DCE_FP32_F16X2 && c->h2_refused) plan_note("f16x2_refused");
    const Plan p = choose_plan(c, zscore, n);
    int rc = DCE_OK;
#if !DCE_EXPERIMENTS
    rc = run_plan(c, p, src, zscore, n, logits, pred, contacts, packed);
#else
    if (p.guarded) { ++c->guard_gen; ++c->guard_launches; }                                     // a generation per guarded launch: no reset of the device word between them
    rc = run_plan(c, p, src, zscore, n, logits, pred, contacts, packed);
    if (rc == DCE_OK && p.guarded) {
        // A window of this launch outside the guarded range has written this launch's generation to the guard word: the DCE_FP32
        // kernel sequence behind it runs then (every workgroup of it reads the word first and leaves when it holds another value)
        // and overwrites the launch's results.  Nothing comes back to the host: device-pointer callers stay asynchronous.
        plan_note("gated_fp32_fallback");                            // (its kernels are not listed: they run only when the gate opens)
        GateScope gate(c);
        rc = run_plan(c, choose_plan(c, zscore, n), src, zscore, n, logits, pred, contacts, packed);
    }
#endif
    if (rc == DCE_OK && c->spans.size() > 4096) rc = drain_spans(c);
    return rc;
}

// feat3 serves DCE_FP32_SPLIT (three bf16 planes of max_batch + 1 rows) and DCE_FP32_F16X2 (two fp16 terms, padded by a tile of rows that ragged
// K-split tiles read: fc_gemm_h2_pad_rows): ONE size, so that a context re-finalized in the other precision never finds it short
size_t feat3_halfs(int64_t max_batch)
{
    return std::max((size_t)(max_batch + 1) * FEAT * 3, (size_t)(max_batch + fc_gemm_h2_pad_rows()) * FEAT * 2);
}

int ensure_in(dce_ctx* c, size_t bytes)
{
    if (c->d_in_bytes >= bytes) return DCE_OK;
    if (c->d_in) { HIP_TRY(c, dev_free(c->d_in)); c->d_in = nullptr; c->d_in_bytes = 0; }
    HIP_TRY(c, dev_alloc(&c->d_in, guard_of(c, 5), bytes));
    c->d_in_bytes = bytes;
    return DCE_OK;
}

int ensure_out(dce_ctx* c, size_t rows)
{
    if (c->d_out_rows >= rows) return DCE_OK;
    c->d_out_rows = 0;
    if (c->d_logits)   { HIP_TRY(c, dev_free(c->d_logits));   c->d_logits = nullptr; }
    if (c->d_pred)     { HIP_TRY(c, dev_free(c->d_pred));     c->d_pred = nullptr; }
    if (c->d_contacts) { HIP_TRY(c, dev_free(c->d_contacts)); c->d_contacts = nullptr; }
    if (c->d_packed)   { HIP_TRY(c, dev_free(c->d_packed));   c->d_packed = nullptr; }
    HIP_TRY(c, dev_alloc(&c->d_packed, guard_of(c, 6), rows * PACKED_ROW));
    HIP_TRY(c, dev_alloc(&c->d_logits, guard_of(c, 6), rows * NCLS * sizeof(float)));
    HIP_TRY(c, dev_alloc(&c->d_pred, guard_of(c, 6), rows * sizeof(int32_t)));
    HIP_TRY(c, dev_alloc(&c->d_contacts, guard_of(c, 6), rows * 4));
    c->d_out_rows = rows;
    return DCE_OK;
}

// packed rows are written (4-byte float / uchar4 stores) and read (unsigned loads) as 32-bit words: a DEVICE pointer to them must
// be 4-byte aligned (the rows themselves are 68 bytes, so every row of an aligned buffer is)
bool misaligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) != 0; }

int check_ready(dce_ctx* c)
{
    if (!c) return DCE_ERR_ARG;
    if (!c->finalized) return fail(c, DCE_ERR_STATE, "weights not finalized: call dce_finalize_weights first");
    return DCE_OK;
}
int check_ready_quiet(dce_ctx* c)                         // ... and the latency mode's resident kernel, if any, has left
{
    const int rc = check_ready(c);
    return rc ? rc : lat_quiesce(c);
}

// Shared driver for forward_windows / infer_sequence: chunk over max_batch.
//   device pointers: kernels only, asynchronous on the ctx stream.
//   host pointers  : staged through ctx-owned device buffers, chunk by chunk on a second stream, so
//                    that the H2D copy of chunk i+1 and the D2H copy of chunk i-1 run under the
//                    kernels of chunk i (the copies are ~10 % of a 1e6-window call when serialised);
//                    returns once every result has landed.
int run_all(dce_ctx* c, const float* src, int zscore, int64_t n, int64_t src_floats, int on_device,
            float* logits, int32_t* pred, uint8_t* contacts, uint8_t* packed = nullptr)
{
    const int64_t row_floats = zscore ? CH : (int64_t)WIN * CH;
    c->call_total = n;
    const int64_t nchunks = (n + c->max_batch - 1) / c->max_batch;
    auto chunk_rows = [&](int64_t i) { const int64_t i0 = i * c->max_batch; return (n - i0) < c->max_batch ? (n - i0) : c->max_batch; };
    if (on_device) {
        for (int64_t i = 0; i < nchunks; ++i) {
            const int64_t i0 = i * c->max_batch;
            int rc = run_chunk(c, src + i0 * row_floats, zscore, chunk_rows(i),
                               logits ? logits + i0 * NCLS : nullptr, pred ? pred + i0 : nullptr,
                               contacts ? contacts + i0 * 4 : nullptr, packed ? packed + i0 * PACKED_ROW : nullptr);
            if (rc) return rc;
        }
        return DCE_OK;
    }
    // ---- host pointers: a ring of RING chunk slots.  Chunk i lives in slot i % RING:
    //   xfer stream : [wait computed(i-RING)] H2D(i) -> staged-in(i)        [wait computed(i)] D2H(i) -> staged-out(i)
    //   ctx stream  : [wait staged-in(i), staged-out(i-RING)] kernels(i) -> computed(i)
    // so the copies of chunks i+1 / i-1 run under the kernels of chunk i and the device footprint is
    // RING * max_batch rows, whatever n is.  The copies go straight from / to the caller's memory
    // (pageable or pinned; HIP stages pageable memory itself).
    constexpr int RING = 3;
    const int64_t mb = c->max_batch < n ? c->max_batch : n;
    const int64_t in_slot_floats = zscore ? (mb + WIN - 1) * CH : mb * row_floats;
    (void)src_floats;
    int rc = ensure_in(c, (size_t)RING * in_slot_floats * sizeof(float));
    if (rc) return rc;
    rc = ensure_out(c, (size_t)RING * mb);
    if (rc) return rc;
    if (!c->xfer_stream) HIP_TRY(c, hipStreamCreateWithFlags(&c->xfer_stream, hipStreamNonBlocking));
    for (auto& slot : c->ring_ev)
        for (auto& e : slot)
            if (!e) HIP_TRY(c, hipEventCreateWithFlags(&e, hipEventDisableTiming));
    hipStream_t xs = c->xfer_stream;
    enum { EV_IN = 0, EV_DONE = 1, EV_OUT = 2 };
    // on ANY failure below: nothing may still be copying into the caller's buffers when we return
    auto bail = [&](int code) { (void)hipStreamSynchronize(xs); (void)hipStreamSynchronize(c->stream); return code; };
#define RING_TRY(expr)                                                                          \
    do { hipError_t e_ = (expr); if (e_ != hipSuccess)                                          \
        return bail(fail(c, DCE_ERR_HIP, "%s failed: %s", #expr, hipGetErrorString(e_))); } while (0)
    auto stage_in = [&](int64_t i) -> int {
        // a sequence chunk needs rows [i0, i0+nb+149): its 149-row halo is copied again (32 KB)
        const int s = (int)(i % RING);
        const int64_t i0 = i * c->max_batch, nb = chunk_rows(i);
        const int64_t lo = i0 * row_floats;
        const int64_t cnt = zscore ? (nb + WIN - 1) * CH : nb * row_floats;
        if (i >= RING) RING_TRY(hipStreamWaitEvent(xs, c->ring_ev[s][EV_DONE], 0));     // slot's previous kernels have read it
        RING_TRY(hipMemcpyAsync(c->d_in + s * in_slot_floats, src + lo, (size_t)cnt * sizeof(float), hipMemcpyHostToDevice, xs));
        RING_TRY(hipEventRecord(c->ring_ev[s][EV_IN], xs));
        return DCE_OK;
    };
    auto stage_out = [&](int64_t i) -> int {
        const int s = (int)(i % RING);
        const int64_t i0 = i * c->max_batch, nb = chunk_rows(i);
        RING_TRY(hipStreamWaitEvent(xs, c->ring_ev[s][EV_DONE], 0));
        if (logits)   RING_TRY(hipMemcpyAsync(logits + i0 * NCLS, c->d_logits + s * mb * NCLS, (size_t)nb * NCLS * sizeof(float), hipMemcpyDeviceToHost, xs));
        if (pred)     RING_TRY(hipMemcpyAsync(pred + i0, c->d_pred + s * mb, (size_t)nb * sizeof(int32_t), hipMemcpyDeviceToHost, xs));
        if (contacts) RING_TRY(hipMemcpyAsync(contacts + i0 * 4, c->d_contacts + s * mb * 4, (size_t)nb * 4, hipMemcpyDeviceToHost, xs));
        if (packed)   RING_TRY(hipMemcpyAsync(packed + i0 * PACKED_ROW, c->d_packed + s * mb * PACKED_ROW, (size_t)nb * PACKED_ROW, hipMemcpyDeviceToHost, xs));
        RING_TRY(hipEventRecord(c->ring_ev[s][EV_OUT], xs));
        return DCE_OK;
    };
    if ((rc = stage_in(0))) return rc;
    for (int64_t i = 0; i < nchunks; ++i) {
        const int s = (int)(i % RING);
        RING_TRY(hipStreamWaitEvent(c->stream, c->ring_ev[s][EV_IN], 0));
        if (i >= RING) RING_TRY(hipStreamWaitEvent(c->stream, c->ring_ev[s][EV_OUT], 0));   // slot's previous results have left
        rc = run_chunk(c, c->d_in + s * in_slot_floats, zscore, chunk_rows(i),
                       logits ? c->d_logits + s * mb * NCLS : nullptr, pred ? c->d_pred + s * mb : nullptr,
                       contacts ? c->d_contacts + s * mb * 4 : nullptr, packed ? c->d_packed + s * mb * PACKED_ROW : nullptr);
        if (rc) return bail(rc);
        RING_TRY(hipEventRecord(c->ring_ev[s][EV_DONE], c->stream));
        if (i + 1 < nchunks && (rc = stage_in(i + 1))) return rc;
        if (i >= 1 && (rc = stage_out(i - 1))) return rc;
    }
    if ((rc = stage_out(nchunks - 1))) return rc;
    RING_TRY(hipStreamSynchronize(xs));
#undef RING_TRY
    return DCE_OK;
}

}  // namespace

extern "C" {

int dce_abi_version(void) { return 2; }

int dce_build_flags(void)
{
    int f = 0;
#if DCE_EXPERIMENTS
    f |= DCE_BUILD_EXPERIMENTS;
#endif
#if defined(DCE_TRACE) && DCE_TRACE
    f |= DCE_BUILD_TRACE;
#endif
#if defined(__SANITIZE_ADDRESS__)
    f |= DCE_BUILD_ASAN;
#elif defined(__has_feature)
#if __has_feature(address_sanitizer)
    f |= DCE_BUILD_ASAN;
#endif
#endif
    return f;
}

int dce_device_count(void)
{
    int n = 0;
    hipError_t e = hipGetDeviceCount(&n);
    if (e != hipSuccess) { fail(nullptr, DCE_ERR_HIP, "hipGetDeviceCount: %s", hipGetErrorString(e)); return DCE_ERR_HIP; }
    return n;
}

int dce_create(dce_ctx** out, int device_id, int64_t max_batch) { return dce_create_ex(out, device_id, max_batch, nullptr); }

int dce_create_ex(dce_ctx** out, int device_id, int64_t max_batch, const char* options)
{
    if (!out || max_batch <= 0 || device_id < 0) return fail(nullptr, DCE_ERR_ARG, "dce_create: bad argument");
    *out = nullptr;
    Tuning parsed;
    {   // the A/B switches: the option string, else DCE_TUNE, over the defaults (one table: kTuneKeys) -- checked before anything else, so
        // that a misspelt option is reported as what it is also on a box without a device
        // DCE_TUNE first, the option string on top of it: a context made with options -- also the empty string a binding passes for "none" -- keeps
        // whatever the user's environment switches that the options do not name
        char msg[256];
        if (!tuning_parse(getenv("DCE_TUNE"), parsed, msg, (int)sizeof msg)) return fail(nullptr, DCE_ERR_ARG, "dce_create: DCE_TUNE: %s", msg);
        if (!tuning_parse(options, parsed, msg, (int)sizeof msg)) return fail(nullptr, DCE_ERR_ARG, "dce_create: %s", msg);
        // the A/B switches were environment variables of their own until round 4 (DCE_GEMM=lockstep, DCE_CONV4=1, ..): a script that still sets one
        // would silently measure the defaults -- say so, once
        static const bool warned = [] {
            for (const char* k : {"DCE_GEMM", "DCE_CONV", "DCE_CONV4", "DCE_X3_PAIR", "DCE_X3_CONV", "DCE_X3_PERSIST", "DCE_X3_PERMK", "DCE_X3_UNFUSED", "DCE_ONLINE_GRAPH",
                                  "DCE_ONLINE_DIRECT", "DCE_FC23", "DCE_GEMV", "DCE_PHASED_MIN_TILES", "DCE_WINO1_MAX", "DCE_BF16_STREAM"})
                if (getenv(k)) fprintf(stderr, "libdce: the environment variable %s is no longer read -- the A/B switches are options of dce_create_ex / keys of DCE_TUNE "
                                               "(\"key=value,key=value\"; the table is kTuneKeys in csrc/dce_api.hip, DESIGN.md appendix)\n", k);
            return true;
        }();
        (void)warned;
    }
    int ndev = 0;
    hipError_t e = hipGetDeviceCount(&ndev);
    if (e != hipSuccess || ndev <= 0)
        return fail(nullptr, DCE_ERR_HIP, "no HIP device available (%s): the HIP path is mandatory, there is no CPU fallback",
                    e == hipSuccess ? "device count 0" : hipGetErrorString(e));
    if (device_id >= ndev) return fail(nullptr, DCE_ERR_ARG, "device %d out of range (%d devices)", device_id, ndev);
    dce_ctx* c = new (std::nothrow) dce_ctx();
    if (!c) return fail(nullptr, DCE_ERR_NOMEM, "out of host memory");
    c->device = device_id;
    c->max_batch = max_batch;
    {
        c->tuning = parsed;
        Tuning& g = c->gate_tuning = c->tuning;                       // the gated DCE_FP32 fallback: two-window conv kernel, tile / phased GEMMs only
        g.gemm_peel = g.conv_peel = false; g.gemv = false;
        g.split_min = 1; g.split_max = 0; g.chain_min = 1; g.chain_max = 0; g.chain_max3 = 0; g.wino1_max = 0;
    }
#define CREATE_TRY(expr)                                                                        \
    do { hipError_t e_ = (expr); if (e_ != hipSuccess) {                                        \
        fail(nullptr, DCE_ERR_HIP, "%s failed: %s", #expr, hipGetErrorString(e_));              \
        dce_destroy(c); return DCE_ERR_HIP; } } while (0)
    DeviceGuard guard(device_id);                        // the caller's current device is put back on return
    CREATE_TRY(guard.err);
    CREATE_TRY(hipStreamCreateWithFlags(&c->own_stream, hipStreamNonBlocking));
    c->stream = c->own_stream;
    (void)roctx();                                       // the marker library, if a tool brought one: resolved here, not on the first hot call
#if DCE_EXPERIMENTS
    CREATE_TRY(init_conv_stack());
#endif
    CREATE_TRY(init_conv_wino());
    CREATE_TRY(init_fc_gemm());
    CREATE_TRY(init_fc_gemm_x3());
    CREATE_TRY(init_conv_x3());
    CREATE_TRY(init_conv_h2());
    CREATE_TRY(init_fc_gemm_h2());
    CREATE_TRY(init_conv_x3p());
    CREATE_TRY(dev_alloc(&c->feat, guard_of(c, 1), (size_t)max_batch * FEAT * sizeof(float)));
    CREATE_TRY(dev_alloc(&c->h1, guard_of(c, 2), (size_t)max_batch * FC1 * sizeof(float)));
    CREATE_TRY(dev_alloc(&c->h2, guard_of(c, 3), (size_t)max_batch * FC2 * sizeof(float)));
    CREATE_TRY(dev_alloc(&c->part, guard_of(c, 4), (size_t)max_batch * 8 * NCLS * sizeof(float)));
    CREATE_TRY(dev_alloc(&c->d_guard, guard_of(c, 9), 4 * sizeof(unsigned)));
    CREATE_TRY(hipMemset(c->d_guard, 0, 4 * sizeof(unsigned)));
    if (c->tuning.latency) {
        // the latency mode's kernel is ONE grid of co-resident workgroups, one per CU: it needs a device with that many CUs to itself
        int cus = 0;
        CREATE_TRY(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device_id));
        if (cus < latency_grid()) {
            fail(nullptr, DCE_ERR_STATE, "latency=1 needs %d CUs (one workgroup each, all resident at once); device %d has %d", latency_grid(), device_id, cus);
            dce_destroy(c); return DCE_ERR_STATE;
        }
        CREATE_TRY(init_latency());
        // what crosses workgroups inside the kernel -- one row of features, h1, h2 and the arrival counters -- lives in FINE-GRAINED device
        // memory (uncached in the XCDs' L2s): the hand-overs then need no cache write-back / invalidate (latency.hip)
        CREATE_TRY(hipExtMallocWithFlags(reinterpret_cast<void**>(&c->lat_x), LAT_X_BYTES, hipDeviceMallocFinegrained));
        c->lat_sync = reinterpret_cast<LatSync*>(c->lat_x + FEAT + 2 * (FC1 + FC2));
        CREATE_TRY(hipMemset(c->lat_x, 0, LAT_X_BYTES));
        if (getenv("DCE_LAT_TRACE")) {                    // debug: wall-clock stamps of the last request's phases, readable by the host (dce_debug_latency_trace)
            CREATE_TRY(hipHostMalloc(reinterpret_cast<void**>(&c->lat_trace), 16 * sizeof(unsigned long long), hipHostMallocMapped | hipHostMallocCoherent));
            memset(c->lat_trace, 0, 16 * sizeof(unsigned long long));
        }
        CREATE_TRY(dev_alloc(&c->lat_hist, guard_of(c, 9), WIN * CH * sizeof(float)));
        CREATE_TRY(dev_alloc(&c->lat_hist_state, guard_of(c, 9), 2 * sizeof(int)));
        CREATE_TRY(hipMemset(c->lat_hist_state, 0, 2 * sizeof(int)));
        CREATE_TRY(hipMemset(c->lat_hist, 0, WIN * CH * sizeof(float)));
        CREATE_TRY(hipHostMalloc(reinterpret_cast<void**>(&c->lat_mbox), sizeof(LatMailbox), hipHostMallocMapped | hipHostMallocCoherent));
        memset(c->lat_mbox, 0, sizeof(LatMailbox));
        CREATE_TRY(hipStreamCreateWithFlags(&c->lat_stream, hipStreamNonBlocking));
        // the micro-batch form: data in ordinary device memory (read through L2 with agent-scope loads), one 64-bit flag per producer in fine-grained memory
        CREATE_TRY(init_latency_mb());
        CREATE_TRY(dev_alloc(&c->lat_mb_feat, guard_of(c, 9), (size_t)LATMB_MAX_N * FEAT * sizeof(float)));
        CREATE_TRY(hipMemset(c->lat_mb_feat, 0, (size_t)LATMB_MAX_N * FEAT * sizeof(float)));
        CREATE_TRY(dev_alloc(&c->lat_mb_h1, guard_of(c, 9), (size_t)LATMB_MAX_N * FC1 * sizeof(float)));
        CREATE_TRY(hipMemset(c->lat_mb_h1, 0, (size_t)LATMB_MAX_N * FC1 * sizeof(float)));
        CREATE_TRY(dev_alloc(&c->lat_mb_plt, guard_of(c, 9), (size_t)32 * LATMB_MAX_N * NCLS * sizeof(float)));
        CREATE_TRY(hipExtMallocWithFlags(reinterpret_cast<void**>(&c->lat_mb_flags), 704 * sizeof(unsigned long long), hipDeviceMallocFinegrained));
        CREATE_TRY(hipMemset(c->lat_mb_flags, 0, 704 * sizeof(unsigned long long)));
        CREATE_TRY(hipDeviceSynchronize());
    }
#undef CREATE_TRY
    *out = c;
    return DCE_OK;
}

void dce_destroy(dce_ctx* c)
{
    if (!c) return;
    DeviceGuard guard(c->device);
    (void)lat_service_stop(c);
    if (c->lat_stream) hipStreamDestroy(c->lat_stream);
    if (c->lat_mbox) hipHostFree(c->lat_mbox);
    dev_free(c->lat_x); dev_free(c->lat_hist); dev_free(c->lat_hist_state);
    dev_free(c->lat_mb_feat); dev_free(c->lat_mb_h1); dev_free(c->lat_mb_plt); dev_free(c->lat_mb_flags);
    if (c->lat_trace) hipHostFree(c->lat_trace);
    if (c->own_stream) hipStreamSynchronize(c->own_stream);
    if (c->stream != c->own_stream) hipStreamSynchronize(c->stream);   // scratch may still be in use there
    for (auto& s : c->spans) { hipEventDestroy(s.a); hipEventDestroy(s.b); }
    for (auto e : c->ev_pool) hipEventDestroy(e);
    (void)dce_comm_destroy(c);
    if (c->comm_stream) hipStreamDestroy(c->comm_stream);
    if (c->comm_ready) hipEventDestroy(c->comm_ready);
    for (auto e : c->comm_done) if (e) hipEventDestroy(e);
    if (c->xstream_ev) hipEventDestroy(c->xstream_ev);
    if (c->xfer_stream) { hipStreamSynchronize(c->xfer_stream); hipStreamDestroy(c->xfer_stream); }
    for (auto& slot : c->ring_ev) for (auto e : slot) if (e) hipEventDestroy(e);
    dev_free(c->d_weights); dev_free(c->feat); dev_free(c->feat3); dev_free(c->h1); dev_free(c->h2); dev_free(c->part);
    dev_free(c->feat_scale); dev_free(c->h1h); dev_free(c->h1_scale); dev_free(c->d_guard); dev_free(c->fc1w_x3_own); dev_free(c->h1p); dev_free(c->f8); dev_free(c->d_in); dev_free(c->d_logits); dev_free(c->d_pred); dev_free(c->d_contacts); dev_free(c->d_packed);
    if (c->online_exec) hipGraphExecDestroy(c->online_exec);
    if (c->online_graph) hipGraphDestroy(c->online_graph);
    dev_free(c->d_ring); dev_free(c->d_online_state);
    if (c->h_online_pin) hipHostFree(c->h_online_pin);
    if (c->own_stream) hipStreamDestroy(c->own_stream);
    delete c;
}

int dce_set_stream(dce_ctx* c, void* hip_stream, int use_own)
{
    if (!c) return DCE_ERR_ARG;
    hipStream_t next = use_own ? c->own_stream : (hipStream_t)hip_stream;
    if (next != c->stream) {
        // the scratch buffers are shared by every call on this ctx: work queued on the new
        // stream must not overtake what is still in flight on the old one
        DEVICE_GUARD(c);
        if (!c->xstream_ev) HIP_TRY(c, hipEventCreateWithFlags(&c->xstream_ev, hipEventDisableTiming));
        HIP_TRY(c, hipEventRecord(c->xstream_ev, c->stream));
        HIP_TRY(c, hipStreamWaitEvent(next, c->xstream_ev, 0));
        c->stream = next;
    }
    return DCE_OK;
}

int dce_load_weight(dce_ctx* c, const char* key, const float* host, const int64_t* shape, int ndim)
{
    if (!c) return DCE_ERR_ARG;
    if (!key || !host || !shape) return fail(c, DCE_ERR_ARG, "dce_load_weight: NULL argument");
    for (int k = 0; k < 14; ++k) {
        if (strcmp(key, kKeys[k].name) != 0) continue;
        if (ndim != kKeys[k].ndim) return fail(c, DCE_ERR_ARG, "%s: expected %d dims, got %d", key, kKeys[k].ndim, ndim);
        size_t count = 1;
        for (int d = 0; d < ndim; ++d) {
            if (shape[d] != kKeys[k].shape[d])
                return fail(c, DCE_ERR_ARG, "%s: dim %d is %lld, expected %lld", key, d, (long long)shape[d], (long long)kKeys[k].shape[d]);
            count *= (size_t)shape[d];
        }
        c->host_w[k].assign(host, host + count);
        c->have[k] = true;
        c->finalized = false;
        return DCE_OK;
    }
    return fail(c, DCE_ERR_KEY, "unexpected state_dict key '%s'", key);
}

int dce_finalize_weights(dce_ctx* c, int precision)
{
    if (!c) return DCE_ERR_ARG;
    if (precision != DCE_FP32 && precision != DCE_BF16_FC && precision != DCE_FP32_SPLIT && precision != DCE_FP32_F16X2 && precision != DCE_FP8_FC)
        return fail(c, DCE_ERR_ARG, "unknown precision %d (0 = fp32, 1 = bf16 FC, 2 = fp32 on three-term bf16 operands, 3 = fp32 tolerance on two-term fp16 operands, 4 = 8-bit FC)", precision);
    const bool bf16_conv = precision == DCE_BF16_FC || precision == DCE_FP8_FC;      // conv stacks that write bf16 features
    for (int k = 0; k < 14; ++k)
        if (!c->have[k]) return fail(c, DCE_ERR_STATE, "missing state_dict key '%s'", kKeys[k].name);
    c->split_alias = false;
#if !DCE_EXPERIMENTS
    // Round 6: the three-term bf16 precision left the product library -- DCE_FP32_F16X2 holds the same contract (fp32 tolerance, argmax exact outside the
    // noise margin) at 1.13 - 2.0 x its speed at every launch size, needs no range guard and no gated fallback (profiles/r6h_retire_split_sweep.txt,
    // profiles/r5_precision_audit.json).  A caller that asks for it gets that precision, and dce_last_plan says so; the kernels themselves live on in the
    // experiments build (libdce_experiments.so).
    if (precision == DCE_FP32_SPLIT) { precision = DCE_FP32_F16X2; c->split_alias = true; }
#endif
    DEVICE_GUARD(c);
    { const int rc = lat_quiesce(c); if (rc) return rc; }
    c->finalized = false;                                  // (until the end: what fails on the way leaves weights of two precisions, or none)
    // a captured online graph holds the old weight pointers / precision: drop it, the next push re-captures
    if (c->online_exec) { hipGraphExecDestroy(c->online_exec); c->online_exec = nullptr; }
    if (c->online_graph) { hipGraphDestroy(c->online_graph); c->online_graph = nullptr; }

    // one host image -> one upload.  Offsets kept 256-B aligned.
    std::vector<float> img;
    auto reserve = [&](size_t floats) { size_t off = (img.size() + 63) & ~size_t(63); img.resize(off + floats); return off; };
    size_t off_w[4], off_ww[4], off_b[4];
    for (int l = 0; l < 4; ++l) {
#if DCE_EXPERIMENTS
        off_w[l] = reserve(conv_pack_floats(l));                      // direct-form pack (conv_stack.hip: experiments build only)
        conv_pack_host(l, c->host_w[2 * l].data(), img.data() + off_w[l]);
#else
        off_w[l] = 0;
#endif
        off_ww[l] = reserve(conv_wino_pack_floats(l));
        conv_wino_pack_host(l, c->host_w[2 * l].data(), img.data() + off_ww[l]);
        off_b[l] = reserve(c->host_w[2 * l + 1].size());
        memcpy(img.data() + off_b[l], c->host_w[2 * l + 1].data(), c->host_w[2 * l + 1].size() * sizeof(float));
    }
    size_t off_fc[6];
    for (int k = 0; k < 6; ++k) {
        const auto& v = c->host_w[8 + k];
        off_fc[k] = reserve(v.size());
        memcpy(img.data() + off_fc[k], v.data(), v.size() * sizeof(float));
    }
    auto to_bf16 = [](const float* v, size_t count, unsigned short* d) {     // round-to-nearest-even; NaN stays NaN
        for (size_t i = 0; i < count; ++i) {
            unsigned u; memcpy(&u, &v[i], 4);
            d[i] = ((u & 0x7fffffffu) > 0x7f800000u) ? (unsigned short)((u >> 16) | 0x40)
                                                     : (unsigned short)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
        }
    };
    // latency mode's micro-batch kernel (latency_mb.hip): fc.0 and fc.3 once more, in the order its lanes hold them
    size_t off_mb1 = 0, off_mb2 = 0;
    const bool want_mb = c->tuning.latency && c->tuning.latency_mb && precision == DCE_FP32;
    if (want_mb) {
        off_mb1 = reserve(latmb_pack_floats(FC1, FEAT)); latmb_pack_host(c->host_w[8].data(), FC1, FEAT, img.data() + off_mb1, 128);
        off_mb2 = reserve(latmb_pack_floats(FC2, FC1));  latmb_pack_host(c->host_w[10].data(), FC2, FC1, img.data() + off_mb2, 0);
    }
    const bool want_cx = precision == DCE_FP32_SPLIT || (bf16_conv && c->tuning.x3_conv);
    const bool want_pair = (want_cx && (c->tuning.x3_pair || c->tuning.x3_permk)) || precision == DCE_FP32_F16X2;      // fc.0's weights once more, K axis in the conv kernels' feature order t' * 128 + c
    std::vector<float> w1p;
    if (want_pair) { w1p.resize(c->host_w[8].size()); fc_perm_k_host(c->host_w[8].data(), FC1, w1p.data()); }
    size_t off_bf[2] = {0, 0}, off_bfp = 0;
    if (precision == DCE_BF16_FC) {
        // bf16 copies of fc.0 / fc.3 weights (round-to-nearest-even), same [out][in] layout
        for (int k = 0; k < 2; ++k) {
            const auto& v = c->host_w[8 + 2 * k];
            off_bf[k] = reserve((v.size() + 1) / 2);
            to_bf16(v.data(), v.size(), reinterpret_cast<unsigned short*>(img.data() + off_bf[k]));
        }
        if (want_pair) {
            off_bfp = reserve((w1p.size() + 1) / 2);
            to_bf16(w1p.data(), w1p.size(), reinterpret_cast<unsigned short*>(img.data() + off_bfp));
        }
    }
    size_t off_x3 = 0, off_x3p = 0, off_x3b = 0, off_cx[4] = {0, 0, 0, 0};
    if (want_cx)
        for (int l = 0; l < 4; ++l) {                     // conv weights as three-term planes, packed per lane (conv_x3.hip)
            off_cx[l] = reserve((conv_x3_pack_halfs(l) + 1) / 2);
            conv_x3_pack_host(l, c->host_w[2 * l].data(), reinterpret_cast<unsigned short*>(img.data() + off_cx[l]));
        }
    if (precision == DCE_FP32_SPLIT) {
        // fc.0's weights as three bf16 planes [3][2048][4736]: w = w1 + w2 + w3 exactly
        const auto& v = c->host_w[8];
        if (!want_pair) {                                 // (with the permuted copy below in use, the reference-order planes -- taps, the A/B routes -- are made on first use: ensure_fc1w_x3)
            off_x3 = reserve((3 * v.size() + 1) / 2);
            split3_host(v.data(), FC1, FEAT, reinterpret_cast<unsigned short*>(img.data() + off_x3));
        }
        if (want_pair) {
            off_x3p = reserve((3 * v.size() + 1) / 2);
            split3_host(w1p.data(), FC1, FEAT, reinterpret_cast<unsigned short*>(img.data() + off_x3p));
        }
        if (!c->feat3) HIP_TRY(c, dev_alloc(&c->feat3, guard_of(c, 7), feat3_halfs(c->max_batch) * sizeof(unsigned short)));
        if (c->tuning.x3_fc3) {                           // fc.3 on three-term operands: its weights as three row-major planes, h1 as three planes out of fc.0
            const auto& v2 = c->host_w[10];
            off_x3b = reserve((3 * v2.size() + 1) / 2);
            split3_rows_host(v2.data(), FC2, FC1, reinterpret_cast<unsigned short*>(img.data() + off_x3b));
            if (!c->h1p) HIP_TRY(c, dev_alloc(&c->h1p, guard_of(c, 8), (size_t)(c->max_batch + 1) * FC1 * 3 * sizeof(unsigned short)));
        }
    }
    // DCE_FP32_F16X2: conv1..4 and fc.0 as two fp16 terms of w * 2^sw (conv_h2.hip has the arithmetic); a non-finite weight or bias refuses the precision
    size_t off_h2[4] = {0, 0, 0, 0}, off_h2fc = 0, off_h2fc2 = 0;
    ConvPackH2 h2pk{};
    int h2_fc_sw = 0, h2_fc2_sw = 0, h2_eW = 0, h2_eB = 0;
    bool h2_bad = false;
    const bool h2_conv_only = bf16_conv && c->tuning.bf16_conv_h2 && want_pair;      // DCE_BF16_FC / DCE_FP8_FC with its conv stack on conv_h2.hip: the conv packs alone
    if (precision == DCE_FP32_F16X2 || h2_conv_only) {
        for (int l = 0; l < 4 && !h2_bad; ++l) {
            const auto& w = c->host_w[2 * l]; const auto& b = c->host_w[2 * l + 1];
            h2pk.sw[l] = h2_weight_shift(w.data(), w.size());
            h2_bad = h2pk.sw[l] == INT_MIN;
            if (!h2_bad) { h2pk.smax[l] = h2_input_smax(b.data(), b.size(), h2pk.sw[l]); h2_bad = h2pk.smax[l] == INT_MIN; }
        }
        if (!h2_bad && !h2_conv_only) { h2_fc_sw = h2_weight_shift(c->host_w[8].data(), c->host_w[8].size()); h2_bad = h2_fc_sw == INT_MIN; }
        for (int k = 9; k < 14; ++k)
            for (float x : c->host_w[k]) h2_bad |= !std::isfinite(x);
        h2pk.smax[4] = 180;                                           // the features: fc.0's bias is added after the scales are taken off (conv_h2.hip H2_SMAX)
        if (!h2_bad) {
            for (int l = 0; l < 4; ++l) {
                off_h2[l] = reserve((conv_h2_pack_halfs(l) + 1) / 2);
                conv_h2_pack_host(l, c->host_w[2 * l].data(), h2pk.sw[l], reinterpret_cast<unsigned short*>(img.data() + off_h2[l]));
            }
            if (!h2_conv_only) {
            off_h2fc = reserve(w1p.size());                           // two halfs per weight
            fc_h2_pack_host(w1p.data(), FC1, FEAT, h2_fc_sw, reinterpret_cast<unsigned short*>(img.data() + off_h2fc));
            }
            if (c->tuning.h2_fc3 && !h2_conv_only) {                                   // fc.3 on two-term operands: its weights likewise; h1's row-scale bound |h1| <= sqrt(K) max|feat| max_n ||W1_n||_2 + max|b1|
                h2_fc2_sw = h2_weight_shift(c->host_w[10].data(), c->host_w[10].size());
                off_h2fc2 = reserve(c->host_w[10].size());
                fc_h2_pack_host(c->host_w[10].data(), FC2, FC1, h2_fc2_sw, reinterpret_cast<unsigned short*>(img.data() + off_h2fc2));
                double wn = 0.0;
                for (int r = 0; r < FC1; ++r) {
                    double q = 0.0;
                    for (int k = 0; k < FEAT; ++k) { const double x = c->host_w[8][(size_t)r * FEAT + k]; q += x * x; }
                    wn = std::max(wn, q);
                }
                const double cw = std::sqrt((double)FEAT) * std::sqrt(wn);
                float bm = 0.f;
                for (float x : c->host_w[9]) bm = std::fmax(bm, std::fabs(x));
                h2_eW = cw > 0.0 ? std::ilogb(cw) + 1 : -300;
                h2_eB = bm > 0.f ? std::ilogb(bm) + 1 : -300;
                const size_t rows = (size_t)c->max_batch + fc_gemm_h2_pad_rows();
                if (!c->h1h) { HIP_TRY(c, dev_alloc(&c->h1h, guard_of(c, 8), rows * FC1 * 2 * sizeof(unsigned short))); HIP_TRY(c, hipMemset(c->h1h, 0, rows * FC1 * 2 * sizeof(unsigned short))); }
                if (!c->h1_scale) { HIP_TRY(c, dev_alloc(&c->h1_scale, guard_of(c, 8), rows * sizeof(int))); HIP_TRY(c, hipMemset(c->h1_scale, 0, rows * sizeof(int))); }
            }
            if (!c->feat3 && !h2_conv_only) {                         // two fp16 terms per feature, padded by a tile of rows (fc_gemm_h2_pad_rows)
                const size_t halfs = feat3_halfs(c->max_batch);
                HIP_TRY(c, dev_alloc(&c->feat3, guard_of(c, 7), halfs * sizeof(unsigned short)));
                HIP_TRY(c, hipMemset(c->feat3, 0, halfs * sizeof(unsigned short)));
            }
            if (!c->feat_scale && !h2_conv_only) HIP_TRY(c, dev_alloc(&c->feat_scale, guard_of(c, 8), (size_t)(c->max_batch + 1) * sizeof(int)));
        }
    }
    if (c->d_weights) { HIP_TRY(c, dev_free(c->d_weights)); c->d_weights = nullptr; }
    HIP_TRY(c, dev_alloc(&c->d_weights, guard_of(c, 0), img.size() * sizeof(float)));
    HIP_TRY(c, hipMemcpy(c->d_weights, img.data(), img.size() * sizeof(float), hipMemcpyHostToDevice));
    for (int l = 0; l < 4; ++l) {
        c->pk.w[l] = DCE_EXPERIMENTS ? c->d_weights + off_w[l] : nullptr; c->pk.ww[l] = c->d_weights + off_ww[l];
        c->pk.b[l] = c->d_weights + off_b[l];
    }
    c->fc1w = c->d_weights + off_fc[0]; c->fc1b = c->d_weights + off_fc[1];
    c->fc2w = c->d_weights + off_fc[2]; c->fc2b = c->d_weights + off_fc[3];
    c->fc3w = c->d_weights + off_fc[4]; c->fc3b = c->d_weights + off_fc[5];
    c->lat_mb_w1 = want_mb ? c->d_weights + off_mb1 : nullptr; c->lat_mb_w2 = want_mb ? c->d_weights + off_mb2 : nullptr;
    c->fc1w_bf16 = precision == DCE_BF16_FC ? c->d_weights + off_bf[0] : nullptr;
    c->fc2w_bf16 = precision == DCE_BF16_FC ? c->d_weights + off_bf[1] : nullptr;
    c->fc1w_bf16p = precision == DCE_BF16_FC && want_pair ? c->d_weights + off_bfp : nullptr;
    for (int l = 0; l < 4; ++l) {
        c->pkx3.w[l] = want_cx ? reinterpret_cast<const unsigned short*>(c->d_weights + off_cx[l]) : nullptr;
        c->pkx3.b[l] = c->pk.b[l];
    }
    if (c->fc1w_x3_own) { HIP_TRY(c, dev_free(c->fc1w_x3_own)); c->fc1w_x3_own = nullptr; }
    c->fc1w_x3 = precision == DCE_FP32_SPLIT && !want_pair ? reinterpret_cast<const unsigned short*>(c->d_weights + off_x3) : nullptr;
    c->fc2w_x3 = precision == DCE_FP32_SPLIT && c->tuning.x3_fc3 ? reinterpret_cast<const unsigned short*>(c->d_weights + off_x3b) : nullptr;
    c->fc1w_x3p = precision == DCE_FP32_SPLIT && want_pair ? reinterpret_cast<const unsigned short*>(c->d_weights + off_x3p) : nullptr;
    c->h2_refused = precision == DCE_FP32_F16X2 && h2_bad;
    c->pkh2 = h2pk;
    for (int l = 0; l < 4; ++l) {
        c->pkh2.w[l] = (precision == DCE_FP32_F16X2 || h2_conv_only) && !h2_bad ? reinterpret_cast<const unsigned short*>(c->d_weights + off_h2[l]) : nullptr;
        c->pkh2.b[l] = c->pk.b[l];
    }
    c->fc1w_h2 = precision == DCE_FP32_F16X2 && !h2_bad ? reinterpret_cast<const unsigned short*>(c->d_weights + off_h2fc) : nullptr;
    c->fc1_sw = h2_fc_sw;
    c->fc2w_h2 = precision == DCE_FP32_F16X2 && !h2_bad && c->tuning.h2_fc3 ? reinterpret_cast<const unsigned short*>(c->d_weights + off_h2fc2) : nullptr;
    c->fc2_sw = h2_fc2_sw; c->fc1_eW = h2_eW; c->fc1_eB = h2_eB;
    c->fc1w_f8 = c->fc1s_f8 = c->fc1w_f8p = c->fc1s_f8p = c->fc2w_f8 = c->fc2s_f8 = nullptr;
    if (precision == DCE_FP8_FC) { const int rc = quantize_weights_f8(c, w1p); if (rc) return rc; }
    c->precision = precision;
    c->guard = dce_ctx::SplitGuard{};
#if DCE_EXPERIMENTS
    if (precision == DCE_FP32_SPLIT) compute_split_guard(c);
#endif
    c->finalized = true;
    return DCE_OK;
}

int dce_forward_windows(dce_ctx* c, const float* windows, int64_t n, int on_device,
                        float* logits, int32_t* pred, uint8_t* contacts)
{
    RoctxRange range_("dce_forward_windows");
    int rc = check_ready_quiet(c);
    if (rc) return rc;
    DEVICE_GUARD(c);
    if (n < 0 || (n > 0 && !windows)) return fail(c, DCE_ERR_ARG, "dce_forward_windows: bad argument");
    if (n == 0) return DCE_OK;
    return run_all(c, windows, 0, n, n * WIN * CH, on_device, logits, pred, contacts);
}

int dce_infer_sequence(dce_ctx* c, const float* seq, int64_t T, int window, int on_device,
                       float* logits, int32_t* pred, uint8_t* contacts)
{
    RoctxRange range_("dce_infer_sequence");
    int rc = check_ready_quiet(c);
    if (rc) return rc;
    DEVICE_GUARD(c);
    if (window != WIN) return fail(c, DCE_ERR_ARG, "window_size must be %d (the model hard-codes 4736 = 128*37), got %d", WIN, window);
    if (T < 0 || (T > 0 && !seq)) return fail(c, DCE_ERR_ARG, "dce_infer_sequence: bad argument");
    const int64_t n = T - WIN + 1;
    if (n <= 0) return DCE_OK;        // contact_dataset.__len__ <= 0: nothing to do
    return run_all(c, seq, 1, n, T * CH, on_device, logits, pred, contacts);
}

int dce_forward_windows_packed(dce_ctx* c, const float* windows, int64_t n, int on_device, uint8_t* packed)
{
    RoctxRange range_("dce_forward_windows_packed");
    int rc = check_ready_quiet(c);
    if (rc) return rc;
    DEVICE_GUARD(c);
    if (n < 0 || (n > 0 && (!windows || !packed))) return fail(c, DCE_ERR_ARG, "dce_forward_windows_packed: bad argument");
    if (on_device && misaligned4(packed)) return fail(c, DCE_ERR_ARG, "dce_forward_windows_packed: device `packed` must be 4-byte aligned");
    if (n == 0) return DCE_OK;
    return run_all(c, windows, 0, n, n * WIN * CH, on_device, nullptr, nullptr, nullptr, packed);
}

int dce_infer_sequence_packed(dce_ctx* c, const float* seq, int64_t T, int window, int on_device, uint8_t* packed)
{
    RoctxRange range_("dce_infer_sequence_packed");
    int rc = check_ready_quiet(c);
    if (rc) return rc;
    DEVICE_GUARD(c);
    if (window != WIN) return fail(c, DCE_ERR_ARG, "window_size must be %d (the model hard-codes 4736 = 128*37), got %d", WIN, window);
    const int64_t n = T - WIN + 1;
    if (T < 0 || (n > 0 && (!seq || !packed))) return fail(c, DCE_ERR_ARG, "dce_infer_sequence_packed: bad argument");
    if (on_device && misaligned4(packed)) return fail(c, DCE_ERR_ARG, "dce_infer_sequence_packed: device `packed` must be 4-byte aligned");
    if (n <= 0) return DCE_OK;
    return run_all(c, seq, 1, n, T * CH, on_device, nullptr, nullptr, nullptr, packed);
}

int dce_unpack_results(dce_ctx* c, const uint8_t* packed, int64_t n, int on_device,
                       float* logits, int32_t* pred, uint8_t* contacts)
{
    if (n < 0 || (n > 0 && !packed) || (on_device && !c)) return fail(c, DCE_ERR_ARG, "dce_unpack_results: bad argument");
    if (on_device && misaligned4(packed)) return fail(c, DCE_ERR_ARG, "dce_unpack_results: device `packed` must be 4-byte aligned");
    if (n == 0) return DCE_OK;
    if (on_device) {
        DEVICE_GUARD(c);
        { const int rc = lat_quiesce(c); if (rc) return rc; }       // (every device-touching entry point: the latency mode's resident kernel leaves first)
        HIP_TRY(c, launch_unpack_results(packed, n, logits, pred, contacts, c->stream));
        return DCE_OK;
    }
    // host rows: plain byte work, no device involved (a row is 16 little-endian fp32 + 4 bits)
    for (int64_t i = 0; i < n; ++i) {
        const uint8_t* r = packed + i * PACKED_ROW;
        if (logits) memcpy(logits + i * NCLS, r, NCLS * sizeof(float));
        if (contacts) memcpy(contacts + i * 4, r + 4 * NCLS, 4);
        if (pred) pred[i] = (r[64] & 1) << 3 | (r[65] & 1) << 2 | (r[66] & 1) << 1 | (r[67] & 1);
    }
    return DCE_OK;
}

int dce_zscore_windows(dce_ctx* c, const float* seq, int64_t T, int64_t first, int64_t n,
                       int on_device, float* windows_out)
{
    if (!c) return DCE_ERR_ARG;
    DEVICE_GUARD(c);
    if (first < 0 || n < 0 || first + n + WIN - 1 > T || !seq || !windows_out)
        return fail(c, DCE_ERR_ARG, "dce_zscore_windows: windows [%lld,%lld) out of range for T=%lld",
                    (long long)first, (long long)(first + n), (long long)T);
    if (n == 0) return DCE_OK;
    { const int rc = lat_quiesce(c); if (rc) return rc; }
    if (on_device) {
        HIP_TRY(c, launch_zscore_windows(seq + first * CH, n, windows_out, c->stream));
        return DCE_OK;
    }
    const size_t in_floats = (size_t)(n + WIN - 1) * CH, out_floats = (size_t)n * WIN * CH;
    int rc = ensure_in(c, (in_floats + out_floats) * sizeof(float));
    if (rc) return rc;
    float* dout = c->d_in + in_floats;
    HIP_TRY(c, hipMemcpyAsync(c->d_in, seq + first * CH, in_floats * sizeof(float), hipMemcpyHostToDevice, c->stream));
    HIP_TRY(c, launch_zscore_windows(c->d_in, n, dout, c->stream));
    HIP_TRY(c, hipMemcpyAsync(windows_out, dout, out_floats * sizeof(float), hipMemcpyDeviceToHost, c->stream));
    HIP_TRY(c, hipStreamSynchronize(c->stream));
    return DCE_OK;
}

int dce_forward_taps(dce_ctx* c, const float* windows, int64_t n, int on_device,
                     void* feat, void* h1, float* h2, float* logits)
{
    int rc = check_ready_quiet(c);
    if (rc) return rc;
    DEVICE_GUARD(c);
    if (n <= 0 || n > c->max_batch || !windows)
        return fail(c, DCE_ERR_ARG, "dce_forward_taps: need 0 < n <= max_batch (%lld)", (long long)c->max_batch);
    if (c->precision == DCE_FP8_FC && (feat || h1))
        return fail(c, DCE_ERR_STATE, "dce_forward_taps: features and h1 are e4m3 with scales in DCE_FP8_FC: h2 and logits only");
    const float* dsrc = windows;
    float* dl = logits;
    if (!on_device) {
        rc = ensure_in(c, (size_t)n * WIN * CH * sizeof(float));
        if (rc) return rc;
        rc = ensure_out(c, (size_t)n);
        if (rc) return rc;
        HIP_TRY(c, hipMemcpyAsync(c->d_in, windows, (size_t)n * WIN * CH * sizeof(float), hipMemcpyHostToDevice, c->stream));
        dsrc = c->d_in; dl = c->d_logits;
    }
    c->want_h2 = h2 != nullptr;
    c->want_feat = feat != nullptr;
    c->want_h1 = h1 != nullptr;
    rc = run_chunk(c, dsrc, 0, n, dl, nullptr, nullptr);
    c->want_h2 = c->want_feat = c->want_h1 = false;
    if (rc) return rc;
    const hipMemcpyKind kind = on_device ? hipMemcpyDeviceToDevice : hipMemcpyDeviceToHost;
    // DCE_BF16_FC: the features and ReLU(fc.0) ARE bf16 in that mode -- the taps hand out the (n,4736) / (n,2048)
    // uint16 bit patterns the next layer consumed
    const size_t es = c->precision == DCE_BF16_FC ? 2 : sizeof(float);
    if (feat) HIP_TRY(c, hipMemcpyAsync(feat, c->feat, (size_t)n * FEAT * es, kind, c->stream));
    if (h1)   HIP_TRY(c, hipMemcpyAsync(h1, c->h1, (size_t)n * FC1 * es, kind, c->stream));
    if (h2)   HIP_TRY(c, hipMemcpyAsync(h2, c->h2, (size_t)n * FC2 * sizeof(float), kind, c->stream));
    if (!on_device) {
        if (logits) HIP_TRY(c, hipMemcpyAsync(logits, dl, (size_t)n * NCLS * sizeof(float), hipMemcpyDeviceToHost, c->stream));
        HIP_TRY(c, hipStreamSynchronize(c->stream));
    }
    return DCE_OK;
}

int dce_conv_layer_taps(dce_ctx* c, const float* windows, int64_t n, int kernel,
                        float* conv1, float* conv2, float* pool1, float* conv3, float* conv4, float* feat)
{
    int rc = check_ready_quiet(c);
    if (rc) return rc;
    DEVICE_GUARD(c);
    if (n <= 0 || n > c->max_batch || n > 64 || !windows || !conv1 || !conv2 || !pool1 || !conv3 || !conv4 || !feat)
        return fail(c, DCE_ERR_ARG, "dce_conv_layer_taps: need 0 < n <= min(64, max_batch) host windows and all six host outputs");
    if (kernel == 7 && c->precision != DCE_FP32_SPLIT)
        return fail(c, DCE_ERR_STATE, "dce_conv_layer_taps: kernel 7 (conv_x3) needs a context finalised with DCE_FP32_SPLIT");
    if (kernel == 8 && (c->precision != DCE_FP32_F16X2 || c->h2_refused))
        return fail(c, DCE_ERR_STATE, "dce_conv_layer_taps: kernel 8 (conv_h2) needs a context finalised with DCE_FP32_F16X2 (and a finite checkpoint)");
    if (c->precision == DCE_BF16_FC || c->precision == DCE_FP8_FC)
        return fail(c, DCE_ERR_STATE, "dce_conv_layer_taps: not available in DCE_BF16_FC / DCE_FP8_FC (its conv stack is the fp32 / three-term one: tap a DCE_FP32 or DCE_FP32_SPLIT context)");
    TuningScope tuning_scope(&c->tuning);                 // the launchers below read this context's switches, not the process defaults
    // host pointers only (a test hook): stage the windows, run ONE named kernel family with its taps on, copy everything out
    const size_t in_f = (size_t)n * WIN * CH;
    const size_t sz[5] = {(size_t)n * 64 * 150, (size_t)n * 64 * 150, (size_t)n * 64 * 75, (size_t)n * 128 * 75, (size_t)n * 128 * 75};
    size_t total = in_f;
    for (size_t s : sz) total += s;
    rc = ensure_in(c, total * sizeof(float));
    if (rc) return rc;
    float* d = c->d_in;
    LayerTaps taps{d + in_f, d + in_f + sz[0], d + in_f + sz[0] + sz[1], d + in_f + sz[0] + sz[1] + sz[2],
                   d + in_f + sz[0] + sz[1] + sz[2] + sz[3]};
    HIP_TRY(c, hipMemcpyAsync(d, windows, in_f * sizeof(float), hipMemcpyHostToDevice, c->stream));
    HIP_TRY(c, hipMemsetAsync(d + in_f, 0xff, (total - in_f) * sizeof(float), c->stream));      // untouched taps read back as NaN
    const hipError_t e = kernel == 8 ? launch_conv_h2_taps(d, n, c->pkh2, c->feat3, c->feat_scale, c->feat, taps, c->stream)
                       : kernel == 7 ? launch_conv_x3_taps(d, n, c->pkx3, c->feat3, c->feat, taps, c->stream)
                                     : launch_conv_taps(kernel, d, n, c->pk, c->feat, taps, c->stream);
    if (e != hipSuccess) return fail(c, e == hipErrorInvalidValue ? DCE_ERR_ARG : DCE_ERR_HIP, "dce_conv_layer_taps: kernel %d: %s", kernel, hipGetErrorString(e));
    float* outs[5] = {conv1, conv2, pool1, conv3, conv4};
    float* srcs[5] = {taps.conv1, taps.conv2, taps.pool1, taps.conv3, taps.conv4};
    for (int i = 0; i < 5; ++i) HIP_TRY(c, hipMemcpyAsync(outs[i], srcs[i], sz[i] * sizeof(float), hipMemcpyDeviceToHost, c->stream));
    HIP_TRY(c, hipMemcpyAsync(feat, c->feat, (size_t)n * FEAT * sizeof(float), hipMemcpyDeviceToHost, c->stream));
    HIP_TRY(c, hipStreamSynchronize(c->stream));
    return DCE_OK;
}

int dce_features(dce_ctx* c, const float* src, int64_t n, int zscore, void* feat)
{
    int rc = check_ready_quiet(c);
    if (rc) return rc;
    DEVICE_GUARD(c);
    if (c->precision != DCE_BF16_FC && c->precision != DCE_FP8_FC) return fail(c, DCE_ERR_STATE, "dce_features: bf16 features need a context finalized with DCE_BF16_FC or DCE_FP8_FC");
    if (!c->pkx3.w[0]) return fail(c, DCE_ERR_STATE, "dce_features: the option x3_conv=0 leaves out the conv kernels it runs");
    if (n < 0 || (n && (!src || !feat)) || (reinterpret_cast<uintptr_t>(feat) & 15)) return fail(c, DCE_ERR_ARG, "dce_features: need n >= 0 and 16-byte aligned features");
    TuningScope tuning_scope(&c->tuning);
    struct PlanScope { explicit PlanScope(std::vector<const char*>* p) { p->clear(); t_plan = p; } ~PlanScope() { t_plan = nullptr; } } plan_scope(&c->plan);
    const int64_t row = zscore ? CH : (int64_t)WIN * CH;
    for (int64_t i = 0; i < n; i += c->max_batch) {                   // (as run_all cuts a call: a launch's size decides its kernel)
        const int64_t m = n - i < c->max_batch ? n - i : c->max_batch;
        unsigned short* out = static_cast<unsigned short*>(feat) + (size_t)i * FEAT;
        if (m >= plan_threshold(c->tuning, T_BF16H2) && c->tuning.bf16_conv_h2 && c->pkh2.w[0]) HIP_TRY(c, launch_conv_h2_bf16(src + i * row, zscore, m, c->pkh2, out, c->stream));
        else HIP_TRY(c, launch_conv_x3_bf16(src + i * row, zscore, m, c->pkx3, out, c->stream, 1, DCE_EXPERIMENTS ? c->tuning.x3_bf16_terms : 2, nullptr));
    }
    return DCE_OK;
}

int dce_confusion_counts(dce_ctx* c, const int32_t* pred, const int64_t* labels, int64_t n,
                         int on_device, int64_t* counts)
{
    if (!c) return DCE_ERR_ARG;
    if (n < 0 || !counts || (n > 0 && (!pred || !labels))) return fail(c, DCE_ERR_ARG, "dce_confusion_counts: bad argument");
    DEVICE_GUARD(c);
    if (n == 0) return DCE_OK;
    { const int rc = lat_quiesce(c); if (rc) return rc; }
    if (on_device) {
        HIP_TRY(c, launch_confusion16(pred, labels, n, reinterpret_cast<unsigned long long*>(counts), c->stream));
        return DCE_OK;
    }
    const size_t pb = (size_t)n * sizeof(int32_t), lb = (size_t)n * sizeof(int64_t), cb = 256 * sizeof(int64_t);
    const size_t lo = (pb + 255) & ~size_t(255), co = lo + ((lb + 255) & ~size_t(255));
    int rc = ensure_in(c, co + cb);
    if (rc) return rc;
    char* base = reinterpret_cast<char*>(c->d_in);
    HIP_TRY(c, hipMemcpyAsync(base, pred, pb, hipMemcpyHostToDevice, c->stream));
    HIP_TRY(c, hipMemcpyAsync(base + lo, labels, lb, hipMemcpyHostToDevice, c->stream));
    HIP_TRY(c, hipMemcpyAsync(base + co, counts, cb, hipMemcpyHostToDevice, c->stream));
    HIP_TRY(c, launch_confusion16(reinterpret_cast<int32_t*>(base), reinterpret_cast<int64_t*>(base + lo), n,
                                  reinterpret_cast<unsigned long long*>(base + co), c->stream));
    HIP_TRY(c, hipMemcpyAsync(counts, base + co, cb, hipMemcpyDeviceToHost, c->stream));
    HIP_TRY(c, hipStreamSynchronize(c->stream));
    return DCE_OK;
}

int dce_online_reset(dce_ctx* c)
{
    if (!c) return DCE_ERR_ARG;
    if (c->lat_mbox) {
        DEVICE_GUARD(c);
        const int rc = lat_quiesce(c);
        if (rc) return rc;
        HIP_TRY(c, hipMemset(c->lat_hist_state, 0, 2 * sizeof(int)));
        c->lat_count = 0;
        c->lat_mbox->a.tag = c->lat_mbox->b.tag = 0;
    }
    c->ring_rows = 0;
    c->online_seq = 0;
    c->online_state_dirty = true;
    if (c->h_online_pin) reinterpret_cast<unsigned*>(c->h_online_pin + 32)[0] = 0;
    return DCE_OK;
}

namespace {

// pinned block: [0,16) logits | [16] pred | [17] contacts | [32] completion flag | [40,94) the incoming sample
constexpr int PIN_FLAG = 32, PIN_SAMPLE = 40, PIN_FLOATS = 96;


int online_wait(dce_ctx* c, unsigned expect)
{
    unsigned* flag = reinterpret_cast<unsigned*>(c->h_online_pin + PIN_FLAG);
    const auto t0 = std::chrono::steady_clock::now();
    for (unsigned spins = 0; __atomic_load_n(flag, __ATOMIC_ACQUIRE) != expect; ++spins) {
        DCE_CPU_RELAX();
        if ((spins & 0xfff) == 0xfff && std::chrono::steady_clock::now() - t0 > std::chrono::milliseconds(50)) {
            HIP_TRY(c, hipStreamSynchronize(c->stream));         // something is wrong or very slow: fall back
            if (__atomic_load_n(flag, __ATOMIC_ACQUIRE) != expect)
                return fail(c, DCE_ERR_HIP, "dce_online_push: the result never arrived");
            break;
        }
    }
    return DCE_OK;
}

// The kernels of one push with CONSTANT launch parameters (what the graph captures): append the
// sample waiting in pinned memory, run the path on the window the device-side cursor points at,
// publish the estimate and the next sequence number to pinned memory.
int online_enqueue(dce_ctx* c)
{
    HIP_TRY(c, launch_online_append_state(c->d_ring, c->d_online_state, c->h_online_pin + PIN_SAMPLE, c->stream));
    const int period = c->prof_period;
    c->prof_period = 0;                                  // no event records inside the (captured) sequence
    c->src_row_dev = &c->d_online_state->src_row;
    c->seq_counter_dev = &c->d_online_state->seq;
    c->done_flag = reinterpret_cast<unsigned*>(c->h_online_pin + PIN_FLAG);
    const int rc = run_chunk(c, c->d_ring, 1, 1, c->h_online_pin, reinterpret_cast<int32_t*>(c->h_online_pin + 16),
                             reinterpret_cast<uint8_t*>(c->h_online_pin + 17));
    c->src_row_dev = nullptr; c->seq_counter_dev = nullptr; c->done_flag = nullptr;
    c->prof_period = period;
    return rc;
}

// online_graph=1: capture online_enqueue once; later pushes are one hipGraphLaunch.  Opt-in:
// measured on MI355X / ROCm 7.2 (three alternating runs of tests/c/abi_client.c) the graph launch
// costs 90.1 us per push against 89.1 us for the same five kernels launched one by one -- the
// launches already hide behind the first kernel -- so plain launches are the default.  Any capture failure (e.g. a caller stream that cannot be captured)
// leaves online_exec null and the push falls back to plain launches.
void online_build_graph(dce_ctx* c)
{
    if (c->online_exec || !c->tuning.online_graph) return;
    if (hipStreamBeginCapture(c->stream, hipStreamCaptureModeThreadLocal) != hipSuccess) { (void)hipGetLastError(); return; }
    const int rc = online_enqueue(c);
    hipGraph_t g = nullptr;
    const hipError_t e = hipStreamEndCapture(c->stream, &g);
    if (rc != DCE_OK || e != hipSuccess || !g) { if (g) hipGraphDestroy(g); (void)hipGetLastError(); return; }
    hipGraphExec_t x = nullptr;
    if (hipGraphInstantiate(&x, g, nullptr, nullptr, 0) != hipSuccess) { hipGraphDestroy(g); (void)hipGetLastError(); return; }
    c->online_graph = g;
    c->online_exec = x;
}

// dce_online_push in the latency mode: the sample goes to the mailbox of the resident kernel (started on the first push, and again
// after it left for want of samples), the estimate comes back through the same mailbox: no launch, no copy, no stream operation.
int lat_push(dce_ctx* c, const float* sample, float* logits, int32_t* pred, uint8_t* contacts)
{
    int rc = lat_check_error(c);
    if (rc) return rc;
    LatMailbox* mb = c->lat_mbox;
    const bool estimate = c->lat_count + 1 >= WIN;
    for (int attempt = 0;; ++attempt) {
        if (c->lat_running && !__atomic_load_n(&mb->alive, __ATOMIC_ACQUIRE)) {      // it left for want of samples (latency_idle_ms): start it again
            HIP_TRY(c, hipStreamSynchronize(c->lat_stream));
            c->lat_running = false;
        }
        if (!c->lat_running && (rc = lat_service_start(c))) return rc;
        memcpy(mb->sample, sample, CH * sizeof(float));
        mb->kind = estimate ? 1u : 0u;
        const unsigned req = ++c->lat_req;
        __atomic_store_n(&mb->req, req, __ATOMIC_RELEASE);
        const unsigned want_done = c->online_seq + 1;
        const auto t0 = std::chrono::steady_clock::now();
        bool dead = false;
        for (unsigned spins = 0;; ++spins) {
            if (estimate ? (__atomic_load_n(&mb->a.tag, __ATOMIC_ACQUIRE) == want_done && __atomic_load_n(&mb->b.tag, __ATOMIC_ACQUIRE) == want_done)
                         : [&] { for (unsigned& a : mb->ack) if (__atomic_load_n(&a, __ATOMIC_ACQUIRE) != req) return false; return true; }()) break;
            DCE_CPU_RELAX();
            if ((spins & 0x3ff) != 0x3ff) continue;
            if (__atomic_load_n(&mb->error, __ATOMIC_ACQUIRE)) return lat_check_error(c);
            if (!__atomic_load_n(&mb->alive, __ATOMIC_ACQUIRE) && __atomic_load_n(&mb->ack[0], __ATOMIC_ACQUIRE) != req) { dead = true; break; }   // it left before it saw this request
            if (std::chrono::steady_clock::now() - t0 > std::chrono::milliseconds(200)) {
                (void)lat_service_stop(c);
                return fail(c, DCE_ERR_HIP, "dce_online_push (latency mode): no answer from the service kernel within 200 ms");
            }
        }
        if (!dead) break;
        HIP_TRY(c, hipStreamSynchronize(c->lat_stream));
        c->lat_running = false;
        if (attempt >= 2) return fail(c, DCE_ERR_HIP, "dce_online_push (latency mode): the service kernel keeps leaving before it takes a request");
    }
    if (c->lat_count < WIN) c->lat_count += 1;
    if (!estimate) return 0;
    c->online_seq += 1;
    if (logits) { memcpy(logits, mb->a.logits, 15 * sizeof(float)); logits[15] = mb->b.logit15; }
    if (pred) *pred = mb->b.pred;
    if (contacts) memcpy(contacts, mb->b.contacts, 4);
    return 1;
}

}  // namespace

int dce_online_push(dce_ctx* c, const float* sample, float* logits, int32_t* pred, uint8_t* contacts)
{
    RoctxRange range_("dce_online_push");
    int rc = check_ready(c);
    if (rc) return rc;
    DEVICE_GUARD(c);
    if (!sample) return fail(c, DCE_ERR_ARG, "dce_online_push: NULL sample");
    if (c->tuning.latency && c->precision == DCE_FP32) return lat_push(c, sample, logits, pred, contacts);
    if (!c->d_ring) {
        HIP_TRY(c, dev_alloc(&c->d_ring, guard_of(c, 10), (size_t)ONLINE_ROWS * CH * sizeof(float)));
        HIP_TRY(c, dev_alloc(&c->d_online_state, guard_of(c, 10), sizeof(OnlineState)));
        HIP_TRY(c, hipHostMalloc(reinterpret_cast<void**>(&c->h_online_pin), PIN_FLOATS * sizeof(float), hipHostMallocMapped | hipHostMallocCoherent));   // polled by the host while a kernel writes it: must be coherent (fine-grained), whatever the defaults / HIP_HOST_COHERENT say
        memset(c->h_online_pin, 0, PIN_FLOATS * sizeof(float));
        // constant-parameter (graph) form needs the Winograd kernels' indirect window start
        c->online_mode = (!(DCE_EXPERIMENTS && c->tuning.conv_direct) && !c->tuning.online_direct) ? 1 : 0;
    }
    float* hl = c->h_online_pin;
    int32_t* hp = reinterpret_cast<int32_t*>(c->h_online_pin + 16);
    uint8_t* hc = reinterpret_cast<uint8_t*>(c->h_online_pin + 17);
    unsigned expect = 0;

    if (c->online_mode == 1) {
        // ---- one graph launch per sample; host and device advance the same cursor
        if (c->online_state_dirty) {
            HIP_TRY(c, hipMemsetAsync(c->d_online_state, 0, sizeof(OnlineState), c->stream));
            c->online_state_dirty = false;
        }
        memcpy(c->h_online_pin + PIN_SAMPLE, sample, CH * sizeof(float));
        if (c->ring_rows == ONLINE_ROWS) c->ring_rows = WIN - 1;       // the append kernel compacts
        c->ring_rows += 1;
        if (c->ring_rows < WIN) {                                      // still filling: append only
            HIP_TRY(c, launch_online_append_state(c->d_ring, c->d_online_state, c->h_online_pin + PIN_SAMPLE, c->stream));
            HIP_TRY(c, hipStreamSynchronize(c->stream));               // the pinned sample is free again
            return 0;
        }
        expect = ++c->online_seq;
        if (!c->online_exec) online_build_graph(c);
        if (c->online_exec) HIP_TRY(c, hipGraphLaunch(c->online_exec, c->stream));
        else if ((rc = online_enqueue(c))) return rc;
    } else {
        // ---- plain launches with per-push parameters (online_direct=1; the experiments build's direct-form conv)
        if (c->ring_rows == ONLINE_ROWS) {              // keep the last 149 rows, restart at the front
            HIP_TRY(c, hipMemcpyAsync(c->d_ring, c->d_ring + (ONLINE_ROWS - (WIN - 1)) * CH,
                                      (WIN - 1) * CH * sizeof(float), hipMemcpyDeviceToDevice, c->stream));
            c->ring_rows = WIN - 1;
        }
        // the sample rides in the kernel arguments of a one-wave append kernel (no H2D copy)
        OnlineSample s;
        memcpy(s.v, sample, CH * sizeof(float));
        HIP_TRY(c, launch_online_append(c->d_ring + c->ring_rows * CH, s, c->stream));
        c->ring_rows += 1;
        if (c->ring_rows < WIN) return 0;
        c->done_flag = reinterpret_cast<unsigned*>(c->h_online_pin + PIN_FLAG);
        expect = c->done_seq = ++c->online_seq;
        rc = run_chunk(c, c->d_ring + (c->ring_rows - WIN) * CH, 1, 1, hl, hp, hc);
        c->done_flag = nullptr;
        if (rc) return rc;
    }
    // The tail kernel wrote the estimate straight into pinned host memory, then the sequence number
    // this thread polls: no D2H copy and no stream synchronisation on the latency path.
    if ((rc = online_wait(c, expect))) return rc;
    if (logits) memcpy(logits, hl, NCLS * sizeof(float));
    if (pred) memcpy(pred, hp, sizeof(int32_t));
    if (contacts) memcpy(contacts, hc, 4);
    return 1;
}

int dce_split_guard_info(dce_ctx* c, dce_split_guard* out)
{
    if (!c || !out) return DCE_ERR_ARG;
    DEVICE_GUARD(c);
    memset(out, 0, sizeof *out);
    out->precision = c->precision;
    out->enabled = c->finalized && c->precision == DCE_FP32_SPLIT && c->tuning.split_guard;
    out->refused = c->guard.refused;
    out->x_hi = c->guard.x_hi; out->x_lo = c->guard.x_lo;
    out->z_max = (float)(149.0 / std::sqrt(150.0));
    for (int l = 0; l < 6; ++l) { out->gain[l] = c->guard.gain[l]; out->offs[l] = c->guard.offs[l]; }
    snprintf(out->reason, sizeof out->reason, "%s", c->split_alias ? "DCE_FP32_SPLIT runs DCE_FP32_F16X2 in this library (no range guard needed); the three-term kernels and their guard live in libdce_experiments.so"
                                                                : c->guard.reason.c_str());
    unsigned w[4] = {0, 0, 0, 0};
    HIP_TRY(c, hipStreamSynchronize(c->stream));
    HIP_TRY(c, hipMemcpy(w, c->d_guard, sizeof w, hipMemcpyDeviceToHost));
    out->guarded_launches = c->guard_launches;
    out->windows_out_of_range = w[1];
    out->fallbacks_run = w[2];
    return DCE_OK;
}

int dce_profile_enable(dce_ctx* c, int on)
{
    if (!c || on < 0) return DCE_ERR_ARG;
    c->prof_period = on;
    c->prof_tick = 0;
    c->prof = false;
    return DCE_OK;
}

int dce_profile_read(dce_ctx* c, double ms[DCE_PROFILE_SLOTS], int64_t launches[DCE_PROFILE_SLOTS], int reset)
{
    if (!c) return DCE_ERR_ARG;
    DEVICE_GUARD(c);
    int rc = drain_spans(c);
    if (rc) return rc;
    for (int s = 0; s < DCE_PROFILE_SLOTS; ++s) {
        if (ms) ms[s] = c->prof_ms[s];
        if (launches) launches[s] = c->prof_n[s];
        if (reset) { c->prof_ms[s] = 0; c->prof_n[s] = 0; }
    }
    return DCE_OK;
}

int dce_last_plan(dce_ctx* c, char* out, int out_len)
{
    if (!c || !out || out_len <= 0) return DCE_ERR_ARG;
    std::string s;
    for (const char* k : c->plan) { if (!s.empty()) s += ' '; s += k; }
    snprintf(out, (size_t)out_len, "%s", s.c_str());
    return DCE_OK;
}

int dce_sync(dce_ctx* c)
{
    if (!c) return DCE_ERR_ARG;
    DEVICE_GUARD(c);
    HIP_TRY(c, hipStreamSynchronize(c->stream));
    if (c->lat_mbox && !c->lat_running) return lat_check_error(c);
    return DCE_OK;
}

int dce_debug_latency_trace(dce_ctx* c, unsigned long long out[16])
{
    if (!c || !out || !c->lat_trace) return DCE_ERR_STATE;
    for (int i = 0; i < 16; ++i) out[i] = __atomic_load_n(&c->lat_trace[i], __ATOMIC_RELAXED);
    if (c->lat_mb_flags) {
        // the micro-batch kernel's fc.0 weight stream: [12] the earliest request, [13] the latest landing over its 128 tiles (38.8 MB between the two)
        DEVICE_GUARD(c);
        HIP_TRY(c, hipStreamSynchronize(c->stream));
        unsigned long long st[256];
        HIP_TRY(c, hipMemcpy(st, c->lat_mb_flags + 320, sizeof st, hipMemcpyDeviceToHost));
        unsigned long long lo = ~0ull, hi = 0;
        for (int i = 0; i < 128; ++i) { if (st[i] < lo) lo = st[i]; if (st[128 + i] > hi) hi = st[128 + i]; }
        out[12] = lo; out[13] = hi;
    }
    return DCE_OK;
}

}  // extern "C"
// (for dce_comm.hip: the exchange entry points quiesce the latency mode's resident kernel like every other device-touching call)
int dce_internal_quiesce(dce_ctx* c) { return lat_quiesce(c); }
extern "C" {

int dce_debug_alloc(dce_ctx* c, size_t bytes, void** out)
{
    if (!c || !out) return DCE_ERR_ARG;
    DEVICE_GUARD(c);
    HIP_TRY(c, dev_alloc_raw(out, bytes, c->tuning.guard_alloc));
    return DCE_OK;
}

int dce_debug_free(dce_ctx* c, void* p)
{
    if (!c) return DCE_ERR_ARG;
    DEVICE_GUARD(c);
    HIP_TRY(c, dev_free_raw(p));
    return DCE_OK;
}

const char* dce_last_error(dce_ctx* c) { return c ? c->err.c_str() : g_create_error.c_str(); }

}  // extern "C"
