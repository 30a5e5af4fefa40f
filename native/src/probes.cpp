// Node-validation probes (N1 gpuinfo, N4 HBM write, N5 MD5 tree, N7 copy/xGMI). Host code;
// compiled with hipcc and linked against the kernels in stream_kernels.hip / md5_kernels.hip.
#include "tk8s/probes.h"

#include <algorithm>
#include <chrono>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <map>
#include <memory>
#include <mutex>
#include <utility>
#include <vector>

#include "tk8s/common.h"

namespace tk8s {

namespace {

std::string hex(const unsigned char* p, size_t n) {
  static const char* d = "0123456789abcdef";
  std::string s;
  for (size_t i = 0; i < n; ++i) {
    s += d[p[i] >> 4];
    s += d[p[i] & 15];
  }
  return s;
}

std::string link_type_name(uint32_t t) {
  switch (t) {
    case 0: return "hypertransport";
    case 1: return "qpi";
    case 2: return "pcie";
    case 3: return "infiniband";
    case 4: return "xgmi";
    default: return "unknown";
  }
}

std::string error_json(const std::string& what) {
  return Json().kv("ok", false).kv("error", what).str();
}

struct DeviceGuard {
  int prev = 0;
  explicit DeviceGuard(int dev) {
    TK8S_HIP_CHECK(hipGetDevice(&prev));
    TK8S_HIP_CHECK(hipSetDevice(dev));
  }
  ~DeviceGuard() { (void)hipSetDevice(prev); }
};

// Per-device scratch arena for the local probes. The validation payload runs HBM, MD5 and copy
// probes back to back; giving each its own hipMalloc/hipFree of 0.25-1 GiB cost ~70 ms per
// device on MI355X (more than all the kernels together), so they share one allocation that
// grows on demand and lives until release_probe_scratch() / process exit. Peer copies keep
// their own buffers (another device's thread may be using its arena concurrently).
struct ScratchSlot {
  std::mutex mu;  // per device: growing one GPU's arena never waits on another's
  void* p = nullptr;
  size_t n = 0;
};
std::mutex g_scratch_mu;                 // guards the map only (node-based: slots never move)
std::map<int, ScratchSlot> g_scratch;

char* scratch(int device, size_t bytes) {
  ScratchSlot* slot;
  {
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    slot = &g_scratch[device];
  }
  std::lock_guard<std::mutex> lock(slot->mu);
  if (slot->n < bytes) {
    if (slot->p) TK8S_HIP_CHECK(hipFree(slot->p));
    slot->p = nullptr;
    slot->n = 0;
    TK8S_HIP_CHECK(hipMalloc(&slot->p, bytes));
    slot->n = bytes;
  }
  return static_cast<char*>(slot->p);
}

// One non-blocking stream per device, created on first use and kept: a ROCm stream is backed
// by a hardware queue, and creating one per probe (plus the legacy null stream for the copy's
// source fill) cost milliseconds each on the validation's critical path. Created outside the
// lock: a first queue costs ~20 ms (profiles/r1_init_costs), and the per-device threads of a
// multi-GPU burn-in must not serialise behind each other's creation.
std::mutex g_stream_mu;
std::map<int, hipStream_t> g_streams;

hipStream_t probe_stream(int device) {
  {
    std::lock_guard<std::mutex> lock(g_stream_mu);
    auto it = g_streams.find(device);
    if (it != g_streams.end()) return it->second;
  }
  hipStream_t s{};
  TK8S_HIP_CHECK(hipStreamCreateWithFlags(&s, hipStreamNonBlocking));
  std::lock_guard<std::mutex> lock(g_stream_mu);
  const auto ins = g_streams.emplace(device, s);
  if (!ins.second) (void)hipStreamDestroy(s);  // another thread of this device won the race
  return ins.first->second;
}

struct CachedStream {
  hipStream_t s;
  explicit CachedStream(int device) : s(probe_stream(device)) {}
};

constexpr size_t kAlign = 4096;
constexpr size_t kMallFlush = size_t(512) << 20;  // 2 x the MI355X's 256 MB Infinity Cache (MALL)
size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

// The xGMI pulls' buffers, kept per device for the life of the process: a source per GPU, filled
// once with the pull pattern and then only read (by every other GPU), and a destination + error
// counter per pulling GPU (its slot lock is held for the whole pull). Allocating and freeing them
// per pull cost a hipMalloc/hipFree each -- and hipFree synchronises the whole device, so a pull
// from GPU s waited for everything else running on s, its own probes and other GPUs' pulls.
struct PeerSlot {
  std::mutex mu;
  void* p = nullptr;
  size_t n = 0;
  bool filled = false;
};
std::mutex g_peer_mu;  // guards the maps only (node-based: slots never move)
std::map<int, PeerSlot> g_peer_src, g_peer_dst;

PeerSlot& peer_slot(std::map<int, PeerSlot>& m, int device) {
  std::lock_guard<std::mutex> lock(g_peer_mu);
  return m[device];
}

std::vector<std::pair<int, void*>> g_peer_retired;  // outgrown buffers (guarded by g_peer_mu)

// Grow `slot` (held locked by the caller) to at least `bytes` on `device`. An outgrown buffer is
// retired, not freed: another GPU may still be reading an outgrown source.
void* peer_buffer(PeerSlot& slot, int device, size_t bytes) {
  if (slot.n < bytes) {
    DeviceGuard g(device);
    void* p = nullptr;
    TK8S_HIP_CHECK(hipMalloc(&p, bytes));
    if (slot.p) {
      std::lock_guard<std::mutex> lock(g_peer_mu);
      g_peer_retired.emplace_back(device, slot.p);
    }
    slot.p = p;
    slot.n = bytes;
    slot.filled = false;
  }
  return slot.p;
}

constexpr uint32_t kPeerPattern = 0xA5A5A5A5u;

}  // namespace

void release_probe_scratch() {
  {
    std::lock_guard<std::mutex> lock(g_stream_mu);
    for (auto& kv : g_streams) (void)hipStreamDestroy(kv.second);
    g_streams.clear();
  }
  {
    std::lock_guard<std::mutex> lock(g_peer_mu);
    for (auto* m : {&g_peer_src, &g_peer_dst})
      for (auto& kv : *m) {
        std::lock_guard<std::mutex> slot_lock(kv.second.mu);
        if (!kv.second.p) continue;
        int prev = 0;
        (void)hipGetDevice(&prev);
        (void)hipSetDevice(kv.first);
        (void)hipFree(kv.second.p);
        (void)hipSetDevice(prev);
        kv.second.p = nullptr;
        kv.second.n = 0;
        kv.second.filled = false;
      }
    g_peer_src.clear();
    g_peer_dst.clear();
    for (const auto& r : g_peer_retired) {
      int prev = 0;
      (void)hipGetDevice(&prev);
      (void)hipSetDevice(r.first);
      (void)hipFree(r.second);
      (void)hipSetDevice(prev);
    }
    g_peer_retired.clear();
  }
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  for (auto& kv : g_scratch) {
    std::lock_guard<std::mutex> slot_lock(kv.second.mu);
    if (!kv.second.p) continue;
    int prev = 0;
    (void)hipGetDevice(&prev);
    (void)hipSetDevice(kv.first);
    (void)hipFree(kv.second.p);
    (void)hipSetDevice(prev);
    kv.second.p = nullptr;
    kv.second.n = 0;
  }
  g_scratch.clear();
}

void reserve_probe_scratch(int device, size_t hbm_bytes, size_t md5_bytes, uint32_t chunk_bytes, size_t copy_bytes) {
  size_t need = kAlign;
  if (hbm_bytes) need = std::max(need, align_up(hbm_bytes) + kAlign);
  if (md5_bytes && chunk_bytes) {
    const size_t ws = md5_tree_workspace(md5_bytes, chunk_bytes);
    need = std::max(need, align_up(std::max<size_t>(md5_bytes, 16)) + 2 * align_up(ws) + kAlign + kMallFlush);
  }
  if (copy_bytes) need = std::max(need, 2 * align_up(copy_bytes) + kAlign);
  DeviceGuard g(device);
  (void)scratch(device, need);
}

std::string gpuinfo_json(bool with_links) {
  const auto t0 = std::chrono::steady_clock::now();
  int n = 0;
  hipError_t e = hipGetDeviceCount(&n);
  if (e != hipSuccess) {
    return Json()
        .kv("ok", false)
        .kv("device_count", 0)
        .kv("error", std::string("hipGetDeviceCount: ") + hipGetErrorString(e))
        .str();
  }
  int rt = 0, drv = 0;
  (void)hipRuntimeGetVersion(&rt);
  (void)hipDriverGetVersion(&drv);
  std::vector<std::string> devs;
  for (int i = 0; i < n; ++i) {
    hipDeviceProp_t p;
    if (hipGetDeviceProperties(&p, i) != hipSuccess) continue;
    char bdf[64] = {0};
    (void)hipDeviceGetPCIBusId(bdf, sizeof bdf, i);
    hipUUID uuid;
    std::memset(&uuid, 0, sizeof uuid);
    (void)hipDeviceGetUuid(&uuid, i);
    std::string arch = p.gcnArchName;
    const std::string gfx = arch.substr(0, arch.find(':'));
    devs.push_back(Json()
                       .kv("index", i)
                       .kv("name", std::string(p.name))
                       .kv("arch", arch)
                       .kv("gfx", gfx)
                       .kv("total_mem_bytes", static_cast<uint64_t>(p.totalGlobalMem))
                       .kv("cu_count", p.multiProcessorCount)
                       .kv("clock_khz", p.clockRate)
                       .kv("mem_clock_khz", p.memoryClockRate)
                       .kv("mem_bus_width", p.memoryBusWidth)
                       .kv("wavefront_size", p.warpSize)
                       .kv("lds_per_block_bytes", static_cast<uint64_t>(p.sharedMemPerBlock))
                       .kv("pci_bus_id", std::string(bdf))
                       .kv("uuid", hex(reinterpret_cast<const unsigned char*>(uuid.bytes), 16))
                       .str());
  }
  std::vector<std::string> rows;
  if (with_links) {
    for (int i = 0; i < n; ++i) {
      std::vector<std::string> row;
      for (int j = 0; j < n; ++j) {
        if (i == j) {
          row.push_back(Json().kv("type", "self").kv("hops", 0).kv("p2p", true).str());
          continue;
        }
        uint32_t type = 0, hops = 0;
        const bool ok = hipExtGetLinkTypeAndHopCount(i, j, &type, &hops) == hipSuccess;
        int can = 0;
        (void)hipDeviceCanAccessPeer(&can, i, j);
        row.push_back(Json()
                          .kv("type", ok ? link_type_name(type) : std::string("unknown"))
                          .kv("hops", static_cast<int>(ok ? hops : 0))
                          .kv("p2p", can != 0)
                          .str());
      }
      rows.push_back(Json::array(row));
    }
  }
  const double ms =
      std::chrono::duration<double, std::milli>(std::chrono::steady_clock::now() - t0).count();
  Json j;
  j.kv("ok", true)
      .kv("device_count", n)
      .kv("runtime_version", rt)
      .kv("driver_version", drv)
      .raw("devices", Json::array(devs));
  if (with_links) j.raw("links", Json::array(rows));
  j.kv("discovery_ms", ms);
  return j.str();
}

std::string hbm_write_probe(size_t bytes, int iters, StoreMode mode, int device, uint32_t value) {
  try {
    if (bytes % 16 || bytes == 0) return error_json("bytes must be a positive multiple of 16");
    iters = std::max(iters, 1);
    // Host-side costs of the first probe on a device (stream = a hardware queue, the arena
    // allocation, event creation, the first launch = code-object load): they, not the kernels,
    // dominate a cold validation run, so they are reported separately.
    const auto h0 = std::chrono::steady_clock::now();
    auto lap = [last = h0]() mutable {
      const auto now = std::chrono::steady_clock::now();
      const double ms = std::chrono::duration<double, std::milli>(now - last).count();
      last = now;
      return ms;
    };
    DeviceGuard g(device);
    CachedStream st(device);
    const double stream_ms = lap();
    char* base = scratch(device, align_up(bytes) + kAlign);
    void* buf = base;
    auto* bad = reinterpret_cast<unsigned long long*>(base + align_up(bytes));
    const double alloc_ms = lap();
    EventTimer cold, warm;
    const double events_ms = lap();
    cold.start(st.s);
    hbm_fill(buf, bytes, value ^ 0xFFFFFFFFu, mode, st.s);  // cold write (first touch)
    cold.stop(st.s);
    const double launch_ms = lap();
    const float cold_ms = cold.elapsed_ms();
    const double cold_wait_ms = lap();
    warm.start(st.s);
    for (int i = 0; i < iters; ++i) hbm_fill(buf, bytes, value, mode, st.s);
    warm.stop(st.s);
    const float ms = warm.elapsed_ms() / iters;
    TK8S_HIP_CHECK(hipMemsetAsync(bad, 0, sizeof(unsigned long long), st.s));
    EventTimer rd;  // the verify pass is also the HBM read measurement (every word compared)
    rd.start(st.s);
    verify_fill(buf, bytes, value, bad, st.s);
    rd.stop(st.s);
    const float read_ms = rd.elapsed_ms();
    unsigned long long nbad = 0;
    TK8S_HIP_CHECK(hipMemcpyAsync(&nbad, bad, sizeof nbad, hipMemcpyDeviceToHost, st.s));
    wait_stream(st.s, "hbm probe");
    return Json()
        .kv("ok", nbad == 0)
        .kv("probe", "hbm_write")
        .kv("read_ms", static_cast<double>(read_ms))
        .kv("read_gbps", bytes / (read_ms * 1e-3) / 1e9)
        .kv("device", device)
        .kv("bytes", static_cast<uint64_t>(bytes))
        .kv("iters", iters)
        .kv("mode", mode == StoreMode::kNonTemporal ? "nontemporal" : "plain")
        .kv("cold_ms", static_cast<double>(cold_ms))
        .kv("ms", static_cast<double>(ms))
        .kv("seconds", ms * 1e-3)
        .kv("gbps", bytes / (ms * 1e-3) / 1e9)
        .kv("bad_words", static_cast<uint64_t>(nbad))
        .raw("host_ms", Json()
                            .kv("stream", stream_ms)
                            .kv("alloc", alloc_ms)
                            .kv("events", events_ms)
                            .kv("first_launch", launch_ms)
                            .kv("first_wait", cold_wait_ms)
                            .str())
        .str();
  } catch (const std::exception& ex) {
    return error_json(ex.what());
  }
}

std::string md5_probe(size_t bytes, uint32_t chunk_bytes, uint64_t seed, int iters, int device) {
  try {
    if (bytes % 16) return error_json("bytes must be a multiple of 16");
    if (chunk_bytes == 0 || chunk_bytes % 64) return error_json("chunk must be a multiple of 64");
    iters = std::max(iters, 1);
    DeviceGuard g(device);
    CachedStream st(device);
    const size_t ws = md5_tree_workspace(bytes, chunk_bytes);
    const size_t o_wa = align_up(std::max<size_t>(bytes, 16)), o_wb = o_wa + align_up(ws), o_out = o_wb + align_up(ws),
                 o_flush = o_out + kAlign;
    char* base = scratch(device, o_flush + kMallFlush);
    void *data = base, *wa = base + o_wa, *wb = base + o_wb, *out = base + o_out, *flush = base + o_flush;
    EventTimer fill_t, cold_t;
    fill_t.start(st.s);
    philox_fill(data, bytes, seed, st.s);
    fill_t.stop(st.s);
    const float fill_ms = fill_t.elapsed_ms();
    cold_t.start(st.s);
    md5_tree(data, bytes, chunk_bytes, wa, wb, out, st.s);
    cold_t.stop(st.s);
    const float cold_ms = cold_t.elapsed_ms();
    // each timed pass starts from HBM: 512 MiB written elsewhere first evicts the input from the
    // memory-side Infinity Cache (a 256 MiB input fits the 256 MB MALL)
    std::vector<std::unique_ptr<EventTimer>> warm;
    for (int i = 0; i < iters; ++i) {
      hbm_fill(flush, kMallFlush, 0x5A5A5A5Au + i, StoreMode::kPlain, st.s);
      warm.push_back(std::make_unique<EventTimer>());
      warm.back()->start(st.s);
      md5_tree(data, bytes, chunk_bytes, wa, wb, out, st.s);
      warm.back()->stop(st.s);
    }
    float total = 0.f;
    for (auto& w : warm) total += w->elapsed_ms();
    const float ms = total / iters;
    unsigned char digest[16];
    TK8S_HIP_CHECK(hipMemcpyAsync(digest, out, 16, hipMemcpyDeviceToHost, st.s));
    wait_stream(st.s, "md5 probe");
    return Json()
        .kv("ok", true)
        .kv("probe", "md5_tree")
        .kv("device", device)
        .kv("bytes", static_cast<uint64_t>(bytes))
        .kv("chunk_bytes", chunk_bytes)
        .kv("seed", static_cast<uint64_t>(seed))
        .kv("iters", iters)
        .kv("digest", hex(digest, 16))
        .kv("fill_ms", static_cast<double>(fill_ms))
        .kv("fill_gbps", bytes / (fill_ms * 1e-3) / 1e9)
        .kv("cold_ms", static_cast<double>(cold_ms))
        .kv("ms", static_cast<double>(ms))
        .kv("seconds", ms * 1e-3)
        .kv("mbps", bytes / (ms * 1e-3) / 1e6)
        .kv("mall_flushed", true)
        .str();
  } catch (const std::exception& ex) {
    return error_json(ex.what());
  }
}

std::string copy_probe(int src_device, int dst_device, size_t bytes, int iters, bool dma) {
  // a failed pull still names its link: xgmi.py counts it as a dead link between the two GPUs
  auto link_error = [&](const std::string& what) {
    return Json().kv("ok", false).kv("probe", src_device != dst_device ? "xgmi_peer_copy" : "local_copy")
        .kv("src_device", src_device).kv("dst_device", dst_device).kv("error", what).str();
  };
  try {
    if (bytes % 16 || bytes == 0) return error_json("bytes must be a positive multiple of 16");
    iters = std::max(iters, 1);
    // TK8S_PROBE_PEER_PATH=1: a copy within one GPU takes the peer path (its cached buffers, no
    // peer grant needed) -- how a one-GPU box exercises the code the xGMI pulls run
    const bool forced = std::getenv("TK8S_PROBE_PEER_PATH") != nullptr && src_device == dst_device;
    const bool peer = src_device != dst_device || forced;
    int can = 1;
    if (peer && !forced) {
      TK8S_HIP_CHECK(hipDeviceCanAccessPeer(&can, dst_device, src_device));
      if (!can) return link_error("no peer access from dst to src");
    }
    // Local: src, dst and the error counter are carved from this device's scratch arena.
    // Peer: the cached peer buffers (PeerSlot): the source filled once, the destination held.
    void *src = nullptr, *dst = nullptr;
    unsigned long long* bad = nullptr;
    std::unique_lock<std::mutex> dst_hold;
    if (!peer) {
      DeviceGuard g(src_device);
      char* base = scratch(src_device, 2 * align_up(bytes) + kAlign);
      src = base;
      dst = base + align_up(bytes);
      bad = reinterpret_cast<unsigned long long*>(base + 2 * align_up(bytes));
      const hipStream_t ss = probe_stream(src_device);
      hbm_fill(src, bytes, kPeerPattern, StoreMode::kPlain, ss);
      wait_stream(ss, "copy source fill");
    } else {
      PeerSlot& ps = peer_slot(g_peer_src, src_device);
      std::lock_guard<std::mutex> lock(ps.mu);
      src = peer_buffer(ps, src_device, align_up(bytes));
      if (!ps.filled) {
        DeviceGuard g(src_device);
        const hipStream_t ss = probe_stream(src_device);
        hbm_fill(src, ps.n, kPeerPattern, StoreMode::kPlain, ss);
        wait_stream(ss, "peer source fill");
        ps.filled = true;
      }
      PeerSlot& pd = peer_slot(g_peer_dst, dst_device);
      dst_hold = std::unique_lock<std::mutex>(pd.mu);
      char* base = static_cast<char*>(peer_buffer(pd, dst_device, align_up(bytes) + kAlign));
      dst = base;
      bad = reinterpret_cast<unsigned long long*>(base + align_up(bytes));
    }
    DeviceGuard g(dst_device);
    if (peer && !forced) {
      const hipError_t pe = hipDeviceEnablePeerAccess(src_device, 0);
      if (pe != hipSuccess && pe != hipErrorPeerAccessAlreadyEnabled) TK8S_HIP_CHECK(pe);
      (void)hipGetLastError();
    }
    CachedStream st(dst_device);
    if (peer) {
      // TK8S_FAULTS probe.exit|crash@peers end the process here; probe.hang@peers stalls this
      // pull's queue, so the bounded waits below must give up and name the link (failfast.h)
      fault_point("probe", "peers", /*host_hang=*/false);
      if (fault_armed("probe", "hang", "peers")) gpu_stall(st.s, 2 * gpu_sync_timeout_s() + 5);
    }
    stream_copy(dst, src, bytes, st.s);  // warm-up
    EventTimer kt, dt;
    kt.start(st.s);
    for (int i = 0; i < iters; ++i) stream_copy(dst, src, bytes, st.s);
    kt.stop(st.s);
    const double bound = peer ? peer_sync_timeout_s() : gpu_sync_timeout_s();  // a link is not waited for
    const float kernel_ms = kt.elapsed_ms(bound) / iters;
    TK8S_HIP_CHECK(hipMemsetAsync(bad, 0, sizeof(unsigned long long), st.s));
    verify_fill(dst, bytes, kPeerPattern, bad, st.s);
    unsigned long long nbad = 0;
    TK8S_HIP_CHECK(hipMemcpyAsync(&nbad, bad, sizeof nbad, hipMemcpyDeviceToHost, st.s));
    // The SDMA-engine path only for peers (where it is a separate xGMI data path worth
    // checking); locally it measured nothing the kernel copy does not, and bringing up the
    // copy engine cost ~10 ms of the validation's critical path.
    float dma_ms = 0.f;
    dma = dma && peer;
    if (dma) {
      dt.start(st.s);
      for (int i = 0; i < iters; ++i)
        TK8S_HIP_CHECK(hipMemcpyPeerAsync(dst, dst_device, src, src_device, bytes, st.s));
      dt.stop(st.s);
      dma_ms = dt.elapsed_ms(bound) / iters;
    }
    wait_stream(st.s, "copy probe", bound);
    Json j;
    j.kv("ok", nbad == 0)
        .kv("probe", peer ? "xgmi_peer_copy" : "local_copy")
        .kv("src_device", src_device)
        .kv("dst_device", dst_device)
        .kv("bytes", static_cast<uint64_t>(bytes))
        .kv("iters", iters)
        .kv("kernel_ms", static_cast<double>(kernel_ms))
        .kv("kernel_gbps", bytes / (kernel_ms * 1e-3) / 1e9);
    if (dma) j.kv("dma_ms", static_cast<double>(dma_ms)).kv("dma_gbps", bytes / (dma_ms * 1e-3) / 1e9);
    return j.kv("bad_words", static_cast<uint64_t>(nbad)).str();
  } catch (const std::exception& ex) {
    return link_error(ex.what());
  }
}

namespace {

// ---- the layer probe's host side: the same values in 64 bits ----------------------------------
double bf16_value(uint16_t v) {
  const uint32_t u = static_cast<uint32_t>(v) << 16;
  float f;
  std::memcpy(&f, &u, 4);
  return f;
}

double e4m3_of(uint8_t v) {
  const int e = v >> 3 & 15, m = v & 7;
  if (e == 15 && m == 7) return std::nan("");
  const double x = e ? std::ldexp(8 + m, e - 10) : std::ldexp(m, -9);
  return v & 128 ? -x : x;
}

double e4m3_value(uint8_t v) {
  static const std::vector<double> table = [] {
    std::vector<double> t(256);
    for (int i = 0; i < 256; ++i) t[i] = e4m3_of(static_cast<uint8_t>(i));
    return t;
  }();
  return table[v];
}

struct Compared {
  double worst = 0;  // the largest error so far, as a share of the allowed one
  uint64_t count = 0;
  void add(double got, double want, double allowed) {
    ++count;
    const double e = std::fabs(got - want);
    worst = std::max(worst, e <= allowed ? (allowed > 0 ? e / allowed : 0.0) : (e == e && allowed > 0 ? e / allowed : 1e30));
  }
};

// Row r of a matrix in 8 bits, in 64: values and scales fetched from the device.
std::vector<double> fetch_row(const Fp8Matrix& m, size_t r, size_t scale_row, size_t k, hipStream_t s) {
  std::vector<uint8_t> v(k), sc(k / 128);
  TK8S_HIP_CHECK(hipMemcpyAsync(v.data(), m.values + r * m.ld, k, hipMemcpyDeviceToHost, s));
  TK8S_HIP_CHECK(hipMemcpy2DAsync(sc.data(), 1, m.scales + scale_row, m.ld_scales, 1, k / 128, hipMemcpyDeviceToHost, s));
  wait_stream(s, "layer probe");
  std::vector<double> x(k);
  for (size_t i = 0; i < k; ++i) x[i] = sc[i / 128] == 255 ? std::nan("") : std::ldexp(e4m3_value(v[i]), sc[i / 128] - 127);
  return x;
}

// `height` pieces of `n` values each, `pitch` bytes apart.
template <class T> std::vector<T> fetch_raw(const void* p, size_t n, size_t pitch, size_t height, hipStream_t s) {
  std::vector<T> v(n * height);
  TK8S_HIP_CHECK(hipMemcpy2DAsync(v.data(), n * sizeof(T), p, pitch, n * sizeof(T), height, hipMemcpyDeviceToHost, s));
  wait_stream(s, "layer probe");
  return v;
}

template <class T> std::vector<double> fetch(const void* p, size_t n, hipStream_t s) {  // 16-bit or 32-bit values
  std::vector<T> v(n);
  TK8S_HIP_CHECK(hipMemcpyAsync(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost, s));
  wait_stream(s, "layer probe");
  std::vector<double> x(n);
  for (size_t i = 0; i < n; ++i)
    if constexpr (sizeof(T) == 2) x[i] = bf16_value(v[i]);
    else x[i] = v[i];
  return x;
}

// One value of a product against its sum in 64 bits. Allowed: k + 2 roundings of 32-bit sums; for 16-bit results
// half a step of theirs, and what a matrix instruction cuts off when it lines up 8 neighbouring
// products (below 2^-13 of the largest).
void compare_dot(Compared& c, double got, const std::vector<double>& x, const std::vector<double>& y, bool is16) {
  double want = 0, size = 0, tops = 0;
  for (size_t i = 0; i < x.size(); i += 8) {
    double top = 0;
    for (size_t j = i; j < i + 8; ++j) {
      const double p = x[j] * y[j];
      want += p;
      size += std::fabs(p);
      top = std::max(top, std::fabs(p));
    }
    tops += top;
  }
  double off = static_cast<double>(x.size() + 2) * std::ldexp(size, -24);
  if (is16) off += 7 * std::ldexp(tops, -13), off += std::ldexp(std::fabs(want) + off, -8);
  c.add(got, want, off);
}

// The E8M0 byte of a block of this largest magnitude: the least power of two that brings it to 448 or below.
int scale_byte_of(double top) {
  if (top == 0) return 127;
  int e = 0;
  const double m = std::frexp(top, &e);
  return std::clamp(e - (m <= 0.875 ? 9 : 8), -127, 127) + 127;
}

// Values in 8 bits that share a scale against the 16-bit ones that they were made of: every byte is given.
void compare_rounded(Compared& c, const uint16_t* source, const uint8_t* values, size_t n, uint8_t scale) {
  double top = 0;
  for (size_t i = 0; i < n; ++i) top = std::max(top, std::fabs(bf16_value(source[i])));
  const int byte = scale_byte_of(top);
  c.add(scale, byte, 0);
  const double by = std::ldexp(1.0, 127 - byte);
  for (size_t i = 0; i < n; ++i) {
    const double v = bf16_value(source[i]) * by, size = std::fabs(v);
    uint64_t binade;  // of the power of two at or below it
    std::memcpy(&binade, &size, 8);
    binade &= uint64_t(0x7ff) << 52;
    double power;
    std::memcpy(&power, &binade, 8);
    const double step = std::max(power, 0x1p-6) / 8;
    c.add(e4m3_value(values[i]), std::nearbyint(v / step) * step, 0);
  }
}

// One value of the norm's weight gradient against its sum in 64 bits: rows + 4 roundings of 32-bit sums.
void compare_weight_sum(Compared& c, double got, const uint16_t* dy, const uint16_t* h, const float* rstd, size_t rows) {
  double want = 0, size = 0;
  for (size_t r = 0; r < rows; ++r) {
    const double p = bf16_value(dy[r]) * bf16_value(h[r]) * rstd[r];
    want += p;
    size += std::fabs(p);
  }
  c.add(got, want, static_cast<double>(rows + 4) * std::ldexp(size, -24));
}

}  // namespace

double layer_rounding_error(const uint16_t* source, const uint8_t* values, size_t n, uint8_t scale) {
  Compared c;
  compare_rounded(c, source, values, n, scale);
  return c.worst;
}

double layer_weight_sum_error(float got, const uint16_t* dy, const uint16_t* h, const float* rstd, size_t rows) {
  Compared c;
  compare_weight_sum(c, got, dy, h, rstd, rows);
  return c.worst;
}

std::string layer_probe(size_t rows, size_t width, uint64_t seed, int iters, int device) {
  try {
    if (rows == 0 || width == 0 || rows % 128 || width % 128 || rows > 16384 || width > 16384)
      return error_json("rows and width must be multiples of 128, from 128 to 16384");
    iters = std::max(iters, 1);
    DeviceGuard g(device);
    CachedStream st(device);
    const size_t blocks = width / 128, row_blocks = rows / 128, tiles = (blocks + 3) / 4 * 4, n = rows * width;
    size_t at = 0;
    auto place = [&](size_t bytes) { return std::exchange(at, at + align_up(bytes)); };
    const size_t o_x = place(2 * n), o_res = place(2 * n), o_nw = place(2 * width), o_w = place(2 * width * width), o_g = place(2 * n);
    const size_t o_h = place(2 * n), o_y = place(2 * n), o_rstd = place(4 * rows), o_dq = place(2 * n);
    const size_t o_q = place(n), o_qs = place(rows * blocks), o_yc = place(n), o_ycs = place(width * row_blocks);
    const size_t o_wt = place(width * width), o_wts = place(tiles * blocks), o_wc = place(width * width), o_wcs = place(width * blocks);
    const size_t o_gr = place(n), o_grs = place(rows * blocks), o_gc = place(n), o_gcs = place(width * row_blocks);
    const size_t o_ws = place(rms_norm_backward_workspace(rows, width));
    const size_t o_out = at;  // what the digest is taken of: y W^T, then the gradients
    const size_t o_c = place(2 * n), o_dx = place(2 * n), o_dw = place(4 * width * width), o_dnw = place(4 * width), out_bytes = at - o_out;
    const size_t tree = md5_tree_workspace(out_bytes, 1024), o_wa = place(tree), o_wb = place(tree), o_md = place(16);
    const size_t o_col = place(2 * std::max(rows, width));
    char* const base = scratch(device, at);
    auto u8 = [&](size_t o) { return reinterpret_cast<uint8_t*>(base + o); };
    const Fp8Matrix q{u8(o_q), width, u8(o_qs), rows}, yc{u8(o_yc), rows, u8(o_ycs), width}, wt{u8(o_wt), width, u8(o_wts), tiles},
        wc{u8(o_wc), width, u8(o_wcs), width}, gr{u8(o_gr), width, u8(o_grs), rows}, gc{u8(o_gc), rows, u8(o_gcs), width}, none{nullptr, 0, nullptr, 0};
    layer_fill(base + o_x, n, seed, st.s);
    layer_fill(base + o_res, n, seed + 1, st.s);
    layer_fill(base + o_nw, width, seed + 2, st.s);
    layer_fill(base + o_w, width * width, seed + 3, st.s);
    layer_fill(base + o_g, n, seed + 4, st.s);
    hbm_fill(base + o_out, out_bytes, 0, StoreMode::kPlain, st.s);  // the digest covers the room between outputs

    enum { kNorm, kRound, kForward, kInput, kWeight, kBackward, kPhases };
    double ms[kPhases] = {};
    auto step = [&](bool timed) {
      std::vector<std::unique_ptr<EventTimer>> timers;
      auto phase = [&](auto&& work) {
        timers.push_back(std::make_unique<EventTimer>());
        timers.back()->start(st.s);
        work();
        timers.back()->stop(st.s);
      };
      phase([&] {
        NormArgs a{};
        a.x = base + o_x, a.ldx = width, a.residual = base + o_res, a.ldr = width, a.weight = base + o_nw, a.h = base + o_h, a.ldh = width;
        a.q = q.values, a.ldq = width, a.scales = q.scales, a.lds = rows, a.y = base + o_y, a.ldy = width;
        a.rstd = reinterpret_cast<float*>(base + o_rstd), a.rows = rows, a.cols = width, a.eps = 1e-5;
        rms_norm_fp8(a, LayerType::kBF16, LayerType::kBF16, st.s);
      });
      phase([&] {
        fp8_quantize({base + o_w, width, width, width, none, wc, wt}, LayerType::kBF16, st.s);
        fp8_quantize({base + o_g, width, rows, width, gr, gc, none}, LayerType::kBF16, st.s);
        fp8_quantize({base + o_y, width, rows, width, none, yc, none}, LayerType::kBF16, st.s);
      });
      phase([&] { fp8_matmul({q, wt, true, base + o_c, width, rows, width, width}, LayerType::kBF16, st.s); });
      phase([&] { fp8_matmul({gr, wc, false, base + o_dq, width, rows, width, width}, LayerType::kBF16, st.s); });
      phase([&] { fp8_matmul({gc, yc, false, base + o_dw, width, width, width, rows}, LayerType::kF32, st.s); });
      phase([&] {
        NormBackwardArgs a{};
        a.dy = base + o_dq, a.lddy = width, a.h = base + o_h, a.ldh = width, a.weight = base + o_nw;
        a.rstd = reinterpret_cast<const float*>(base + o_rstd), a.dh = base + o_g, a.lddh = width, a.dx = base + o_dx, a.lddx = width;
        a.dw = reinterpret_cast<float*>(base + o_dnw), a.workspace = reinterpret_cast<float*>(base + o_ws), a.rows = rows, a.cols = width;
        rms_norm_backward(a, LayerType::kBF16, LayerType::kBF16, st.s);
      });
      md5_tree(base + o_out, out_bytes, 1024, base + o_wa, base + o_wb, base + o_md, st.s);
      unsigned char digest[16];
      TK8S_HIP_CHECK(hipMemcpyAsync(digest, base + o_md, 16, hipMemcpyDeviceToHost, st.s));
      wait_stream(st.s, "layer probe");
      if (timed)
        for (int i = 0; i < kPhases; ++i) ms[i] += timers[i]->elapsed_ms();
      return hex(digest, 16);
    };
    const std::string digest = step(false);
    int differ = 0;
    for (int i = 0; i < iters; ++i) differ += step(true) != digest;
    for (double& m : ms) m /= iters;

    // sampled rows and columns again on the host
    Compared norm, rounding, forward, input, weight, backward;
    const std::vector<double> nw = fetch<uint16_t>(base + o_nw, width, st.s);
    const std::vector<float> rstds = fetch_raw<float>(base + o_rstd, rows, 4 * rows, 1, st.s);
    constexpr size_t kSamples = 12;
    auto sample = [](size_t i, size_t count) { return (i * (count - 1) / (kSamples - 1) + 37 * i) % count; };
    std::vector<std::vector<double>> w_rows, wc_rows, yc_rows;
    for (size_t j = 0; j < kSamples; ++j) {
      const size_t col = sample(j, width);
      w_rows.push_back(fetch_row(wt, col, col / 128, width, st.s));
      wc_rows.push_back(fetch_row(wc, col, col, width, st.s));
      yc_rows.push_back(fetch_row(yc, col, col, rows, st.s));
    }
    // what the roundings made of their 16-bit values: a row of the first layout, a column of the transposed ones, a tile
    auto check_blocks = [&](const std::vector<uint16_t>& source, const Fp8Matrix& m, size_t r) {
      const auto v = fetch_raw<uint8_t>(m.values + r * m.ld, source.size(), source.size(), 1, st.s);
      const auto sc = fetch_raw<uint8_t>(m.scales + r, 1, m.ld_scales, source.size() / 128, st.s);
      for (size_t b = 0; b < sc.size(); ++b) compare_rounded(rounding, &source[b * 128], &v[b * 128], 128, sc[b]);
    };
    auto column = [&](size_t of, size_t col, size_t count) {  // put together on the device: the host would fetch it value by value
      TK8S_HIP_CHECK(hipMemcpy2DAsync(base + o_col, 2, base + of + 2 * col, 2 * width, 2, count, hipMemcpyDeviceToDevice, st.s));
      return fetch_raw<uint16_t>(base + o_col, count, 2 * count, 1, st.s);
    };
    for (size_t i = 0; i < kSamples; ++i) {
      const size_t r = sample(i, rows), col = sample(i, width), tile_r = sample(i, blocks), tile_c = (tile_r + 5 * i) % blocks;
      check_blocks(fetch_raw<uint16_t>(base + o_g + 2 * r * width, width, 2 * width, 1, st.s), gr, r);
      check_blocks(column(o_g, col, rows), gc, col);
      check_blocks(column(o_y, col, rows), yc, col);
      check_blocks(column(o_w, col, width), wc, col);
      const auto source = fetch_raw<uint16_t>(base + o_w + 2 * 128 * (tile_r * width + tile_c), 128, 2 * width, 128, st.s);
      const auto tile = fetch_raw<uint8_t>(wt.values + 128 * (tile_r * width + tile_c), 128, width, 128, st.s);
      compare_rounded(rounding, source.data(), tile.data(), 128 * 128,
                      fetch_raw<uint8_t>(wt.scales + tile_c * wt.ld_scales + tile_r, 1, 1, 1, st.s)[0]);
      compare_weight_sum(backward, fetch_raw<float>(base + o_dnw + 4 * col, 1, 4, 1, st.s)[0], column(o_dq, col, rows).data(),
                         column(o_h, col, rows).data(), rstds.data(), rows);
    }
    for (size_t i = 0; i < kSamples; ++i) {
      const size_t r = sample(i, rows);
      const auto q_scales = fetch_raw<uint8_t>(q.scales + r, 1, q.ld_scales, blocks, st.s);
      const auto x = fetch<uint16_t>(base + o_x + 2 * r * width, width, st.s), res = fetch<uint16_t>(base + o_res + 2 * r * width, width, st.s);
      const auto h = fetch<uint16_t>(base + o_h + 2 * r * width, width, st.s), y = fetch<uint16_t>(base + o_y + 2 * r * width, width, st.s);
      const auto qr = fetch_row(q, r, r, width, st.s), gq = fetch_row(gr, r, r, width, st.s);
      const auto gv = fetch<uint16_t>(base + o_g + 2 * r * width, width, st.s), dq = fetch<uint16_t>(base + o_dq + 2 * r * width, width, st.s);
      const auto dx = fetch<uint16_t>(base + o_dx + 2 * r * width, width, st.s), c = fetch<uint16_t>(base + o_c + 2 * r * width, width, st.s);
      double squares = 0, along = 0, along_size = 0;
      for (double v : h) squares += v * v;
      const double rstd = 1 / std::sqrt(squares / static_cast<double>(width) + 1e-5);
      norm.add(rstds[r], rstd, std::ldexp(rstd, -24) * (1 + 1e-6));
      const double sums = static_cast<double>(width + 8) * std::ldexp(1.0, -24);  // of 32-bit sums, relative to their size
      for (size_t j = 0; j < width; ++j) {
        const double want = h[j] * rstd * nw[j];
        norm.add(h[j], x[j] + res[j], std::ldexp(std::fabs(x[j] + res[j]), -8));
        norm.add(y[j], want, std::ldexp(std::fabs(want), -8) * (1 + 1e-6));
        // 8-bit values: half a step of e4m3, at least that of the smallest (2^-10 of the block's 2^e >= amax / 448)
        double top = 0;
        for (size_t b = j / 128 * 128; b < j / 128 * 128 + 128; ++b) top = std::max(top, std::fabs(h[b] * rstd * nw[b]));
        rounding.add(qr[j], want, (std::ldexp(std::fabs(want), -4) + std::ldexp(top / 224, -10)) * (1 + 1e-6));
        // its scale, too, unless the host's last bits decide between two
        if (j % 128 == 0 && scale_byte_of(top * (1 - 1e-9)) == scale_byte_of(top * (1 + 1e-9))) rounding.add(q_scales[j / 128], scale_byte_of(top), 0);
        along += dq[j] * nw[j] * h[j];
        along_size += std::fabs(dq[j] * nw[j] * h[j]);
      }
      for (size_t j = 0; j < width; ++j) {
        const double part = h[j] * rstd * rstd * rstd / static_cast<double>(width), want = gv[j] + rstd * dq[j] * nw[j] - part * along;
        const double off = sums * (std::fabs(rstd * dq[j] * nw[j]) + std::fabs(part) * along_size + std::fabs(gv[j]));
        backward.add(dx[j], want, std::ldexp(std::fabs(want) + off, -8) + off);
      }
      for (size_t j = 0; j < kSamples; ++j) {
        const size_t col = sample(j, width);
        compare_dot(forward, c[col], qr, w_rows[j], true);
        compare_dot(input, dq[col], gq, wc_rows[j], true);
      }
      const size_t wr = sample(i, width);
      const auto gcr = fetch_row(gc, wr, wr, rows, st.s);
      const auto dw = fetch<float>(base + o_dw + 4 * wr * width, width, st.s);
      for (size_t j = 0; j < kSamples; ++j) compare_dot(weight, dw[sample(j, width)], gcr, yc_rows[j], false);
    }
    const double worst = std::max({norm.worst, rounding.worst, forward.worst, input.worst, weight.worst, backward.worst});
    const double flops = 2.0 * static_cast<double>(n) * static_cast<double>(width), e = static_cast<double>(n);
    const double ww = static_cast<double>(width) * static_cast<double>(width);
    auto rate = [](double amount, double msec, double unit) { return amount / (msec * 1e-3) / unit; };
    double total = 0;
    for (double m : ms) total += m;
    return Json()
        .kv("ok", differ == 0 && worst <= 1)
        .kv("probe", "layer")
        .kv("device", device)
        .kv("rows", static_cast<uint64_t>(rows))
        .kv("width", static_cast<uint64_t>(width))
        .kv("seed", static_cast<uint64_t>(seed))
        .kv("iters", iters)
        .kv("digest", digest)
        .kv("steps_that_differ", differ)
        .kv("error", worst)
        .raw("errors", Json().kv("norm", norm.worst).kv("rounding", rounding.worst).kv("forward", forward.worst)
                           .kv("input_gradient", input.worst).kv("weight_gradient", weight.worst).kv("norm_gradient", backward.worst).str())
        .raw("compared", Json().kv("norm", norm.count).kv("rounding", rounding.count).kv("forward", forward.count)
                             .kv("input_gradient", input.count).kv("weight_gradient", weight.count).kv("norm_gradient", backward.count).str())
        .kv("ms", total)
        .kv("forward_tflops", rate(flops, ms[kForward], 1e12))
        .kv("input_gradient_tflops", rate(flops, ms[kInput], 1e12))
        .kv("weight_gradient_tflops", rate(flops, ms[kWeight], 1e12))
        .kv("norm_gbps", rate(9 * e, ms[kNorm], 1e9))               // x, residual in; h, y and 8 bits out
        .kv("rounding_gbps", rate(7 * e + 4 * ww, ms[kRound], 1e9))  // W, gradient and y in; two, two and one of 8 bits out
        .kv("norm_gradient_gbps", rate(8 * e, ms[kBackward], 1e9))  // dy, h, dh in; dx out
        .str();
  } catch (const std::exception& ex) {
    return error_json(ex.what());
  }
}

}  // namespace tk8s
