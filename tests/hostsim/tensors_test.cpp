// The host side of the first-order steps (stochqn_amd/csrc/tensors.cpp, compiled unchanged) on the CPU: what it hands to the kernels and what it
// refuses.  Device memory is address ranges that nothing dereferences; the launchers write down the tables they are given.
#include "tensors.hpp"
#include "runtime.hpp"
#include "stochqn_hip.h"

#include <atomic>
#include <chrono>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <random>
#include <thread>
#include <vector>

// ---- a HIP runtime of address ranges ---------------------------------------------------------------------------------------------------
struct Block { uintptr_t at; size_t bytes; int device; };
static std::vector<Block> g_blocks;
static thread_local int g_device = 0, g_launch_error = 0;
static int g_fail_after = -1;
static bool g_capturing = false;
static uintptr_t g_next = (uintptr_t) 1 << 40;       // far below what the process itself uses

static void* device_block(size_t bytes, int device = 0, size_t shift = 0)
{
	g_next += (1 << 20);
	const uintptr_t at = g_next + shift;
	g_blocks.push_back({g_next, bytes + shift, device});
	g_next += (bytes + shift + 4095) / 4096 * 4096;
	return (void*) at;
}
static const Block* find(const void* p)
{
	for (const Block& b : g_blocks)
		if ((uintptr_t) p >= b.at && (uintptr_t) p < b.at + b.bytes) return &b;
	return nullptr;
}
static bool failing() { return g_fail_after >= 0 && g_fail_after-- == 0; }         // (one thread only)

extern "C" {
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* a, const void* p)
{
	if (failing()) return hipErrorUnknown;
	const Block* b = find(p);
	if (!b) return hipErrorInvalidValue;
	std::memset(a, 0, sizeof *a);
	a->type = hipMemoryTypeDevice;
	a->device = b->device;
	return hipSuccess;
}
hipError_t hipMemGetAddressRange(hipDeviceptr_t* base, size_t* size, hipDeviceptr_t p)
{
	const Block* b = find(p);
	if (!b || failing()) return hipErrorInvalidValue;
	*base = (void*) b->at;
	*size = b->bytes;
	return hipSuccess;
}
hipError_t hipGetDevice(int* d) { if (failing()) return hipErrorUnknown; *d = g_device; return hipSuccess; }
hipError_t hipSetDevice(int d) { if (failing()) return hipErrorUnknown; g_device = d; return hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t s, hipDevice_t* d) { if (failing()) return hipErrorUnknown; *d = (int) ((uintptr_t) s >> 8); return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) { if (failing()) return hipErrorUnknown; *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone; return hipSuccess; }
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { if (failing()) return hipErrorUnknown; *v = 256; return hipSuccess; }
hipError_t hipGetLastError() { const int e = g_launch_error; g_launch_error = 0; return (hipError_t) e; }
const char* hipGetErrorString(hipError_t) { return "an error"; }
}

// ---- the launchers ---------------------------------------------------------------------------------------------------------------------
struct Launch { char kind; int bits, tile, grid, on; hipStream_t st; sqn::Table<sqn::AdamwArgs, sqn::kEntries> a; sqn::Table<sqn::NormArgs, sqn::kEntries> n; int count; bool out; };
static std::vector<Launch> g_launches;
static int g_ranks = 1;
static bool g_fail_launch = false, g_fail_reduce = false, g_on_the_host = false;
static std::atomic<bool> g_meeting{false};
static std::atomic<int> g_arrived{0};
static std::mutex g_mu;
static void launched_one(Launch l) { std::lock_guard<std::mutex> lk(g_mu); l.on = g_device; g_launches.push_back(l); if (g_fail_launch) g_launch_error = hipErrorLaunchFailure; }
namespace sqn {
void launch_adamw(hipStream_t st, int bits, int tile, int grid, const Table<AdamwArgs, kEntries>& t) { Launch l{}; l.kind = 'a'; l.bits = bits; l.tile = tile; l.grid = grid; l.st = st; l.a = t; launched_one(l); }
void launch_norm(hipStream_t st, int tile, int grid, const Table<NormArgs, kEntries>& t) { Launch l{}; l.kind = 'n'; l.tile = tile; l.grid = grid; l.st = st; l.n = t; l.out = t.a.out; launched_one(l); }
void launch_norm_sum(hipStream_t st, double*, int count, double, double, float* out) { Launch l{}; l.kind = 's'; l.st = st; l.count = count; l.out = out; launched_one(l); }
void launch_norm_verdict(hipStream_t st, const double*, double, double, float* out) { Launch l{}; l.kind = 'v'; l.st = st; l.out = out; launched_one(l); }
bool device_ready() { return true; }
int comm_nranks() { return g_ranks; }
bool reduces_on_the_host() { return g_on_the_host; }
bool reduce_in_place(double*, int, hipStream_t)
{
	if (g_meeting.load()) {                                                     // a reducer that returns when both ranks are there, or gives up
		const int mine = ++g_arrived;
		for (int k = 0; k < 5000 && g_arrived.load() < (mine + 1) / 2 * 2; k++) std::this_thread::sleep_for(std::chrono::milliseconds(1));
		return g_arrived.load() >= (mine + 1) / 2 * 2;
	}
	return !g_fail_reduce;
}
}

#define CHECK(x) do { if (!(x)) { std::printf("FAILED line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)

struct Lists {
	std::vector<void*> p, g;
	std::vector<size_t> n;
	std::vector<int> tp, tg;
	stochqn_hip_tensors *params, *grads;
	explicit Lists(const std::vector<size_t>& sizes, int device = 0, unsigned seed = 0) : n(sizes)
	{
		std::mt19937 r(seed);
		for (size_t k : n) {
			tp.push_back((int) (r() % 3));
			tg.push_back((int) (r() % 3));
			p.push_back(k ? device_block(k * sqn::type_size(tp.back()), device, 4 * (r() % 3)) : nullptr);
			g.push_back(k ? device_block(k * sqn::type_size(tg.back()), device, 4 * (r() % 3)) : nullptr);
		}
		params = stochqn_hip_tensors_create((int) n.size(), p.data(), n.data(), tp.data());
		grads = stochqn_hip_tensors_create((int) n.size(), g.data(), n.data(), tg.data());
		CHECK(params && grads);
	}
	~Lists() { stochqn_hip_tensors_destroy(params); stochqn_hip_tensors_destroy(grads); }
	stochqn_hip_adamw_setup setup(int bits, int device = 0) const
	{
		const size_t state = stochqn_hip_tensors_state(params, nullptr);
		stochqn_hip_adamw_setup s{};
		s.beta1 = 0.9; s.beta2 = 0.999; s.eps = 1e-8; s.state_bits = bits;
		s.m = device_block(state * bits / 8 + 16, device);
		s.v = device_block(state * bits / 8 + 16, device);
		s.master = (float*) device_block(state * 4 + 16, device);
		if (bits == 8) { s.m_scale = (unsigned char*) device_block(state / 128 + 1, device); s.v_scale = (unsigned char*) device_block(state / 128 + 1, device); }
		s.count = (long long*) device_block(16, device);
		s.work = device_block(4096, device);
		return s;
	}
};

// every element of every tensor is in exactly one tile of one launch, with its own state
template <class T> static void check_table(const Lists& l, const std::vector<size_t>& offset, size_t& next, const T& t, int tile, bool step)
{
	uint64_t tiles = 0;
	CHECK(t.a.entries >= 0 && t.a.entries <= sqn::kEntries);
	for (int k = 0; k < t.a.entries; k++) {
		while (next < l.n.size() && !l.n[next]) next++;
		CHECK(next < l.n.size());
		const sqn::TensorEntry& e = t.entry[k];
		CHECK(e.grad == l.g[next] && (e.info & sqn::kCountMask) == l.n[next] && (int) (e.info >> 58 & 3) == l.tg[next]);
		CHECK(e.tile0 == tiles);
		tiles += (l.n[next] + tile - 1) / tile;
		if (step) CHECK(e.param == l.p[next] && (int) (e.info >> 56 & 3) == l.tp[next]);
		next++;
	}
	CHECK(t.a.tiles == tiles);
}

static void covers(const std::vector<size_t>& sizes, int bits, unsigned seed)
{
	Lists l(sizes, 0, seed);
	std::vector<size_t> offset(sizes.size() + 1);
	const size_t state = stochqn_hip_tensors_state(l.params, offset.data());
	size_t at = 0, all = 0;
	for (size_t i = 0; i < sizes.size(); i++) { CHECK(offset[i] == at && at % 128 == 0); at += (sizes[i] + 127) / 128 * 128; all += sizes[i]; }
	CHECK(state == at);
	stochqn_hip_adamw_setup s = l.setup(bits);
	std::vector<unsigned char> decay(sizes.size() + 1, 1);
	if (!sizes.empty()) decay[sizes.size() / 2] = 0;
	s.decay = decay.data();
	stochqn_hip_adamw* o = stochqn_hip_adamw_create(l.params, &s);
	CHECK(o);
	decay.assign(decay.size(), 1);                                            // copied, not referred to
	g_launches.clear();
	CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, nullptr, nullptr, nullptr) == 0);
	size_t next = 0;
	CHECK(!g_launches.empty());
	for (size_t k = 0; k < g_launches.size(); k++) {
		const Launch& q = g_launches[k];
		CHECK(q.kind == 'a' && q.bits == bits && q.grid >= 1 && (q.a.a.last != 0) == (k + 1 == g_launches.size()));
		const size_t before = next;
		check_table(l, offset, next, q.a, q.tile, true);
		size_t i = before;
		for (int e = 0; e < q.a.a.entries; e++, i++) {
			while (!l.n[i]) i++;
			CHECK((q.a.a.block_base + q.a.entry[e].block0) * 128 == offset[i]);
			CHECK((q.a.entry[e].info >> 60 & 1) == (i == sizes.size() / 2));
		}
		CHECK((uint64_t) q.grid <= std::max<uint64_t>(q.a.a.tiles, 1));
	}
	while (next < l.n.size() && !l.n[next]) next++;
	CHECK(next == l.n.size());
	stochqn_hip_adamw_destroy(o);

	for (int ranks : {1, 2}) {
		g_ranks = ranks;
		const size_t work = stochqn_hip_tensors_norm_work(l.grads);
		float* out = (float*) device_block(8);
		double* w = (double*) device_block(work * 8);
		g_launches.clear();
		CHECK(stochqn_hip_tensors_norm(l.grads, 1.0, INFINITY, out, w, nullptr) == 0);
		next = 0;
		size_t parts = 0;
		bool finished = false;
		for (const Launch& q : g_launches) {
			if (q.kind == 'n') {
				check_table(l, offset, next, q.n, q.tile, false);
				CHECK(!finished && (q.out ? q.grid == 1 && q.n.a.tiles <= 1 : (uint64_t) q.grid <= q.n.a.tiles));
				CHECK(q.out || q.n.a.part == w + 1 + parts);
				parts += q.grid;
				CHECK(q.out || 1 + parts <= work);
				finished = q.out;
			} else if (q.kind == 's') {
				CHECK(!finished && q.count == (int) parts && q.out == (ranks == 1));
				finished = q.out;
			} else { CHECK(q.kind == 'v' && ranks == 2 && !finished); finished = true; }
		}
		CHECK(finished);
		while (next < l.n.size() && !l.n[next]) next++;
		CHECK(next == l.n.size());
		g_ranks = 1;
	}
}

static void refusals()
{
	Lists l({1000, 50, 0, 7});
	int one = 0, bad_type = 3;
	size_t n = 1000, far = (size_t) 1 << 42;
	float host[8];
	void* ptr = host;
	CHECK(!stochqn_hip_tensors_create(1, &ptr, &n, &one));
	ptr = nullptr;
	CHECK(!stochqn_hip_tensors_create(1, &ptr, &n, &one));
	ptr = device_block(3999);
	CHECK(!stochqn_hip_tensors_create(1, &ptr, &n, &one));                     // past the end by one byte
	ptr = (char*) device_block(5000) + 2;
	CHECK(!stochqn_hip_tensors_create(1, &ptr, &n, &one));                     // misaligned
	CHECK(!stochqn_hip_tensors_create(1, &ptr, &n, &bad_type));
	CHECK(!stochqn_hip_tensors_create(1, &ptr, &far, &one));
	CHECK(!stochqn_hip_tensors_create(-1, &ptr, &n, &one) && !stochqn_hip_tensors_create(1, nullptr, &n, &one));
	{
		void* two[2] = {device_block(4000, 0), device_block(4000, 1)};
		size_t ns[2] = {1000, 1000};
		int ts[2] = {0, 0};
		CHECK(!stochqn_hip_tensors_create(2, two, ns, ts));                       // two devices
	}
	stochqn_hip_adamw_setup good = l.setup(32);
	const auto refused = [&](auto&& change) {
		stochqn_hip_adamw_setup s = good;
		change(s);
		stochqn_hip_adamw* o = stochqn_hip_adamw_create(l.params, &s);
		const bool no = !o;
		stochqn_hip_adamw_destroy(o);
		return no;
	};
	CHECK(!refused([](auto&) {}));
	CHECK(refused([](auto& s) { s.beta1 = 1; }) && refused([](auto& s) { s.beta2 = -0.1; }) && refused([](auto& s) { s.beta2 = NAN; }));
	CHECK(refused([](auto& s) { s.eps = 0; }) && refused([](auto& s) { s.eps = 1e-39; }) && refused([](auto& s) { s.eps = 1e39; }) && refused([](auto& s) { s.weight_decay = INFINITY; }));
	CHECK(refused([](auto& s) { s.state_bits = 16; }) && refused([](auto& s) { s.state_bits = 8; }) && refused([](auto& s) { s.m_scale = (unsigned char*) device_block(100); }));
	CHECK(refused([](auto& s) { s.m = nullptr; }) && refused([](auto& s) { s.count = nullptr; }) && refused([](auto& s) { s.work = nullptr; }));
	CHECK(refused([](auto& s) { s.v = s.m; }) && refused([](auto& s) { s.m = (char*) s.m + 4; }) && refused([&](auto& s) { s.master = (float*) l.p[0]; }));
	CHECK(refused([](auto& s) { s.m = device_block(16); }) && refused([](auto& s) { s.m = device_block(1 << 16, 1); }) && refused([](auto& s) { s.stochastic = 1; }));
	CHECK(!refused([](auto& s) { s.eps = 0x1p126; }) && refused([](auto& s) { s.eps = 0x1.000002p126; }) && refused([](auto& s) { s.eps = 3e38; }));      // its reciprocal is subnormal
	stochqn_hip_adamw* o = stochqn_hip_adamw_create(l.params, &good);
	CHECK(o);
	g_launches.clear();
	CHECK(stochqn_hip_adamw_step(nullptr, l.grads, 0.1, nullptr, nullptr, nullptr) == -1000);
	CHECK(stochqn_hip_adamw_step(o, nullptr, 0.1, nullptr, nullptr, nullptr) == -1000);
	CHECK(stochqn_hip_adamw_step(o, l.grads, NAN, nullptr, nullptr, nullptr) == -1000);
	CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, host, nullptr, nullptr) == -1000);
	CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, nullptr, (float*) device_block(8, 1), nullptr) == -1000);
	CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, nullptr, nullptr, (void*) 0x100) == -1000);      // a stream of device 1
	CHECK(stochqn_hip_adamw_step(o, l.params, 0.1, nullptr, nullptr, nullptr) == -1000);
	{
		Lists other({1000, 50, 7}), longer({1000, 51, 0, 7});
		CHECK(stochqn_hip_adamw_step(o, other.grads, 0.1, nullptr, nullptr, nullptr) == -1000);
		CHECK(stochqn_hip_adamw_step(o, longer.grads, 0.1, nullptr, nullptr, nullptr) == -1000);
		Lists away({1000, 50, 0, 7}, 1);
		CHECK(stochqn_hip_adamw_step(o, away.grads, 0.1, nullptr, nullptr, nullptr) == -1000);
	}
	{	// a gradient that reaches into m from below, and one that begins inside it
		std::vector<void*> g = l.g;
		const uintptr_t block = (uintptr_t) device_block(100000);
		for (long shift : {-1996l, 0l, 400l}) {
			stochqn_hip_adamw_setup s = good;
			s.m = (void*) (block + 40960);
			stochqn_hip_adamw* q = stochqn_hip_adamw_create(l.params, &s);
			g[0] = (void*) (block + 40960 + shift);
			const int rebound = stochqn_hip_tensors_rebind(l.grads, g.data());
			CHECK(q && rebound == 0);
			CHECK(stochqn_hip_adamw_step(q, l.grads, 0.1, nullptr, nullptr, nullptr) == -1000);
			stochqn_hip_adamw_destroy(q);
		}
		CHECK(stochqn_hip_tensors_rebind(l.grads, l.g.data()) == 0);
	}
	CHECK(g_launches.empty());
	void* hosts[4] = {host, host, nullptr, host};
	CHECK(stochqn_hip_tensors_rebind(l.grads, hosts) == -1000);                // and the list is as before:
	g_fail_launch = true;
	CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, nullptr, nullptr, nullptr) == -1000);
	g_fail_launch = false;
	g_launches.clear();
	CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, nullptr, nullptr, (void*) 0x1) == 0 && g_launches.size() == 1 && g_launches[0].a.entry[0].grad == l.g[0]);
	float* out = (float*) device_block(8);
	double* work = (double*) device_block(8 * stochqn_hip_tensors_norm_work(l.grads));
	CHECK(stochqn_hip_tensors_norm(l.grads, 1, 0, out, work, nullptr) == -1000 && stochqn_hip_tensors_norm(l.grads, NAN, 1, out, work, nullptr) == -1000);
	CHECK(stochqn_hip_tensors_norm(l.grads, 1, 1, host, work, nullptr) == -1000 && stochqn_hip_tensors_norm(l.grads, 1, 1, out, (double*) device_block(8), nullptr) == -1000);
	CHECK(stochqn_hip_tensors_norm(l.grads, 1, 1, out, nullptr, nullptr) == -1000);
	g_ranks = 2;
	g_fail_reduce = true;
	CHECK(stochqn_hip_tensors_norm(l.grads, 1, 1, out, work, nullptr) == -1000);
	g_fail_reduce = false;
	// a sum that the host forms is not captured: refused in front of the first launch; any other call goes on
	for (bool capturing : {false, true})
		for (bool host_side : {false, true})
			for (int ranks : {1, 2}) {
				g_capturing = capturing;
				g_on_the_host = host_side;
				g_ranks = ranks;
				g_launches.clear();
				const int rc = stochqn_hip_tensors_norm(l.grads, 1, 1, out, work, nullptr);
				const bool no = capturing && host_side && ranks == 2;
				CHECK(rc == (no ? -1000 : 0) && g_launches.empty() == no);
				CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, nullptr, nullptr, nullptr) == 0);
			}
	g_capturing = g_on_the_host = false;
	g_ranks = 1;
	// another current device: the launches go to the tensors', and the caller's is current again
	{
		Lists away({5000}, 3);
		stochqn_hip_adamw_setup s = away.setup(8, 3);
		stochqn_hip_adamw* q = stochqn_hip_adamw_create(away.params, &s);
		g_launches.clear();
		CHECK(q && stochqn_hip_adamw_step(q, away.grads, 0.1, nullptr, nullptr, nullptr) == 0);
		CHECK(g_launches.size() == 1 && g_launches[0].on == 3 && g_device == 0);
		stochqn_hip_adamw_destroy(q);
	}
	// every HIP call failing in turn: an error or the same launches, never anything else
	for (int k = 0; k < 200; k++) {
		g_fail_after = k;
		stochqn_hip_tensors* t = stochqn_hip_tensors_create(4, l.p.data(), l.n.data(), l.tp.data());
		stochqn_hip_adamw* q = t ? stochqn_hip_adamw_create(t, &good) : nullptr;
		g_launches.clear();
		const int rc = q ? stochqn_hip_adamw_step(q, l.grads, 0.1, nullptr, out, nullptr) : -1000;
		CHECK((rc == 0 && g_launches.size() == 1) || (rc == -1000 && g_launches.empty()));
		const int rn = stochqn_hip_tensors_norm(l.grads, 1, 1, out, work, nullptr);
		CHECK(rn == 0 || rn == -1000);
		g_fail_after = -1;
		CHECK(g_device == 0);
		stochqn_hip_adamw_destroy(q);
		stochqn_hip_tensors_destroy(t);
	}
	stochqn_hip_adamw_destroy(o);
}

// what a call reads or writes besides the tensors does not overlap what it writes
static void overlaps_in_a_call()
{
	Lists l({1000, 50, 0, 7});
	const size_t blocks = stochqn_hip_tensors_state(l.params, nullptr) / 128;
	for (int bits : {32, 8}) {
		stochqn_hip_adamw_setup s = l.setup(bits);
		stochqn_hip_adamw* o = stochqn_hip_adamw_create(l.params, &s);
		CHECK(o);
		float* apart = (float*) device_block(8);
		std::vector<void*> written{l.p[0], l.p[3], s.m, (char*) s.m + blocks * 128 * bits / 8 - 4, s.v, s.master, s.count, (char*) s.count + 12, s.work, (char*) s.work + 4092};
		if (bits == 8) written.push_back((void*) (((uintptr_t) s.m_scale + 3) & ~(uintptr_t) 3));
		g_launches.clear();
		for (void* p : written) {
			CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, (float*) p, apart, nullptr) == -1000);
			CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, apart, (float*) p, nullptr) == -1000);
		}
		CHECK(g_launches.empty());
		CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, apart, apart + 1, nullptr) == 0 && stochqn_hip_adamw_step(o, l.grads, 0.1, apart, apart, nullptr) == 0);
		CHECK(stochqn_hip_adamw_step(o, l.grads, 0.1, (float*) l.g[0], nullptr, nullptr) == 0);        // the step only reads gradients
		stochqn_hip_adamw_destroy(o);
	}
	const size_t doubles = stochqn_hip_tensors_norm_work(l.grads);
	char* work = (char*) device_block(8 * doubles + 8);
	float* out = (float*) device_block(16);
	const auto norm = [&](void* to, void* with) { return stochqn_hip_tensors_norm(l.grads, 1, 1, (float*) to, (double*) with, nullptr); };
	g_launches.clear();
	CHECK(norm(work, work) == -1000 && norm(work + 8 * doubles - 4, work) == -1000 && norm(l.g[0], work) == -1000 && norm((char*) l.g[1] + 4, work) == -1000);
	CHECK(norm(out, (void*) (((uintptr_t) l.g[0] + 7) & ~(uintptr_t) 7)) == -1000);
	CHECK(g_launches.empty());
	CHECK(norm(work + 8 * doubles, work) == 0 && norm(out, work) == 0 && norm(l.p[0], work) == 0);
}

// which tile a list's sizes choose, on both sides of every threshold (the stand-in device has 256 units)
static void tiles_by_size()
{
	const auto step = [](const std::vector<size_t>& n, int bits) {
		Lists l(n);
		stochqn_hip_adamw_setup s = l.setup(bits);
		stochqn_hip_adamw* o = stochqn_hip_adamw_create(l.params, &s);
		g_launches.clear();
		CHECK(o && stochqn_hip_adamw_step(o, l.grads, 0.1, nullptr, nullptr, nullptr) == 0);
		stochqn_hip_adamw_destroy(o);
		return g_launches[0];
	};
	const auto norm = [](const std::vector<size_t>& n) {
		Lists l(n);
		float* out = (float*) device_block(8);
		double* work = (double*) device_block(8 * stochqn_hip_tensors_norm_work(l.grads));
		g_launches.clear();
		CHECK(stochqn_hip_tensors_norm(l.grads, 1, 1, out, work, nullptr) == 0);
		return g_launches[0];
	};
	const size_t units = 256;
	for (int bits : {32, 8}) {
		const size_t tile = bits == 32 ? sqn::kTile32 : sqn::kTile8, few = (bits == 32 ? 64 : 32) * units * tile;
		CHECK(step({few - tile}, bits).tile == sqn::kTileSmall && step({few - tile + 1}, bits).tile == (int) tile && step({few - 2 * tile, 1}, bits).tile == sqn::kTileSmall);
		CHECK(step({few - 2 * tile, 1, 1}, bits).tile == (int) tile);
		const size_t most = bits == 32 ? 16 * units : 32 * units;              // workgroups; a list with more tiles goes round
		CHECK(step({few}, bits).grid == (int) most && step({2 * few}, bits).grid == (int) most && step({most * sqn::kTileSmall - 1, 1}, bits).grid == (int) most);
		CHECK(step({most * sqn::kTileSmall - sqn::kTileSmall}, bits).grid == (int) most - 1);
	}
	CHECK(norm({2 * units * sqn::kTileNormMid - sqn::kTileNormMid}).tile == sqn::kTileSmall && norm({2 * units * sqn::kTileNormMid}).tile == sqn::kTileNormMid);
	CHECK(norm({4 * units * sqn::kTileNorm - sqn::kTileNorm}).tile == sqn::kTileNormMid && norm({4 * units * sqn::kTileNorm}).tile == sqn::kTileNorm);
	CHECK(norm({9 * units * sqn::kTileNorm}).grid == (int) (8 * units));
}

// A list that two optimizers read while a third thread rebinds it and a fourth takes its norm: every table is of one binding or the other.
static void concurrent()
{
	Lists l({3000, 40, 0, 70000}, 0, 1);
	std::vector<void*> other;
	for (size_t i = 0; i < l.n.size(); i++) other.push_back(l.n[i] ? device_block(l.n[i] * 4) : nullptr);
	stochqn_hip_adamw_setup a = l.setup(8);
	Lists m({3000, 40, 0, 70000}, 0, 2);
	stochqn_hip_adamw_setup b = m.setup(32);
	stochqn_hip_adamw *o = stochqn_hip_adamw_create(l.params, &a), *q = stochqn_hip_adamw_create(m.params, &b);
	float* out = (float*) device_block(8);
	double* work = (double*) device_block(8 * stochqn_hip_tensors_norm_work(l.grads));
	CHECK(o && q);
	g_launches.clear();
	const auto many = [](auto&& f) { for (int k = 0; k < 300; k++) CHECK(f(k) == 0); };
	std::thread t[] = {
		std::thread([&] { many([&](int) { return stochqn_hip_adamw_step(o, l.grads, 0.1, nullptr, nullptr, nullptr); }); }),
		std::thread([&] { many([&](int) { return stochqn_hip_adamw_step(o, l.grads, 0.1, nullptr, nullptr, nullptr); }); }),
		std::thread([&] { many([&](int) { return stochqn_hip_adamw_step(q, l.grads, 0.1, nullptr, nullptr, nullptr); }); }),
		std::thread([&] { many([&](int k) { return stochqn_hip_tensors_rebind(l.grads, k & 1 ? l.g.data() : other.data()); }); }),
		std::thread([&] { many([&](int) { return stochqn_hip_tensors_norm(l.grads, 1, 1, out, work, nullptr); }); }),
	};
	for (std::thread& x : t) x.join();
	for (const Launch& x : g_launches) {
		if (x.kind == 's') continue;
		const sqn::TensorEntry* e = x.kind == 'a' ? x.a.entry : x.n.entry;
		const std::vector<void*>& from = e[0].grad == l.g[0] ? l.g : other;
		CHECK(e[0].grad == from[0] && e[1].grad == from[1] && e[2].grad == from[3]);
	}
	stochqn_hip_adamw_destroy(o);
	stochqn_hip_adamw_destroy(q);
}

// Two ranks of one process that take the norm of one list at once: a list must not be held while its rank waits for the other.
static void two_ranks_of_one_list()
{
	Lists l({3000, 40});
	const size_t bytes = 8 * stochqn_hip_tensors_norm_work(l.grads);
	g_ranks = 2;
	g_meeting = true;
	const auto rank = [&](float* out, double* work) { for (int k = 0; k < 3; k++) CHECK(stochqn_hip_tensors_norm(l.grads, 1, 1, out, work, nullptr) == 0); };
	float *one = (float*) device_block(8), *two = (float*) device_block(8);
	double *w1 = (double*) device_block(bytes), *w2 = (double*) device_block(bytes);
	std::thread a([&] { rank(one, w1); }), b([&] { rank(two, w2); });
	a.join();
	b.join();
	CHECK(g_arrived == 6);
	g_ranks = 1;
	g_meeting = false;
}

int main(int argc, char**)
{
	if (argc > 1) { concurrent(); two_ranks_of_one_list(); std::printf("ok\n"); return 0; }
	for (int bits : {32, 8}) {
		covers({}, bits, 0);
		covers({0, 0, 0}, bits, 0);
		covers({1}, bits, 1);
		covers({2048, 2049, 1, 0, 8192, 8193}, bits, 2);
		covers(std::vector<size_t>(111, 5), bits, 3);
		covers(std::vector<size_t>(112, 5), bits, 4);
		covers(std::vector<size_t>(113, 5), bits, 5);
		covers({(size_t) 1 << 33, 77, ((size_t) 1 << 31) + 5}, bits, 6);
		covers(std::vector<size_t>(20, (size_t) 1 << 33), bits, 7);              // more tiles than one launch of several tensors counts
		std::mt19937 r(8);
		for (int k = 0; k < 20; k++) {
			std::vector<size_t> n;
			for (int i = (int) (r() % 400); i > 0; i--) n.push_back(r() % 4 ? r() % (r() % 5 ? 3000 : 3000000) : 0);
			covers(n, bits, k);
		}
	}
	tiles_by_size();
	refusals();
	overlaps_in_a_call();
	std::printf("ok\n");
	return 0;
}
