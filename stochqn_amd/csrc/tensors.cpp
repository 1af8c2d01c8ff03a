// tensors.cpp -- C entry points of the first-order steps over the tensors of a model (include/stochqn_hip.h: "first-order steps"):
// lists of tensors, the AdamW step, the norm over a list.  Plans are checked when they are made; a step only fills the table that its
// kernels take by value and launches them on the caller's stream: no allocation, no copy, no synchronisation.
#include "tensors.hpp"
#include "runtime.hpp"
#include "stochqn_hip.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <memory>
#include <mutex>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

using namespace sqn;

namespace {

// Most workgroups per compute unit.  Measured at 1.28e9 elements: 32-bit moments 6.51 ms with 8, 6.50 with 16 (at 7.7e6 elements
// 43.3 and 40.3 us); 8-bit moments 2.53 ms with 8, 2.47 with 16, 2.44 with 32, 2.46 with 64; the norm 466 us with 4, 377 with 8,
// 379 with 16.
constexpr int kPerUnit32 = 16, kPerUnit8 = 32, kPerUnitNorm = 8;

struct Range { const char* at; size_t bytes; };                              // of device memory
bool before(const Range& a, const Range& b) { return a.at < b.at; }
bool overlap(const Range& a, const Range& b) { return a.at < b.at + b.bytes && b.at < a.at + a.bytes; }
// with one of the sorted ranges that do not overlap each other
bool overlaps(const std::vector<Range>& sorted, const Range& r)
{
	const auto after = std::upper_bound(sorted.begin(), sorted.end(), r, before);
	return (after != sorted.end() && overlap(r, *after)) || (after != sorted.begin() && overlap(r, *(after - 1)));
}

struct Item { void* p; size_t n; int type; };

std::atomic<unsigned long long> g_versions{0};

// Refused input: the message goes to stderr, the entry returns -1000 / NULL (what the library does everywhere).
struct Refused : std::runtime_error { using std::runtime_error::runtime_error; };
[[noreturn]] void refuse(const std::string& why) { throw Refused(why); }

template <class R, class F> R guarded(const char* who, R failed, F&& body)
{
	try {
		return body();
	} catch (const std::exception& e) {
		std::fprintf(stderr, "stochqn: %s: %s\n", who, e.what());
	} catch (...) {
		std::fprintf(stderr, "stochqn: %s: unexpected failure\n", who);
	}
	(void) hipGetLastError();
	return failed;
}

// device memory of `device` (any, and told, while it is < 0) from p on for `bytes`
void check_memory(const void* p, size_t bytes, int& device, const char* what)
{
	hipPointerAttribute_t at;
	if (!p || hipPointerGetAttributes(&at, p) != hipSuccess || (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged))
		refuse(std::string(what) + " is not device memory");
	if (device >= 0 && at.device != device) refuse(std::string(what) + " lies on another device than the first tensor");
	device = at.device;
	hipDeviceptr_t base = nullptr;
	size_t size = 0;
	if (hipMemGetAddressRange(&base, &size, const_cast<void*>(p)) == hipSuccess) {
		if (static_cast<const char*>(p) + bytes > static_cast<const char*>(base) + size) refuse(std::string(what) + " reaches past the end of its allocation");
	} else (void) hipGetLastError();
}

void check_aligned(const void* p, size_t to, const char* what)
{
	if (reinterpret_cast<uintptr_t>(p) % to) refuse(std::string(what) + " is not aligned to " + std::to_string(to) + " bytes");
}

uint64_t tiles_of(size_t n, int tile) { return (n + tile - 1) / tile; }

// Large tiles keep more loads of a lane in flight; a list with fewer than `few` of them for each compute unit is cut into smaller ones, whose
// kernels need fewer registers (80 against 122, 92 against 156 with 8-bit moments: more waves a unit).  Where the two meet, in us with small and with large tiles at that many large
// tiles a unit (one vector; lists of layers are alike):
//   8-bit moments   f32:         8: 51.1 57.4   16: 103 107   24: 157 156   32: 211 204   48: 323 307   128: 907 816
//                   bf16 alone:  8: 35.7 39.1   16: 63.3 68.0   32: 120 128   48: 190 190   64: 250 250   128: 592 487      -> 32
//   32-bit moments  f32:         8: 42.8 44.9   16: 83.4 85.1   32: 162 165   48: 243 245   64: 318 309   96: 478 455      -> 64
//                   bf16 alone:  8: 34.0 36.0   32: 125 130   64: 245 251   96: 374 371   128: 508 493
//   the norm (small, 8192, 16384 elements; at that many tiles of 16384 a unit)
//                   bf16:  1: 9.1 9.4 8.9   3: 9.5 9.5 9.2   4: 10.6 10.1 10.8   6: 13.2 12.4 13.1   8: 15.7 15.3 15.5   16: 25.5 25.1 24.8   32: 44.7 45.0 43.4
//                   f32:   1: 8.8 9.6 9.5   2: 10.8 10.5 10.1   4: 16.3 16.0 15.8   8: 27.1 26.4 26.3   16: 49.2 47.5 47.4   32: 93.6 89.9 89.4      -> 2 of 8192, 4 of 16384
LaunchShape shape_of(const std::vector<Item>& items, int units, int per_unit, std::initializer_list<std::pair<int, int>> tile_and_few)
{
	for (const auto& [tile, few] : tile_and_few) {
		uint64_t tiles = 0;
		for (const Item& it : items) tiles += tiles_of(it.n, tile);
		if (tiles >= few * (uint64_t) units) return {tile, units * per_unit};
	}
	return {kTileSmall, units * per_unit};
}

size_t blocks_of(size_t n) { return (n + kStateBlock - 1) / kStateBlock; }

// the device of a plan is current for as long as this lives
struct OnDevice {
	int was = -1;
	explicit OnDevice(int device)
	{
		if (hipGetDevice(&was) != hipSuccess) refuse("no current device");
		if (was == device) was = -1;
		else if (hipSetDevice(device) != hipSuccess) refuse("the tensors' device cannot be made current");
	}
	~OnDevice() { if (was >= 0) (void) hipSetDevice(was); }
};

hipStream_t check_stream(void* stream, int device)
{
	hipStream_t st = static_cast<hipStream_t>(stream);
	hipDevice_t on = device;
	if (st && hipStreamGetDevice(st, &on) != hipSuccess) refuse("the stream cannot be used");
	if (on != device) refuse("the stream belongs to another device than the tensors");
	return st;
}

void check_scalar(const void* p, int device, const char* what)
{
	if (!p) return;
	check_aligned(p, sizeof(float), what);
	check_memory(p, sizeof(float), device, what);
}

int launched()
{
	const hipError_t e = hipGetLastError();
	if (e != hipSuccess) refuse(std::string("the launch failed: ") + hipGetErrorString(e));
	return 0;
}

int units_of(int device)
{
	int units = 0;
	if (hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || units <= 0) refuse("the device cannot be asked");
	return units;
}

}  // namespace

struct stochqn_hip_tensors {
	std::mutex mu;                     // rebind against the calls that read the addresses
	std::vector<Item> items;
	int device = -1;
	LaunchShape norm{};                // how the norm cuts the list up
	int units = 0;                     // compute units
	unsigned long long version = 0;    // another one for every set of addresses
};

struct stochqn_hip_adamw {
	std::mutex mu;
	std::vector<Item> items;
	std::vector<unsigned char> no_decay;
	std::vector<size_t> block;         // first block of each tensor's state
	std::vector<Range> written;        // sorted
	stochqn_hip_adamw_setup s;
	int device = -1;
	LaunchShape shape{};
	unsigned long long checked = 0;    // version of the gradients that have been held against `written`
};

namespace {

void set_items(std::vector<Item>& items, int& device, void* const ptr[])
{
	int on = device;
	for (size_t i = 0; i < items.size(); i++) {
		if (!items[i].n) continue;
		const std::string what = "tensor " + std::to_string(i);
		check_aligned(ptr[i], type_size(items[i].type), what.c_str());
		check_memory(ptr[i], items[i].n * type_size(items[i].type), on, what.c_str());
	}
	for (size_t i = 0; i < items.size(); i++) items[i].p = items[i].n ? ptr[i] : nullptr;
	device = on;
}

// Tiles of a launch with several tensors: their blocks are counted in 32 bits (64 to the largest tile).
constexpr uint64_t kMostTiles = 1 << 25;

// The tables of a list, one launch after the other: fill(i, entry) for every tensor with elements, fire(base block, entries, tiles) for every
// table that is full or the last.
template <class Fill, class Fire> void for_launches(const std::vector<Item>& items, int tile, TensorEntry* entry, Fill&& fill, Fire&& fire)
{
	int used = 0;
	uint64_t tiles = 0;
	for (size_t i = 0; i < items.size(); i++) {
		if (!items[i].n) continue;
		const uint64_t mine = tiles_of(items[i].n, tile);
		if (used == kEntries || (used && tiles + mine > kMostTiles)) {
			fire(used, (uint32_t) tiles, false);
			used = 0;
			tiles = 0;
		}
		entry[used].tile0 = (uint32_t) tiles;
		fill(i, used);
		used++;
		tiles += mine;
	}
	fire(used, (uint32_t) tiles, true);
}

}  // namespace

extern "C" {

stochqn_hip_tensors* stochqn_hip_tensors_create(int count, void* const ptr[], const size_t size[], const int type[])
{
	return guarded("stochqn_hip_tensors_create", (stochqn_hip_tensors*) nullptr, [&] {
		if (count < 0 || (count && (!ptr || !size || !type))) refuse("no tensors");
		if (!device_ready()) refuse("no usable HIP device");
		auto t = std::make_unique<stochqn_hip_tensors>();
		for (int i = 0; i < count; i++) {
			if (type[i] < T_F32 || type[i] > T_F16) refuse("tensor " + std::to_string(i) + " has an unknown type");
			if (size[i] > ((size_t) 1 << 41)) refuse("tensor " + std::to_string(i) + " is too large");
			t->items.push_back({nullptr, size[i], type[i]});
		}
		set_items(t->items, t->device, ptr);
		if (t->device < 0 && hipGetDevice(&t->device) != hipSuccess) refuse("no current device");
		t->units = units_of(t->device);
		t->norm = shape_of(t->items, t->units, kPerUnitNorm, {{kTileNorm, 4}, {kTileNormMid, 2}});
		t->version = ++g_versions;
		return t.release();
	});
}

int stochqn_hip_tensors_rebind(stochqn_hip_tensors* t, void* const ptr[])
{
	return guarded("stochqn_hip_tensors_rebind", -1000, [&] {
		if (!t || (!ptr && !t->items.empty())) refuse("no tensors");
		std::lock_guard<std::mutex> lk(t->mu);
		int device = t->device;
		set_items(t->items, device, ptr);
		t->version = ++g_versions;
		return 0;
	});
}

void stochqn_hip_tensors_destroy(stochqn_hip_tensors* t) { delete t; }

size_t stochqn_hip_tensors_state(const stochqn_hip_tensors* t, size_t offset[])
{
	if (!t) return 0;
	size_t blocks = 0;
	for (size_t i = 0; i < t->items.size(); i++) {
		if (offset) offset[i] = blocks * kStateBlock;
		blocks += blocks_of(t->items[i].n);
	}
	return blocks * kStateBlock;
}

size_t stochqn_hip_tensors_norm_work(const stochqn_hip_tensors* t)
{
	if (!t) return 0;
	size_t parts = 0;
	TensorEntry table[kEntries];
	for_launches(t->items, t->norm.tile, table, [](size_t, int) {}, [&](int, uint32_t tiles, bool) { parts += std::min<size_t>(tiles, t->norm.grid); });
	return 1 + parts;
}

int stochqn_hip_tensors_norm(stochqn_hip_tensors* t, double grad_scale, double max_norm, float out[], double work[], void* hip_stream)
{
	return guarded("stochqn_hip_tensors_norm", -1000, [&] {
		if (!t || !out || !work) refuse("an argument is NULL");
		if (!std::isfinite(grad_scale)) refuse("grad_scale is not finite");
		if (!(max_norm > 0)) refuse("max_norm is not positive");
		std::unique_lock<std::mutex> lk(t->mu);
		int device = t->device;
		check_aligned(out, sizeof(float), "out");
		check_aligned(work, sizeof(double), "work");
		const Range result{reinterpret_cast<const char*>(out), 2 * sizeof(float)};
		const Range scratch{reinterpret_cast<const char*>(work), stochqn_hip_tensors_norm_work(t) * sizeof(double)};
		check_memory(out, result.bytes, device, "out");
		check_memory(work, scratch.bytes, device, "work");
		if (overlap(result, scratch)) refuse("out overlaps work");
		for (const Item& it : t->items) {
			const Range r{static_cast<const char*>(it.p), it.n * type_size(it.type)};
			if (it.n && (overlap(r, result) || overlap(r, scratch))) refuse("out or work overlaps a tensor");
		}
		OnDevice on(device);
		hipStream_t st = check_stream(hip_stream, device);
		const bool reduced = comm_nranks() > 1;
		if (reduced && reduces_on_the_host()) {
			hipStreamCaptureStatus capture;
			if (hipStreamIsCapturing(st, &capture) != hipSuccess || capture != hipStreamCaptureStatusNone) refuse("the ranks' sums are formed on the host: they cannot be captured");
		}
		(void) hipGetLastError();                                  // somebody else's: only what the launches below leave counts
		Table<NormArgs, kEntries> table;
		NormArgs& a = table.a;
		a.grad_scale = grad_scale;
		a.max_norm = max_norm;
		int parts = 0, launches = 0;
		bool done = false;
		for_launches(t->items, t->norm.tile, table.entry,
			[&](size_t i, int k) {
				table.entry[k].grad = t->items[i].p;
				table.entry[k].info = entry_info(t->items[i].n, 0, t->items[i].type, false);
			},
			[&](int used, uint32_t tiles, bool) {
				a.entries = used;
				a.tiles = tiles;
				a.part = work + 1 + parts;
				done = tiles <= 1 && !launches && !reduced;             // one workgroup sees everything: it finishes
				a.out = done ? out : nullptr;
				const int grid = (int) std::min<size_t>(done ? 1 : tiles, t->norm.grid);
				if (grid) launch_norm(st, t->norm.tile, grid, table);
				parts += grid;
				launches++;
			});
		lk.unlock();                                                // the launches have the addresses; a reducer may wait for a thread that wants this list
		if (!done) launch_norm_sum(st, work, parts, grad_scale, max_norm, reduced ? nullptr : out);
		if (reduced) {
			if (!reduce_in_place(work, 1, st)) refuse("the reduction over the ranks failed");
			launch_norm_verdict(st, work, grad_scale, max_norm, out);
		}
		return launched();
	});
}

stochqn_hip_adamw* stochqn_hip_adamw_create(stochqn_hip_tensors* params, const stochqn_hip_adamw_setup* setup)
{
	return guarded("stochqn_hip_adamw_create", (stochqn_hip_adamw*) nullptr, [&] {
		if (!params || !setup) refuse("an argument is NULL");
		const stochqn_hip_adamw_setup& s = *setup;
		if (!(s.beta1 >= 0 && s.beta1 < 1) || !(s.beta2 >= 0 && s.beta2 < 1)) refuse("beta1 and beta2 lie in [0, 1)");
		if (!(s.eps >= FLT_MIN && s.eps <= 1 / FLT_MIN)) refuse("eps lies in 2^-126 .. 2^126");       // sqrt(v) adds nothing to the largest, whose reciprocal is not subnormal
		if (!std::isfinite(s.weight_decay)) refuse("weight_decay is not finite");
		if (s.state_bits != 32 && s.state_bits != 8) refuse("state_bits is 32 or 8");
		if (s.state_bits == 32 && (s.m_scale || s.v_scale)) refuse("moments in 32 bits have no scales");
		if (s.stochastic && s.master) refuse("stochastic rounding is for weights without f32 weights beside them");
		auto o = std::make_unique<stochqn_hip_adamw>();
		std::lock_guard<std::mutex> lk(params->mu);
		o->items = params->items;
		o->device = params->device;
		o->shape = s.state_bits == 8 ? shape_of(o->items, params->units, kPerUnit8, {{kTile8, 32}}) : shape_of(o->items, params->units, kPerUnit32, {{kTile32, 64}});
		o->s = s;
		size_t blocks = 0;
		for (size_t i = 0; i < o->items.size(); i++) {
			const Item& it = o->items[i];
			if (it.type == T_F16 && s.stochastic) refuse("stochastic rounding is for bf16 weights (tensor " + std::to_string(i) + " is f16)");
			o->no_decay.push_back(s.decay && !s.decay[i]);
			o->block.push_back(blocks);
			blocks += blocks_of(it.n);
			if (it.n) o->written.push_back({static_cast<char*>(it.p), it.n * type_size(it.type)});
		}
		o->s.decay = nullptr;
		if (!s.count || !s.work || (blocks && (!s.m || !s.v || (s.state_bits == 8 && (!s.m_scale || !s.v_scale))))) refuse("an array of the state is NULL");
		const size_t state = blocks * kStateBlock, moment = state * (s.state_bits / 8);
		const auto array = [&](const void* p, size_t bytes, size_t to, const char* what) {
			if (!p || !bytes) return;
			check_aligned(p, to, what);
			check_memory(p, bytes, o->device, what);
			o->written.push_back({static_cast<const char*>(p), bytes});
		};
		array(s.m, moment, 16, "m");
		array(s.v, moment, 16, "v");
		array(s.m_scale, s.state_bits == 8 ? blocks : 0, 1, "m_scale");
		array(s.v_scale, s.state_bits == 8 ? blocks : 0, 1, "v_scale");
		array(s.master, state * sizeof(float), 16, "master");
		array(s.count, 2 * sizeof(long long), 8, "count");
		array(s.work, kGates * kGateStride, 8, "work");
		std::sort(o->written.begin(), o->written.end(), before);
		for (size_t i = 1; i < o->written.size(); i++)
			if (o->written[i - 1].at + o->written[i - 1].bytes > o->written[i].at) refuse("two arrays that the step writes overlap");
		return o.release();
	});
}

void stochqn_hip_adamw_destroy(stochqn_hip_adamw* o) { delete o; }

int stochqn_hip_adamw_step(stochqn_hip_adamw* o, stochqn_hip_tensors* grads, double step_size, const float* step_size_dev,
                           const float* grad_scale, void* hip_stream)
{
	return guarded("stochqn_hip_adamw_step", -1000, [&] {
		if (!o || !grads) refuse("an argument is NULL");
		if (!step_size_dev && !std::isfinite(step_size)) refuse("step_size is not finite");
		std::lock_guard<std::mutex> lk(o->mu);
		std::lock_guard<std::mutex> lg(grads->mu);
		const std::vector<Item>& g = grads->items;
		if (g.size() != o->items.size()) refuse("as many gradients as parameters are wanted");
		for (size_t i = 0; i < g.size(); i++)
			if (g[i].n != o->items[i].n) refuse("gradient " + std::to_string(i) + " has another size than its parameter");
		if (o->checked != grads->version) {
			if (grads->device != o->device) refuse("the gradients lie on another device than the parameters");
			for (size_t i = 0; i < g.size(); i++) {
				if (!g[i].n) continue;
				const Range r{static_cast<char*>(g[i].p), g[i].n * type_size(g[i].type)};
				if (overlaps(o->written, r)) refuse("gradient " + std::to_string(i) + " overlaps an array that the step writes");
			}
			o->checked = grads->version;
		}
		check_scalar(step_size_dev, o->device, "step_size");
		check_scalar(grad_scale, o->device, "grad_scale");
		for (const float* scalar : {step_size_dev, grad_scale})             // read by every workgroup, whatever others have written by then
			if (scalar && overlaps(o->written, {reinterpret_cast<const char*>(scalar), sizeof(float)})) refuse("step_size or grad_scale overlaps an array that the step writes");
		OnDevice on(o->device);
		hipStream_t st = check_stream(hip_stream, o->device);
		(void) hipGetLastError();
		const stochqn_hip_adamw_setup& s = o->s;
		Table<AdamwArgs, kEntries> table;
		AdamwArgs& a = table.a;
		a.master = s.master;
		a.m = s.m;
		a.v = s.v;
		a.m_scale = s.m_scale;
		a.v_scale = s.v_scale;
		a.count = s.count;
		a.gates = static_cast<char*>(s.work);
		a.grad_scale = grad_scale;
		a.step_size_dev = step_size_dev;
		a.step_size = step_size;
		a.beta1 = s.beta1;
		a.beta2 = s.beta2;
		a.weight_decay = s.weight_decay;
		a.eps = (float) s.eps;
		a.seed = s.seed;
		a.stochastic = s.stochastic;
		for_launches(o->items, o->shape.tile, table.entry,
			[&](size_t i, int k) {
				TensorEntry& e = table.entry[k];
				if (!k) a.block_base = o->block[i];
				e.param = o->items[i].p;
				e.grad = g[i].p;
				e.info = entry_info(g[i].n, o->items[i].type, g[i].type, o->no_decay[i]);
				e.block0 = (uint32_t) (o->block[i] - a.block_base);
			},
			[&](int used, uint32_t tiles, bool last) {
				a.entries = used;
				a.tiles = tiles;
				a.last = last;
				launch_adamw(st, s.state_bits, o->shape.tile, (int) std::min<size_t>(std::max<uint32_t>(tiles, 1), o->shape.grid), table);
			});
		return launched();
	});
}

}  // extern "C"
