// hip_stub.cpp's runtime with two devices, and what the launches of the packed and
// 4-bit attention carry: their sequences, splits and partials, and the device
// that was current at a launch or an allocation.
#define hipLaunchKernel base_launch_kernel
#define hipGetDeviceCount base_get_device_count
#define hipGetDevice base_get_device
#define hipSetDevice base_set_device
#define hipMalloc base_malloc
#include "hip_stub.cpp"
#undef hipLaunchKernel
#undef hipGetDeviceCount
#undef hipGetDevice
#undef hipSetDevice
#undef hipMalloc

namespace
{
	struct flash
	{
		bool is_flash = false, merge = false;
		nnchip::flash_params p;
		nnchip::flash_seqs<nnchip::kFlashSeqs> s;
		unsigned block, device;
	};
	std::vector<flash> g_flash; // beside g_launches
	int g_device = 0, g_malloc_devices = 0; // a bit per device that was current at an allocation

	template <int N>
	void take(flash& f, void** args)
	{
		f.p = *static_cast<nnchip::flash_params*>(args[0]);
		const auto& s = *static_cast<nnchip::flash_seqs<N>*>(args[1]);
		f.s.n = s.n;
		f.s.key_groups = s.key_groups;
		for (int i = 0; i < s.n; ++i)
		{
			f.s.start[i] = s.start[i];
			f.s.len[i] = s.len[i];
			f.s.tile[i] = s.tile[i];
			f.s.split[i] = s.split[i];
			f.s.part[i] = s.part[i];
		}
	}
}

extern "C" {

void stub_flash_clear()
{
	g_flash.clear();
	g_malloc_devices = 0;
	stub_clear();
}
int stub_malloc_devices() { return g_malloc_devices; }
int stub_device() { return g_device; }
// Launch i: 0 another kernel, 1 attention, 2 its merge; then the device, the grid,
// threads, sequences, key groups, heads, KV heads, head_dim.
void stub_flash(int i, long long* out)
{
	const flash& f = g_flash[i];
	const long long v[9] = {f.is_flash ? f.merge ? 2 : 1 : 0, f.device, g_launches[i].grid.x, f.block, f.s.n, f.s.key_groups,
	                        f.p.n_head, f.p.n_kv, f.p.head_dim};
	std::memcpy(out, v, sizeof v);
}
const void* stub_flash_part(int i) { return g_flash[i].p.part; }
const void* stub_symbol() { return g_symbol; }
// Sequence s of launch i: start, length, first tile, splits, first row of its partials.
void stub_flash_seq(int i, int s, int* out)
{
	const auto& q = g_flash[i].s;
	const int v[5] = {q.start[s], q.len[s], q.tile[s], q.split[s], q.part[s]};
	std::memcpy(out, v, sizeof v);
}

hipError_t hipMalloc(void** p, size_t n)
{
	g_malloc_devices |= 1 << g_device;
	return base_malloc(p, n);
}
hipError_t hipGetDeviceCount(int* n)
{
	*n = 2;
	return hipSuccess;
}
hipError_t hipGetDevice(int* d)
{
	*d = g_device;
	return hipSuccess;
}
hipError_t hipSetDevice(int d)
{
	g_device = d;
	return hipSuccess;
}
hipError_t hipLaunchKernel(const void* fn, dim3 grid, dim3 block, void** args, size_t lds, hipStream_t stream)
{
	const hipError_t e = base_launch_kernel(fn, grid, block, args, lds, stream);
	flash f{};
	const std::string& name = g_launches.back().name;
	f.block = block.x;
	f.device = static_cast<unsigned>(g_device);
	f.is_flash = name.find("flash_params") != std::string::npos;
	f.merge = name.find("flash_merge") != std::string::npos;
	if (f.is_flash && name.find("ELi1EEEv") != std::string::npos) take<1>(f, args); // (the sequences: the last template argument)
	else if (f.is_flash) take<nnchip::kFlashSeqs>(f, args);
	g_flash.push_back(f);
	return e;
}
}
