# Build of the MI355X (gfx950) hot-path library.  `python -c "import __graft_entry__ as g; g.build()"`
# runs this Makefile.
HIPCC ?= /opt/rocm/bin/hipcc
ARCH  ?= gfx950
# packed float32 operations stay off: some of their forms have given wrong results on gfx950
NOPK     = -Xclang -target-feature -Xclang -packed-fp32-ops
HIPFLAGS = -O3 -std=c++17 --offload-arch=$(ARCH) -fPIC -Wall -Wno-unused-result $(NOPK)

LIB  = v2e2v_amd/libcista_hip.so
OBJ  = build/cista_abi.o build/cista_voxel.o build/cista_ssim.o build/cista_v2e.o build/cista_optim.o

# host library between Python's lists of tensors and the C ABI (links the installed torch)
TLIB  = v2e2v_amd/libcista_torch.so
PY    ?= python3
TORCH := $(shell $(PY) -c "import importlib.util as u, os; print(os.path.dirname(u.find_spec('torch').origin))" 2>/dev/null)
PYINC = $(shell $(PY) -c "import sysconfig; print(sysconfig.get_paths()['include'])")

all: $(LIB) $(TLIB)

$(OBJ): Makefile

build/cista_abi.o: v2e2v_amd/csrc/cista_abi.hip v2e2v_amd/csrc/cista_kernels.hpp \
                   v2e2v_amd/csrc/cista_backward.hpp include/cista_lstc.h
	@mkdir -p build
	$(HIPCC) $(HIPFLAGS) -c -o $@ $<

build/cista_voxel.o: v2e2v_amd/csrc/cista_voxel.hip include/cista_voxel.h include/cista_lstc.h
	@mkdir -p build
	$(HIPCC) $(HIPFLAGS) -c -o $@ $<

build/cista_ssim.o: v2e2v_amd/csrc/cista_ssim.hip include/cista_loss.h include/cista_lstc.h
	@mkdir -p build
	$(HIPCC) $(HIPFLAGS) -c -o $@ $<

build/cista_v2e.o: v2e2v_amd/csrc/cista_v2e.hip include/cista_v2e.h include/cista_voxel.h include/cista_lstc.h
	@mkdir -p build
	$(HIPCC) $(HIPFLAGS) -c -o $@ $<

build/cista_optim.o: v2e2v_amd/csrc/cista_optim.hip include/cista_optim.h include/cista_lstc.h
	@mkdir -p build
	$(HIPCC) $(HIPFLAGS) -c -o $@ $<

$(LIB): $(OBJ)
	$(HIPCC) --offload-arch=$(ARCH) -shared -o $@ $(OBJ)

# version.py: another torch has another C++ ABI (_lib.torch_lib() refuses a library built for one)
$(TLIB): v2e2v_amd/csrc/cista_torch.cpp include/cista_optim.h include/cista_lstc.h $(TORCH)/version.py Makefile
	$(CXX) -O2 -std=c++17 -fPIC -Wall -shared -D__HIP_PLATFORM_AMD__ -DUSE_ROCM -I$(PYINC) -isystem $(TORCH)/include \
	    -isystem $(TORCH)/include/torch/csrc/api/include -isystem /opt/rocm/include -o $@ $< \
	    -L$(TORCH)/lib -ltorch_python -ltorch_cpu -lc10 -lc10_hip

clean:
	rm -rf build $(LIB) $(TLIB)

.PHONY: all clean
