# Top-level build of libbooster_b200.so (the product) — sm_100a only, in-tree.
NVCC      ?= $(shell command -v nvcc 2>/dev/null || echo /usr/local/cuda/bin/nvcc)
ARCH      := -gencode arch=compute_100a,code=sm_100a
NVCCFLAGS := $(ARCH) -O3 -std=c++17 -lineinfo -Xcompiler -fPIC,-Wall,-Wno-unused-function -Xptxas -v
CSRC      := booster_b200/csrc
OBJDIR    := build
LIB       := booster_b200/libbooster_b200.so
SERVE     := booster_b200/_serve.so
PYTHON    ?= $(shell command -v python3 2>/dev/null || command -v python 2>/dev/null)
# the torch that $(PYTHON) would load, with its headers (nothing: none is there, and the library is built without the module of torch tensors)
TORCH     := $(shell $(PYTHON) -c 'import importlib.metadata as m, importlib.util as u, os, sys; r = os.path.dirname(u.find_spec("torch").origin); os.stat(r + "/include/torch/csrc"); print(m.version("torch") + "-" + sys.implementation.cache_tag)' 2>/dev/null)

OBJS := $(OBJDIR)/engine.o $(OBJDIR)/stack.o $(OBJDIR)/serve.o $(OBJDIR)/serve16.o $(OBJDIR)/safetensors.o $(OBJDIR)/gguf.o $(OBJDIR)/bridge.o $(OBJDIR)/tokenizer.o $(OBJDIR)/janus.o

all: $(LIB) $(if $(TORCH),$(SERVE),no-torch)

$(OBJDIR)/engine.o: $(CSRC)/engine.cu $(CSRC)/kernels.cuh $(CSRC)/token_kernel.cuh $(CSRC)/attn_cluster.cuh $(CSRC)/matvec_q80.cuh $(CSRC)/matvec_kq.cuh $(CSRC)/prefill.cuh $(CSRC)/prefill_mma.cuh $(CSRC)/prefill_umma.cuh $(CSRC)/prefill_umma_q80.cuh $(CSRC)/gguf.hpp $(CSRC)/tokenizer.hpp $(CSRC)/stack.hpp $(CSRC)/serve.hpp $(CSRC)/safetensors.hpp include/booster_b200.h
	@mkdir -p $(OBJDIR)
	$(NVCC) $(NVCCFLAGS) -c $< -o $@ 2> $(OBJDIR)/engine.ptxas.log || (cat $(OBJDIR)/engine.ptxas.log; false)

$(OBJDIR)/stack.o: $(CSRC)/stack.cu $(CSRC)/stack_kernels.cuh $(CSRC)/stack_kernels_f32.cuh $(CSRC)/stack_kernels_pair.cuh $(CSRC)/stack_kernels_mix.cuh $(CSRC)/stack_kernels_hyper.cuh $(CSRC)/stack_kernels_scan.cuh $(CSRC)/stack_kernels_side.cuh $(CSRC)/stack.hpp $(CSRC)/safetensors.hpp
	@mkdir -p $(OBJDIR)
	$(NVCC) $(NVCCFLAGS) -c $< -o $@ 2> $(OBJDIR)/stack.ptxas.log || (cat $(OBJDIR)/stack.ptxas.log; false)

$(OBJDIR)/serve.o: $(CSRC)/serve.cu $(CSRC)/serve.hpp $(CSRC)/serve_host.cuh $(CSRC)/serve_cache.cuh $(CSRC)/serve_attn.cuh $(CSRC)/serve_prompt.cuh $(CSRC)/serve_pages.cuh $(CSRC)/serve_sample.cuh include/booster_b200.h
	@mkdir -p $(OBJDIR)
	$(NVCC) $(NVCCFLAGS) -c $< -o $@ 2> $(OBJDIR)/serve.ptxas.log || (cat $(OBJDIR)/serve.ptxas.log; false)

$(OBJDIR)/serve16.o: $(CSRC)/serve16.cu $(CSRC)/serve.hpp $(CSRC)/serve_host.cuh $(CSRC)/serve_cache.cuh $(CSRC)/serve_attn.cuh $(CSRC)/serve_prompt.cuh $(CSRC)/serve_tma.cuh $(CSRC)/serve_kv16.cuh $(CSRC)/serve_kv16_prompt.cuh include/booster_b200.h
	@mkdir -p $(OBJDIR)
	$(NVCC) $(NVCCFLAGS) -c $< -o $@ 2> $(OBJDIR)/serve16.ptxas.log || (cat $(OBJDIR)/serve16.ptxas.log; false)

$(OBJDIR)/%.o: $(CSRC)/%.cpp $(CSRC)/gguf.hpp $(CSRC)/tokenizer.hpp $(CSRC)/janus.hpp $(CSRC)/unicode_tables.hpp $(CSRC)/safetensors.hpp include/bridge.h include/booster_b200.h
	@mkdir -p $(OBJDIR)
	$(NVCC) $(ARCH) -O3 -std=c++17 -Xcompiler -fPIC,-Wall,-O3 -c $< -o $@

$(LIB): $(OBJS)
	$(NVCC) $(ARCH) -shared -o $@ $^ -ldl

# booster_b200/serve.py's module of torch tensors: the flags are those of the torch that will load it, and another torch makes it anew
$(OBJDIR)/torch-$(TORCH).stamp:
	@mkdir -p $(OBJDIR)
	@rm -f $(OBJDIR)/torch-*.stamp
	@touch $@

$(SERVE): $(CSRC)/serve_torch.cpp include/booster_b200.h $(OBJDIR)/torch-$(TORCH).stamp
	flags=$$($(PYTHON) -c 'import os, sysconfig, torch; r = os.path.dirname(torch.__file__); inc = sysconfig.get_path("include"); print(f"-I{r}/include -I{r}/include/torch/csrc/api/include -isystem /usr/local/cuda/include -I{inc} -D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)} -L{r}/lib")') && \
	$(CXX) -O2 -std=c++17 -fPIC -shared -Wall -Wno-unused-function $< -o $@ $$flags -lc10 -lc10_cuda -ltorch_cpu -ltorch_python

no-torch:
	@echo "no torch with headers for '$(PYTHON)': booster_b200/serve.py's module is not built (make PYTHON=... names another)"

oracle:
	$(MAKE) -C oracle all

clean:
	rm -rf $(OBJDIR) $(LIB) $(SERVE)

.PHONY: all no-torch oracle clean
