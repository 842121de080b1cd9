"""GPU: a wait that gives up says so, also where it finds that an earlier wait did, and a call over a used workspace starts clean."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import PKG, ROOT

pytestmark = pytest.mark.gpu

TIMEOUT = 16  # PA_STATUS_WAIT_TIMEOUT

SOURCE = """
#include "bounded_wait.cuh"
namespace pa {
struct Word {
  unsigned int* word;
  unsigned int by;
  int* status;
  __device__ bool marked() const { return *reinterpret_cast<volatile unsigned int*>(word) == by; }
  __device__ void mark() const { atomicExch(word, by); }
  __device__ void report() const { set_status(status, ST_WAIT_TIMEOUT); }
};
// Thread 0 waits twice on a barrier that nobody arrives at, then on one whose phase is over; what each wait returned.
__global__ void waits(unsigned int* word, unsigned int mark, int* status, int* got) {
  __shared__ __align__(8) unsigned long long bars[2];
  const uint32_t never = smem_u32(&bars[0]), over = smem_u32(&bars[1]);
  if (threadIdx.x != 0) return;
  mbar_init(never, 1);
  mbar_init(over, 1);
  fence_mbar_init();
  mbar_arrive(over);
  for (int i = 0; i < 2; ++i) got[i] = bounded_wait<512, 64>(never, 0, Word{word, mark, status});
  got[2] = bounded_wait<512, 64>(over, 0, Word{word, mark, status});
}
}  // namespace pa
extern "C" int run_waits(unsigned int* word, unsigned int mark, int* status, int* got, void* stream) {
  pa::waits<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(word, mark, status, got);
  return static_cast<int>(cudaGetLastError());
}
"""


@pytest.fixture(scope="module")
def run_waits(tmp_path_factory):
    """The wait as the kernels use it, in a kernel of its own."""
    import build

    d = tmp_path_factory.mktemp("waits")
    (d / "waits.cu").write_text(SOURCE)
    subprocess.run([build.nvcc_path(), *build.ARCH, "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
                    "-I", os.path.join(PKG, "csrc"), "-I", os.path.join(ROOT, "include"), str(d / "waits.cu"), "-o", str(d / "waits.so")],
                   check=True, capture_output=True)
    fn = ctypes.CDLL(str(d / "waits.so")).run_waits
    fn.argtypes = [ctypes.c_void_p, ctypes.c_uint, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]

    def call(word, status, mark=1):
        got = torch.full((3,), -1, dtype=torch.int32, device="cuda")
        assert fn(word.data_ptr(), mark, status.data_ptr(), got.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        return got.tolist()

    return call


def test_a_wait_that_gives_up(run_waits):
    word, status = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
    assert run_waits(word, status) == [0, 0, 1]  # a phase that is over is seen whatever the word says
    assert word.item() == 1 and status.item() == TIMEOUT


def test_a_wait_that_finds_the_mark_of_another(run_waits):
    """The caller has cleared the status, as after a failed replay: the next one sets it again."""
    word = torch.ones(1, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert run_waits(word, status) == [0, 0, 1]
    assert status.item() == TIMEOUT
    word.fill_(7)  # another call's mark is none
    status.zero_()
    assert run_waits(word, status, mark=8) == [0, 0, 1]
    assert word.item() == 8 and status.item() == TIMEOUT


@pytest.mark.parametrize("pool", [torch.float16, torch.int8])
def test_shared_prefixes_over_a_used_workspace(pool):
    """What a workspace held, another call's word of given-up waits too, does not reach a call, captured or not."""
    from pie_b200 import _lib, ops
    from test_gpu_shared_prefix import Problem

    p = Problem([(40, 1600), (6, 320)], [[9] * 40, [30] * 6], pool=pool, seed=3)
    want = ops.shared_prefix_attention(*p.args())
    Q, K, V, ql, bt, nb, BS, kl, gs, pl, ks, vs = p.args()
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kc, keep = ops.kv_cache_desc(K, V, ks, vs), []
    pg = ops.paging_desc(bt, nb, ql, kl, keep)
    io = _lib.PaAttnIO()
    io.q, io.q_dtype, io.num_q_heads, io.max_q_len = Q.data_ptr(), ops._TORCH2PA[Q.dtype], p.Hq, p.maxq
    io.q_stride_seq, io.q_stride_head, io.q_stride_row = Q.stride()[:3]
    io.o, io.lse = out.data_ptr(), lse.data_ptr()
    io.o_stride_seq, io.o_stride_head, io.o_stride_row = out.stride()[:3]
    io.l_stride_seq, io.l_stride_head, io.l_stride_row = lse.stride()
    gr = _lib.PaGroups(gs.data_ptr(), pl.data_ptr(), pl.numel(), 0)
    lib, size = _lib.load(), ctypes.c_size_t(0)
    assert lib.shared_prefix_workspace_size(io, kc, pg, gr, ctypes.byref(size)) == 0
    ws = torch.empty(size.value, dtype=torch.uint8, device="cuda")

    def call():
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.shared_prefix_attn(io, kc, pg, gr, ws.data_ptr(), size.value, status.data_ptr(), stream) == 0

    graph = torch.cuda.CUDAGraph()
    for what in (call, None, graph.replay, graph.replay):
        if what is None:
            with torch.cuda.graph(graph):
                call()
            continue
        for fill in (0x00, 0x01, 0xff):
            ws.fill_(fill)
            ws[:size.value // 4 * 4].view(torch.int32)[::4] = 1  # every fourth word as a mark
            ws[:size.value // 4 * 4].view(torch.int32)[3::4] = 1
            out.fill_(7)
            lse.fill_(7)
            what()
            torch.cuda.synchronize()
            assert status.item() == 0
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
