"""Tensors of the C++ host mirror (vqa::moe::Session::new_tensor) of every type a tensor can have: ggml's strides.  On the
CPU: the mirror is compiled with an allocator and a context of its own.  And Q8_K in GGUF files: a type of rows, not of stored tensors."""
import pathlib
import subprocess

import mimoe as M
from test_gguf import write_gguf

ROOT = pathlib.Path(__file__).resolve().parents[1]
PKG = ROOT / "skyvision.cpp_amd"

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "mi_moe.h"
#include "mi_moe_util.h"
static int host_malloc(void **p, size_t n) { return (*p = std::malloc(n)) ? 0 : -1; }
static int host_free(void *p) { std::free(p); return 0; }
static int host_copy(void *d, const void *s, size_t n) { std::memcpy(d, s, n); return 0; }
template <typename T> static int stand_in(T **p) { static int v; *p = (T *)(void *)&v; return 0; }
#define mi_dev_malloc(p, n) host_malloc((void **)(p), n)
#define mi_dev_free(p) host_free(p)
#define mi_memcpy_h2d(d, s, n) host_copy(d, s, n)
#define mi_memcpy_d2d(d, s, n) host_copy(d, s, n)
#define mi_moe_ctx_create(p, d) stand_in(p)
#define mi_moe_ctx_destroy(c) (void)(c)
#define mi_moe_ctx_reserve(...) 0
#define mi_moe_expert_ffn(...) MI_MOE_ERR_TYPE
#define mi_stream_create(p) stand_in(p)
#define mi_stream_destroy(s) 0
#define mi_stream_synchronize(s) 0
#include "vqa_moe.cpp"
int main(int argc, char **argv) {
    using namespace vqa::moe;
    Session s(0);
    for (int i = 1; i + 1 < argc; i += 2) {
        const Tensor *t = s.new_tensor(std::atoi(argv[i]), std::atoll(argv[i + 1]), 5, 2);
        if (!t) std::printf("none\n");
        else std::printf("%zu %zu %zu %zu\n", (size_t)t->nb[0], (size_t)t->nb[1], (size_t)t->nb[2], (size_t)t->nb[3]);
    }
    Session b(0);
    std::vector<Tensor *> r8(1, b.new_tensor(MI_TYPE_Q8_K, 256, 256));
    Tensor *x = b.new_tensor(MI_TYPE_F32, 256, 1), *w = b.new_tensor(MI_TYPE_F32, 1, 1);
    const bool built = build_expert_ffn(b, x, r8, r8, r8, w) != nullptr;
    std::printf("slots %d status %d\n", (int)built, b.status());
}
"""


def run(tmp_path, calls):
    (tmp_path / "t.cpp").write_text(PROGRAM)
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-O0", f"-I{ROOT / 'include'}", f"-I{PKG / 'host'}", str(tmp_path / "t.cpp"),
                    f"-L{PKG}", "-lmimoe", f"-Wl,-rpath,{PKG}", "-o", str(exe)], check=True)
    args = [str(v) for c in calls for v in c]
    return [l.split() for l in subprocess.run([str(exe)] + args, capture_output=True, text=True, timeout=120, check=True).stdout.splitlines()]


def test_new_tensor_strides(tmp_path):
    """nb[0] the bytes of a block (one value of the plain types), rows and planes back to back; rows that are no whole
    blocks are refused"""
    kinds = [(M.TYPE_F32, 3, 4, 1), (M.TYPE_I32, 3, 4, 1), (M.TYPE_F16, 96, 2, 1)] + \
        [(t, 512, b, 256) for t, b in M.BLOCK_BYTES.items() if t in (M.TYPE_Q4_K, M.TYPE_Q6_K, M.TYPE_Q8_K)] + \
        [(t, 96, b, 32) for t, b in M.BLOCK_BYTES.items() if t not in (M.TYPE_Q4_K, M.TYPE_Q6_K, M.TYPE_Q8_K)]
    assert len(kinds) == 3 + len(M.BLOCK_BYTES)
    calls = [(t, n) for t, n, _, _ in kinds] + [(M.TYPE_Q8_K, 300), (M.TYPE_Q4_0, 40), (99, 256)]
    got = run(tmp_path, calls)[:-1]
    for (t, n, block, values), strides in zip(kinds, got):
        row = n // values * block
        assert [int(v) for v in strides] == [block, row, 5 * row, 10 * row], t
    assert got[len(kinds):] == [["none"]] * 3


def test_slots_of_rows_are_refused(tmp_path):
    """the per-slot builder returns nullptr for tensors of a type that no table has, and the session goes on"""
    assert run(tmp_path, [])[-1] == ["slots", "0", "status", "0"]


def test_gguf_q8_K_is_not_read(tmp_path):
    """a file that holds a Q8_K tensor is as one with any type the library does not read: its size is 0, it may be cut
    short, and the tensors beside it are there"""
    p = tmp_path / "rows.gguf"
    write_gguf(p, [], [("a", M.TYPE_F32, [4, 2], bytes(32)), ("rows", M.TYPE_Q8_K, [512, 3], bytes(3 * 584))])
    for cut in (0, 100):
        data = p.read_bytes()
        p.write_bytes(data[:len(data) - cut])
        g = M.Gguf(p)
        assert g.tensor_info("rows") == (M.TYPE_Q8_K, [512, 3, 1, 1], 0)
        assert g.tensor_info("a") == (M.TYPE_F32, [4, 2, 1, 1], 32)
        g.close()
