"""CPU checks of the chunk operators (store_rope, mla_chunk_attention_paged,
verify_drafts): the C ABI's argument errors and the Python refusals.  No
kernel is launched."""
import ctypes

import pytest
import torch

FAKE, MIS = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10008)   # never dereferenced


def chunk(L, q=FAKE, sq=(9216, 576), kv=FAKE, int8=0, page=73728, row=1152, pages=4, block=64, cu=FAKE, lens=FAKE, bt=FAKE,
          reqs=2, bts=4, cols=4, T=2, H=16, ws=FAKE, wsb=1 << 40, out=FAKE, so=(8192, 512)):
    return L.glm53_chunk_mla(q, *sq, kv, int8, page, row, pages, block, cu, lens, bt, reqs, bts, cols, T, H, 0.04, ws, wsb,
                             out, *so, None, None)


def test_chunk_mla_argument_errors():
    import _glm53_lib
    L = _glm53_lib.load()
    assert chunk(L, T=0) == 0 and chunk(L, reqs=0) == 0
    for bad in ({"T": -1}, {"reqs": -1}, {"H": 0}, {"block": 0}, {"cols": -1}, {"pages": -1}, {"row": 1136},
                {"int8": 1, "row": 512}, {"page": -16}, {"T": 1 << 28}, {"reqs": 1 << 31}, {"reqs": 1 << 27},
                {"block": 1 << 31}, {"cols": 1 << 31}, {"pages": 1 << 31}):
        assert chunk(L, **bad) == -2, bad
    for bad in ({"q": None}, {"kv": None}, {"cu": None}, {"lens": None}, {"bt": None}, {"out": None}):
        assert chunk(L, **bad) == -1, bad
    for bad in ({"q": MIS}, {"sq": (9217, 576)}, {"sq": (9216, 577)}, {"kv": MIS}, {"page": 73736}, {"row": 1160},
                {"out": ctypes.c_void_p(0x10004)}, {"so": (8194, 512)}, {"so": (8192, 513)}, {"ws": MIS}):
        assert chunk(L, **bad) == -3, bad
    need = L.glm53_chunk_mla_workspace_bytes(2, 2, 16)
    assert need > 0
    assert chunk(L, ws=None) == -4 and chunk(L, wsb=need - 1) == -4
    assert L.glm53_chunk_mla_workspace_bytes(0, 2, 16) == 0 and L.glm53_chunk_mla_workspace_bytes(2, 0, 16) == 0
    assert L.glm53_chunk_mla_workspace_bytes(1 << 20, 2, 16) == 0    # a workgroup per tile: no partials


def rope(L, x=FAKE, sx=512, k=FAKE, sk=64, pos=FAKE, table=FAKE, max_pos=100, norm=None, cache=FAKE, page=73728, row=1152,
         block=64, cap=256, slots=FAKE, n=4, q=FAKE, sq=(1024, 64), o=FAKE, so=(1024, 64), H=16):
    return L.glm53_store_rope(x, sx, k, sk, pos, 1, table, 1, max_pos, 0, norm, 1e-6, cache, page, row, block, cap, slots, 1,
                              n, q, *sq, o, *so, H, None)


def test_store_rope_argument_errors():
    import _glm53_lib
    L = _glm53_lib.load()
    assert rope(L, n=0) == 0
    for bad in ({"n": -1}, {"block": 0}, {"max_pos": -1}, {"H": -1}, {"cap": -1}, {"H": 65537}, {"n": 1 << 41},
                {"n": 1 << 35}):
        assert rope(L, **bad) == -2, bad
    for bad in ({"x": None}, {"k": None}, {"pos": None}, {"table": None}, {"cache": None}, {"slots": None}, {"q": None},
                {"o": None}):
        assert rope(L, **bad) == -1, bad
    for bad in ({"x": MIS}, {"sx": 513}, {"k": MIS}, {"sk": 65}, {"table": MIS}, {"norm": MIS}, {"cache": MIS}, {"page": 8},
                {"row": 1160}, {"q": MIS}, {"sq": (1025, 64)}, {"sq": (1024, 65)}, {"o": MIS}, {"so": (1028, 64)},
                {"so": (1024, 68)}):
        assert rope(L, **bad) == -3, bad


def drafts(L, p=FAKE, st=100, rows=6, q=FAKE, ids=FAKE, D=4, cu=FAKE, u=FAKE, s=FAKE, R=2, vocab=100, most=2, ws=FAKE,
           wsb=1 << 30, tokens=FAKE, accepted=FAKE):
    return L.glm53_verify_drafts(p, st, rows, q, 100, ids, 0, D, cu, u, s, R, vocab, most, ws, wsb, tokens, accepted, None)


def test_verify_drafts_argument_errors():
    import _glm53_lib
    L = _glm53_lib.load()
    assert drafts(L, R=0) == 0
    for bad in ({"rows": -1}, {"D": -1}, {"R": -1}, {"vocab": 0}, {"most": -1}, {"R": 65536}, {"vocab": 0x7fffffff}):
        assert drafts(L, **bad) == -2, bad
    for bad in ({"p": None}, {"ids": None}, {"cu": None}, {"u": None}, {"s": None}, {"tokens": None}, {"accepted": None}):
        assert drafts(L, **bad) == -1, bad
    need = L.glm53_verify_drafts_workspace_bytes(2, 100)
    assert drafts(L, ws=None) == -4 and drafts(L, wsb=need - 1) == -4
    assert drafts(L, ws=ctypes.c_void_p(0x10004)) == -3


B, F, I32 = torch.bfloat16, torch.float32, torch.int32


def test_chunk_attention_refusals():
    from titan_mla import mla_chunk_attention_paged as attend

    def call(q=torch.zeros(2, 16, 576, dtype=B), c=torch.zeros(3, 64, 576, dtype=B), cu=torch.zeros(2, dtype=I32),
             lens=torch.zeros(1, dtype=I32), t=torch.zeros(1, 2, dtype=I32), **kw):
        return attend(q, c, cu, lens, t, 0.04, **kw)

    for bad in ({"q": torch.zeros(2, 576, dtype=B)}, {"q": torch.zeros(2, 16, 512, dtype=B)},
                {"q": torch.zeros(2, 16, 576, dtype=torch.float16)}, {"c": torch.zeros(3, 64, 576)},
                {"c": torch.zeros(3, 64, 512, dtype=B)}, {"c": torch.zeros(3, 64, 528, dtype=torch.int8)},
                {"c": torch.zeros(3, 0, 576, dtype=B)}, {"cu": torch.zeros(2, dtype=torch.int64)},
                {"lens": torch.zeros(1, dtype=torch.int64)}, {"t": torch.zeros(1, 2, dtype=torch.int64)},
                {"cu": torch.zeros(3, dtype=I32)}, {"t": torch.zeros(2, 2, dtype=I32)}, {"t": torch.zeros(2, dtype=I32)},
                {"q": torch.zeros(2, 0, 576, dtype=B)}, {}):                         # the last: CPU tensors
        with pytest.raises(ValueError):
            call(**bad)


def test_store_rope_refusals():
    from titan_kv import store_rope

    def call(x=torch.zeros(4, 512, dtype=B), k=torch.zeros(4, 64, dtype=B), pos=torch.zeros(4, dtype=I32),
             t=torch.zeros(9, 64), c=torch.zeros(2, 16, 576, dtype=B), s=torch.zeros(4, dtype=I32), **kw):
        return store_rope(x, k, pos, t, c, s, **kw)

    q = torch.zeros(4, 2, 64, dtype=B)
    for bad in ({"x": torch.zeros(4, 256, dtype=B)}, {"x": torch.zeros(4, 512)}, {"k": torch.zeros(4, 32, dtype=B)},
                {"k": torch.zeros(3, 64, dtype=B)}, {"pos": torch.zeros(4)}, {"pos": torch.zeros(5, dtype=I32)},
                {"t": torch.zeros(9, 32)}, {"t": torch.zeros(9, 64, dtype=torch.float16)},
                {"c": torch.zeros(2, 16, 512, dtype=B)}, {"c": torch.zeros(2, 16, 576)},
                {"c": torch.zeros(2, 16, 577, dtype=B)[:, :, 1:]}, {"s": torch.zeros(5, dtype=I32)}, {"s": torch.zeros(4)},
                {"norm_weight": torch.zeros(512)}, {"norm_weight": torch.zeros(64, dtype=B)}, {"q_out": q},
                {"q_pe": torch.zeros(4, 2, 32, dtype=B)}, {"q_pe": q, "q_out": torch.zeros(4, 3, 64, dtype=B)},
                {"q_pe": q, "q_out": torch.zeros(4, 2, 65, dtype=B)[:, :, 1:]}, {}):
        with pytest.raises(ValueError):
            call(**bad)


def test_verify_drafts_refusals():
    from titan_spec import verify_drafts

    def call(p=torch.zeros(5, 10), ids=torch.zeros(3, dtype=I32), q=torch.zeros(3, 10), cu=torch.zeros(3, dtype=I32),
             u=torch.zeros(3), s=torch.zeros(2, dtype=torch.float64), most=2):
        return verify_drafts(p, ids, q, cu, u, s, most)

    for bad in ({"p": torch.zeros(5, 10, dtype=B)}, {"p": torch.zeros(5, 0)}, {"p": torch.zeros(10)},
                {"ids": torch.zeros(3)}, {"ids": torch.zeros(3, 1, dtype=I32)}, {"q": torch.zeros(4, 10)},
                {"q": torch.zeros(3, 10, dtype=B)}, {"cu": torch.zeros(3, dtype=torch.int64)},
                {"cu": torch.zeros(0, dtype=I32)}, {"u": torch.zeros(2)}, {"u": torch.zeros(3, dtype=torch.float64)},
                {"s": torch.zeros(2)}, {"s": torch.zeros(3, dtype=torch.float64)}, {"most": -1}, {}):
        with pytest.raises(ValueError):
            call(**bad)


def test_importing_touches_no_device():
    import subprocess
    import sys
    from pathlib import Path
    pkg = Path(__file__).resolve().parents[1] / "glm-5.3-kernels_amd"
    code = "import titan_spec, titan_kv, titan_mla, torch; assert not torch.cuda.is_initialized()"
    subprocess.run([sys.executable, "-c", code], check=True, cwd=pkg)
