"""A small random-init Q4_K_M Llama file written with the `gguf` package, loaded through
rnb_b200_gguf_open / rnb_b200_decoder_load_gguf (mmap, page registration, upload from the mapped
pages) and decoded greedily against the oracle fed the same tensors."""
import numpy as np
import pytest

import oracle as orc
from synth import llama_description, max_err_vs_norm
from gguf_util import write_llama_gguf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("register_pages", [True, False])
def test_decoder_loaded_from_gguf_matches_oracle(tmp_path, register_pages):
    from runnburn_b200 import build, ops
    from runnburn_b200.gguf import load_decoder
    build.build_library()
    ops.open()
    desc = llama_description(seed=8, n_layer=2, hidden=512, n_head=4, n_kv_head=2, n_ff=1024, vocab=1024)
    path = tmp_path / "model.gguf"
    write_llama_gguf(path, desc, context_length=64)
    dec, f = load_decoder(str(path), register_pages=register_pages)
    assert dec.cfg.n_layer == 2 and dec.cfg.hidden == 512 and dec.cfg.vocab == 1024 and dec.cfg.max_ctx == 64
    ref = orc.Model(desc, 64)
    tok_g = tok_c = None
    prompt = np.random.default_rng(2).integers(0, 1024, 6).tolist()
    pos = 0
    for t in prompt + [None] * 24:
        if t is None:
            assert tok_g == tok_c, f"greedy ids diverge at position {pos}"
            t = tok_g
        tok_g, lg = dec.step(t, pos, want_logits=True)
        lc = ref.decode(t, pos)
        tok_c = orc.argmax_last(lc)
        assert max_err_vs_norm(lg, lc) <= 1e-3
        pos += 1
    dec.close()
    f.close()
    ops.clear_host_registered_ranges()
    ref.close()


def small_file(path, seed):
    desc = llama_description(seed=seed, n_layer=2, hidden=512, n_head=4, n_kv_head=2, n_ff=1024, vocab=1024)
    write_llama_gguf(path, desc, context_length=64)


def in_memory(path, offset):
    """The file's bytes `offset` behind the beginning of a page."""
    data = np.fromfile(path, np.uint8)
    room = np.zeros(data.size + 3 * 4096, np.uint8)
    start = -room.ctypes.data % 4096 + offset
    room[start:start + data.size] = data
    return room[start:start + data.size]


def is_pinned(address):
    import ctypes as C

    class Attributes(C.Structure):
        _fields_ = [("type", C.c_int), ("device", C.c_int), ("device_pointer", C.c_void_p), ("host_pointer", C.c_void_p)]
    a = Attributes()
    assert C.CDLL("libcudart.so.12").cudaPointerGetAttributes(C.byref(a), C.c_void_p(address)) == 0
    return a.type != 0


def logits(dec):
    return np.concatenate([dec.step(t, i, want_logits=True)[1] for i, t in enumerate((5, 900, 77, 3))])


@pytest.mark.parametrize("offset", [0, 32, 2080, 4064])
def test_weights_of_a_caller_s_memory_are_uploaded_from_pinned_pages(tmp_path, offset):
    """Tensors at the edges of what is pinned too: the first page and the last one are not the file's alone."""
    from runnburn_b200 import Decoder, build, ops
    from runnburn_b200.gguf import GgufFile, check, load
    build.build_library()
    ops.open()
    small_file(tmp_path / "m.gguf", 11)
    f = GgufFile(data=memoryview(in_memory(tmp_path / "m.gguf", offset)))
    got = []
    for pin in (0, 1):
        dec = Decoder(f.model_config())
        check(load().rnb_b200_decoder_load_gguf(dec._h, f._h, pin))
        got.append(logits(dec))
        dec.close()
    ops.clear_host_registered_ranges()
    assert np.array_equal(got[0], got[1]) and np.isfinite(got[0]).all()
    f.close()


@pytest.mark.parametrize("where", ["memory", "file", "file in memory"])
def test_nothing_stays_pinned_behind_a_load(tmp_path, where):
    """Pages that stay pinned when the file is closed would be taken for those of the next file at their address.  (Whether a mapped
    file can be pinned goes by the file system.)"""
    import os
    from runnburn_b200 import Decoder, RnbError, build, ops
    from runnburn_b200.gguf import GgufFile, check, load
    build.build_library()
    ops.open()
    path = f"/dev/shm/runnburn-{os.getpid()}.gguf" if where == "file in memory" else str(tmp_path / "m.gguf")
    try:
        small_file(path, 12)
        data = in_memory(path, 32)
        f = GgufFile(data=memoryview(data)) if where == "memory" else GgufFile(path)
    finally:
        if where == "file in memory":
            os.unlink(path)
    tensor = f.tensor("blk.0.attn_q.weight")["data"]
    cfg = f.model_config()
    dec = Decoder(cfg)
    check(load().rnb_b200_decoder_load_gguf(dec._h, f._h, 1))
    assert not is_pinned(tensor)
    want = logits(dec)
    # nor behind one that fails
    with pytest.raises(RnbError, match="already running"):
        check(load().rnb_b200_decoder_load_gguf(dec._h, f._h, 1))
    assert not is_pinned(tensor)
    dec.close()
    # but what the caller has pinned does
    if where == "memory":
        section = data[f.info()["data_start"]:]
        ops.register_host_range(section)
        dec = Decoder(cfg)
        check(load().rnb_b200_decoder_load_gguf(dec._h, f._h, 1))
        assert is_pinned(tensor) and np.array_equal(logits(dec), want)
        dec.close()
        ops.clear_host_registered_ranges()
        assert not is_pinned(tensor)
    f.close()


def test_files_one_after_another(tmp_path):
    """Each decoder has its own file's weights, wherever the files are mapped."""
    from runnburn_b200 import build, ops
    from runnburn_b200.gguf import load_decoder
    build.build_library()
    ops.open()
    got = []
    for pin in (False, True):
        for seed in (21, 22, 23):
            small_file(tmp_path / "m.gguf", seed)
            dec, f = load_decoder(str(tmp_path / "m.gguf"), register_pages=pin)
            (tmp_path / "m.gguf").unlink()
            f.close()
            got.append(logits(dec))
            dec.close()
    for a, b in zip(got[:3], got[3:]):
        assert np.array_equal(a, b)
    assert not np.array_equal(got[0], got[1])
