"""CPU: launches that the runtime would refuse are refused before any of a call's launches. It counts a
launch's threads in 32 bits: 2^24 workgroups of 256."""
import ctypes

from acestep_ops import _lib
from acestep_ops._lib import BF16, F32, I32, Q4_0, MiTensor

R = ctypes.byref
L = _lib.load()
SIZE = {F32: 4, I32: 4, BF16: 2, Q4_0: 18}


def _rows(shape, typ=F32, data=1 << 20):
    """Rows of ne[0] elements, all at one place (stride 0): a fake pointer, never dereferenced."""
    d = MiTensor()
    d.data, d.type, d.reserved = data, typ, 0
    for i in range(4):
        d.ne[i], d.nb[i] = (list(shape) + [1] * 4)[i], 0
    d.nb[0] = SIZE[typ]
    return d


def test_adapters():
    a, b, ws = _rows([32, 8, 1], BF16), _rows([8, 4, 1], BF16), ctypes.c_size_t(0)
    last = (1 << 28) - 16  # rows: 2^24 - 1 tiles of 16
    assert L.mi_lora_add_workspace(R(_rows([32, last])), R(a), R(b), R(ws)) == 0
    for m in (last + 1, last + 16, 1 << 28, 1 << 29, 1 << 30):
        x, y = _rows([32, m]), _rows([4, m], data=3 << 20)
        assert L.mi_lora_add_workspace(R(x), R(a), R(b), R(ws)) == -7, m
        assert L.mi_lora_add(R(y), R(x), R(a), R(b), R(_rows([m], I32)), None, R(y), 16 << 20, 1 << 50, None, None) == -7, m


def test_attention():
    """One query position of 2^24 sequences and heads; 4096 positions (256 workgroups) of 65536."""
    ws = ctypes.c_size_t(0)
    for heads, seqs, n_q, want in ((4096, 4095, 1, 0), (4096, 4096, 1, -7), (256, 255, 4096, 0), (256, 256, 4096, -7),
                                   (255, 257, 4096 - 15, 0), (256, 256, 4096 - 15, -7)):
        q, k = _rows([128, n_q, heads, seqs]), _rows([128, 64, heads, seqs], Q4_0)
        assert L.mi_flash_attn_ext_workspace(R(q), R(k), R(k), R(ws)) == want, (heads, seqs, n_q)
        if want:
            y = _rows([128, heads, n_q, seqs], data=3 << 20)
            assert L.mi_flash_attn_ext(R(q), R(k), R(k), None, 0.1, 0.0, 0.0, R(y), None, 0, None) == want


def test_attention_merge():
    """More keys than one workgroup of the kernel for many rows lists are always split; the merge's workgroups count too."""
    ws = ctypes.c_size_t(0)
    for n_q, want in ((1 << 14, 0), ((1 << 15) - 1, 0), (1 << 15, -7)):
        q, k = _rows([256, n_q, 512, 1]), _rows([256, 1 << 21, 512, 1], Q4_0)
        assert L.mi_flash_attn_ext_workspace(R(q), R(k), R(k), R(ws)) == want, n_q
