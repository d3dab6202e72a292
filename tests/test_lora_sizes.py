"""CPU check of the sizes that ti_lora_add takes: its kernels step through K and N in 32 bits, so both end where every step still fits."""
import ctypes as C

import pytest

from tabinfer_amd import abi

P, FAR = 0x10000, 1 << 46                            # addresses that a refused call does not touch
END = 2 ** 30


@pytest.mark.parametrize("T,K,N,r", [(1, 64, END + 1, 1), (1, 64, 2 ** 31 - 16383, 8), (1, 64, 2 ** 31 - 256, 1), (9000, 64, 2 ** 31 - 256, 1),
                                     (1, END + 32, 40, 1), (1, 2 ** 31 - 2048, 40, 128), (1, 2 ** 31 - 256, 40, 16), (600, 2 ** 31 - 256, 40, 16)])
@pytest.mark.parametrize("bf16", [0, 1])
def test_sizes_that_steps_would_pass_are_refused(T, K, N, r, bf16):
    ctx = C.addressof(C.create_string_buffer(1 << 16))
    rc = abi.lib().ti_lora_add(ctx, P, P, P, P, P, FAR, T, K, N, r, 2, 0, 0, bf16)
    assert rc == abi.TI_ERR_INVALID and b"ti_lora_add: K = %d, N = %d" % (K, N) in abi.lib().ti_last_error()
