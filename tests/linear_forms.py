"""Sizes (M rows, K inputs, N outputs) for every form that linear_act's products take: tests/test_gpu_block_forms.py runs them on the device,
tests/test_block_calls_host.py holds them against the choice, so that a change of the choice cannot leave a form without a test."""

# product -> {(tile form, contraction split): size}
ALONE = {
    "y": {(0, False): (16383, 72, 776), (0, True): (1001, 6000, 4104), (1, False): (4351, 72, 2304), (1, True): (519, 4096, 2304),
          (2, False): (8199, 200, 776), (2, True): (5999, 8200, 72), (3, False): (5999, 520, 520), (3, True): (67, 6000, 4104),
          (4, False): (67, 72, 72), (4, True): (67, 2056, 72)},
    "dx": {(0, False): (6001, 2056, 72), (0, True): (2175, 2056, 8200), (1, False): (2999, 4096, 72), (1, True): (5999, 200, 4104),
           (2, False): (2999, 2056, 200), (2, True): (67, 6000, 8200), (3, False): (519, 6000, 520), (3, True): (2999, 72, 8200),
           (4, False): (67, 72, 72), (4, True): (67, 72, 2304)},
    "dw": {(0, False): (67, 6000, 2304), (0, True): (16383, 200, 4104), (2, False): (201, 768, 8200), (2, True): (8199, 6000, 72),
           (3, False): (519, 6000, 520), (3, True): (2999, 72, 8200), (4, False): (67, 72, 72), (4, True): (2175, 72, 72)},
}
# both products of a backward pass in one launch: {(tile form, dx split, dw split): size}
PAIRED = {(2, False, False): (201, 8200, 200), (2, False, True): (8199, 520, 72), (2, True, False): (201, 2056, 2304),
          (2, True, True): (8199, 72, 8200), (3, False, False): (67, 8200, 72), (3, False, True): (5999, 200, 200),
          (3, True, False): (999, 200, 4104), (3, True, True): (4351, 72, 4104), (4, False, False): (67, 72, 72),
          (4, False, True): (2175, 72, 72), (4, True, False): (67, 72, 2304)}
# both wanted, in launches of their own: {(dx split, dw split): size}
SEPARATE = {(False, False): (4352, 4096, 4096), (True, False): (301, 4096, 8200), (False, True): (4351, 4096, 72), (True, True): (4663, 75, 14016)}
# up to 64 rows in the form of their own: {blocks of 16 rows: size}
FEW = {1: (13, 1030, 520), 2: (29, 770, 776), 3: (34, 768, 768), 4: (64, 130, 50)}


def form(L, product, size):
    """(tile form or -1 for few rows, splits) of one product, as the library chooses it."""
    import ctypes
    M, K, N = size
    f, s = ctypes.c_int(), ctypes.c_int()
    sides = {"y": (M, N, K, 0), "dx": (M, K, N, 1), "dw": (N, K, M, 2)}[product]
    assert L.hopmi_gemm16_form(*sides, ctypes.byref(f), ctypes.byref(s)) == 0
    return f.value, s.value


def backward_form(L, size):
    """(one launch, dx's tile form, its splits, dw's, its splits) of a backward pass that wants both."""
    import ctypes
    M, K, N = size
    v = [ctypes.c_int() for _ in range(5)]
    assert L.hopmi_linear16_bwd_form(M, N, K, *map(ctypes.byref, v)) == 0
    return tuple(i.value for i in v)
