"""The C entry points of the prompt attention and the paged cache refuse every pointer that is not memory of the device, one by one,
before anything is launched."""

import numpy as np
import pytest
import torch

from reskv_b200._extension import ERR_INVALID, library

DEV = "cuda"


def refusals(call, arguments, pointers):
    """``call`` with the arguments succeeds; with a host address in the place of each pointer it is refused by that pointer's name."""
    host = np.zeros(1 << 16, np.uint8)
    address = host.ctypes.data + (-host.ctypes.data) % 64
    assert call(*arguments) == 0
    for place, name in pointers.items():
        changed = list(arguments)
        assert changed[place] is not None
        changed[place] = address
        assert call(*changed) == ERR_INVALID, name
        assert f": {name} ".encode() in library().reskv_last_error(), library().reskv_last_error()
    torch.cuda.synchronize()
    assert not host.any()


@pytest.mark.gpu
def test_prompt_attention():
    x = torch.zeros(4, 2, 128, dtype=torch.float16, device=DEV)
    out, lse, cu = torch.empty_like(x), torch.empty(4, 2, device=DEV), torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    p = [t.data_ptr() for t in (x, x, x, cu)]
    stream = torch.cuda.current_stream().cuda_stream
    arguments = [*p, 1, 4, 2, 2, 0, *[256, 128] * 3, 0.1, 1, out.data_ptr(), lse.data_ptr(), word.data_ptr(), stream]
    refusals(library().reskv_prompt_attention_reporting, arguments,
             {0: "q", 1: "k", 2: "v", 3: "cu_seqlens", 17: "out", 18: "lse", 19: "status"})


@pytest.mark.gpu
def test_paged_cache():
    lib, stream = library(), torch.cuda.current_stream().cuda_stream
    x = torch.zeros(1, 1, 128, dtype=torch.float16, device=DEV)
    out, lse = torch.empty_like(x), torch.empty(1, 1, device=DEV)
    pages = torch.zeros(2, 1, 9216, dtype=torch.uint8, device=DEV)
    cu, zero, one, word = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([0, 1], [0], [1], [0]))
    a, b, c = cu.data_ptr(), zero.data_ptr(), word.data_ptr()
    refusals(lib.reskv_paged_write, [x.data_ptr(), x.data_ptr(), 0, 128, 128, 128, 128, a, b, b, 1, 1, 1, 1, pages.data_ptr(), 2, c, stream],
             {0: "k", 1: "v", 7: "cu_seqlens", 8: "starts", 9: "table", 14: "pages", 16: "status"})
    refusals(lib.reskv_paged_read, [out.data_ptr(), out.data_ptr(), 0, a, b, b, 1, 1, 1, 1, pages.data_ptr(), 2, c, stream],
             {0: "k", 1: "v", 3: "cu_seqlens", 4: "starts", 5: "table", 10: "pages", 12: "status"})
    need = lib.reskv_paged_attention_workspace_bytes(1, 1, 1)
    workspace = torch.empty(need, dtype=torch.uint8, device=DEV)
    refusals(lib.reskv_paged_attention, [x.data_ptr(), 0, 128, 128, one.data_ptr(), b, 1, 1, 1, 1, pages.data_ptr(), 2, 0.1, workspace.data_ptr(), need,
                                         out.data_ptr(), lse.data_ptr(), c, stream],
             {0: "q", 4: "lengths", 5: "table", 10: "pages", 13: "workspace", 15: "out", 16: "lse", 17: "status"})
    src, dst = np.array([0], np.int32), np.array([1], np.int32)  # host arrays
    refusals(lib.reskv_copy_pages, [pages.data_ptr(), 1, 2, 9216, src.ctypes.data, dst.ctypes.data, 1, stream], {0: "pages"})
    assert word.item() == 0
