"""Views fed one after another to a VGGT-shaped aggregator (random init) with
8-bit caches in its global blocks and, with --int8, 8-bit Linears.

    python examples/stream_views.py --frames 16 --int8
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ress_b200 import kernels as K  # noqa: E402
from ress_b200 import stream, vggt  # noqa: E402


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--frames", type=int, default=16)
    ap.add_argument("--streams", type=int, default=1)
    ap.add_argument("--size", type=int, default=518, help="image side, a multiple of 14")
    ap.add_argument("--depth", type=int, default=24)
    ap.add_argument("--int8", action="store_true", help="8-bit Linears in the aggregator's blocks")
    a = ap.parse_args()
    torch.manual_seed(0)
    model = vggt.VGGTAggregatorModel(depth=a.depth, encoder_depth=a.depth, img=a.size,
                                     intermediate=(a.depth - 1,)).cuda().bfloat16().eval()
    agg = model.aggregator
    if a.int8:
        n = stream.quantize_linears(agg.frame_blocks) + stream.quantize_linears(agg.global_blocks)
        print(f"{n} Linears in 8 bits")
    tokens = (a.size // 14) ** 2 + agg.patch_start_idx
    stream.apply_stream(model, streams=a.streams, max_frames=a.frames, frame_tokens=tokens)
    print(f"caches: {sum(c.nbytes for c in stream.stream_caches(model)) / 2 ** 20:.0f} MiB for {a.frames} frames")
    frames = torch.rand(a.streams, a.frames, 3, a.size, a.size, device="cuda")
    with torch.inference_mode():
        for scene in range(2):  # the first scene warms up
            stream.reset_stream(model)
            for i in range(a.frames):
                start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
                start.record()
                out, _ = model(frames[:, i:i + 1], first_frame=i == 0)
                end.record()
                end.synchronize()
                if scene == 1:
                    print(f"frame {i:3d}: {start.elapsed_time(end):7.2f} ms, {(i + 1) * tokens} tokens held")
    K.check_status()
    assert all(torch.isfinite(o).all() for o in out if o is not None)


if __name__ == "__main__":
    main()
