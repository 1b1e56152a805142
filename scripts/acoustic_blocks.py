#!/usr/bin/env python3
"""What MXFP4 changes in the acoustic model: time of its convolution blocks and mel head, of a whole call, and how far
the mel moves.  Random weights, one sentence of 165 phonemes and 64 x 865 frames.  Prints one JSON line.
scripts/acoustic_blocks.py > profiles/acoustic_blocks.json"""
import json
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from tts_amd.acoustic import FastSpeechAcousticModel  # noqa: E402


def microseconds(call, n=30, rounds=5):
    for _ in range(5):
        call()
    times = []
    for _ in range(rounds):
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(n):
            call()
        torch.cuda.synchronize()
        times.append((time.perf_counter() - start) / n * 1e6)
    return round(sorted(times)[rounds // 2], 1)


def main():
    torch.manual_seed(0)
    model = FastSpeechAcousticModel(72).cuda()
    ids = np.random.default_rng(0).integers(1, 72, (1, 165))
    inputs = ids, np.log(np.full(ids.shape, 5.0)).astype(np.float32)

    def blocks(x):
        x = model.encoder.block2(model.encoder.block1(x))
        return model.duration_predictor(x), model.mel_out(x.transpose(1, 2))

    sentence, batch = torch.randn(1, 165, 256, device="cuda"), torch.randn(64, 865, 256, device="cuda")
    out, mels = {"device": torch.cuda.get_device_name(), "unit": "us, median of 5 x 30 calls"}, {}
    with torch.no_grad():
        for form in ("float32", "mxfp4"):
            model.use_mxfp4(form == "mxfp4")
            out[form] = {"whole_call_165_phonemes": microseconds(lambda: model(inputs)),
                         "blocks_and_mel_head_1x165": microseconds(lambda: blocks(sentence)),
                         "blocks_and_mel_head_64x865": microseconds(lambda: blocks(batch))}
            mels[form] = model(inputs)
    out["mel_relative_l2"] = round(((mels["mxfp4"] - mels["float32"]).norm() / mels["float32"].norm()).item(), 4)
    print(json.dumps(out))


if __name__ == "__main__":
    main()
