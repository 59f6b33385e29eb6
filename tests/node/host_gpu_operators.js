// GPU run of BlockNormKernel, Q4GemmKernel and TokenScoreKernel together: the
// norm of a block's output with gate and residual, the 4-bit head product of
// the next norm, and the scores of given tokens, in one command buffer.
// Usage: node host_gpu_operators.js <case.json>; run by
// tests/test_node_operators.py, which checks what it writes.
"use strict";
const assert = require("assert");
const fs = require("fs");
const path = require("path");
const host = require(path.join(__dirname, "..", "..", "parakeet.wgsl_amd", "host"));

function bytesOf(file) {
  const b = fs.readFileSync(file);
  return new Uint8Array(b.buffer, b.byteOffset, b.byteLength);
}

async function main() {
  const spec = JSON.parse(fs.readFileSync(process.argv[2], "utf8"));
  const { rows, channels, columns, classes, groupSize, alternatives, active } = spec;
  const device = host.HipGpuDevice.create();
  const arena = new host.GpuActivationArena(device, 32 * 1024 * 1024);
  let at = 0;
  function slice(name, bytes, file) {
    const s = arena.slice(name, at, bytes);
    at += Math.ceil(bytes / 256) * 256;
    if (file) arena.upload(device, s, bytesOf(file));
    return s;
  }
  const matrix = rows * channels * 2;
  const input = slice("input", matrix, spec.input), residual = slice("residual", matrix, spec.residual);
  const gate = slice("gate", channels * 2, spec.gate), tokens = slice("tokens", rows * 4, spec.tokens);
  const output = slice("output", matrix), normed = slice("normed", matrix), logits = slice("logits", rows * columns * 2);
  const logProbs = slice("logProbs", rows * 4), entropies = slice("entropies", rows * 4);
  const topTokens = slice("topTokens", rows * alternatives * 4), topLogProbs = slice("topLogProbs", rows * alternatives * 4);
  const vector = (file) => host.createGpuTensor(device, host.channelTensorRecords(channels), bytesOf(file));
  const norm = await host.BlockNormKernel.create(device, arena);
  const gemm = await host.Q4GemmKernel.create(device, arena);
  const score = await host.TokenScoreKernel.create(device, arena);
  const records = host.q4TensorRecords({ inner: channels, columns, groupSize });
  const dispatches = [
    norm.createDispatch({
      label: "block", rows, channels, kind: "rms", input, gamma: vector(spec.gamma), gate, gateRows: 0, residual,
      residualScale: 0.5, output, next: { gamma: vector(spec.nextGamma), output: normed },
    }),
    gemm.createDispatch({
      label: "head", rows, inner: channels, columns, groupSize, a: normed,
      packed: host.createGpuTensor(device, records.packed, bytesOf(spec.packed)),
      scales: host.createGpuTensor(device, records.scales, bytesOf(spec.scales)),
      bias: host.createGpuTensor(device, host.channelTensorRecords(columns), bytesOf(spec.bias)), output: logits,
    }),
    score.createDispatch({
      label: "confidence", rows, columns: classes, rowStride: columns, logits, tokens, logProbs, entropies, alternatives,
      topTokens, topLogProbs,
    }),
  ];
  const timestamps = device.createQuerySet({ type: "timestamp", count: 6 });
  const encoder = device.createCommandEncoder({ label: "operators" });
  dispatches.forEach((d, i) => d.encode(encoder, {
    querySet: timestamps, beginningOfPassWriteIndex: 2 * i, endOfPassWriteIndex: 2 * i + 1 }, { rows: active }));
  device.queue.submit([encoder.finish()]);
  await device.queue.onSubmittedWorkDone();
  for (let i = 0; i < 3; ++i) assert.ok(timestamps.elapsedMs(2 * i, 2 * i + 1) > 0);
  for (const [name, s] of [["output", output], ["normed", normed], ["logits", logits], ["logProbs", logProbs],
                           ["entropies", entropies], ["topTokens", topTokens], ["topLogProbs", topLogProbs]])
    fs.writeFileSync(path.join(spec.directory, `${name}.out`),
                     Buffer.from(await device.queue.readBuffer(arena.buffer, s.byteOffset, s.byteLength)));
  assert.throws(() => dispatches[0].encode(encoder, undefined, { rows: rows + 1 }), RangeError);
  for (const d of dispatches) {
    d.destroy();
    assert.throws(() => d.encode(encoder), /was destroyed/);
  }
  console.log("host_gpu_operators ok");
}
main().catch((e) => { console.error(e); process.exit(1); });
