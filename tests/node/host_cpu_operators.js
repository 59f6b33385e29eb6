// Contracts of BlockNormKernel, Q4GemmKernel and TokenScoreKernel without a
// GPU: descriptor checks and their messages. Run by tests/test_node_operators.py.
"use strict";
const assert = require("assert");
const path = require("path");
const host = require(path.join(__dirname, "..", "..", "parakeet.wgsl_amd", "host"));

const MB = 1024 * 1024;
const arena = new host.GpuActivationArena({ createBuffer: ({ size }) => ({ address: BigInt(0x10000000), size }) }, 64 * MB);
let next = BigInt(0x90000000);
function tensor(records) {
  next += BigInt(16 * MB);
  return {
    sourceRecord: records.sourceRecord, runtimeRecord: records.runtimeRecord,
    binding: { buffer: { address: next, size: records.runtimeRecord.byteLength }, offset: 0,
               size: records.runtimeRecord.byteLength },
  };
}
function throwsLike(fn, type, message) {
  assert.throws(fn, (e) => e instanceof type && e.message.includes(message) || assert.fail(`${e.name}: ${e.message}`));
}
function check(kernel, make, cases) {
  kernel.validateDescriptor(make());
  for (const [change, type, message] of cases)
    throwsLike(() => kernel.validateDescriptor(Object.assign(make(), change)), type, message);
  kernel.destroy();
  throwsLike(() => kernel.createDispatch(make()), Error, "kernel was destroyed");
}

async function main() {
  const affine = host.channelTensorRecords(1000);
  const norm = () => ({
    label: "block", rows: 16, channels: 1000, kind: "rms", input: arena.slice("x", 0, 32000),
    gamma: tensor(affine), gate: arena.slice("gate", MB, 2000), gateRows: 0, residual: arena.slice("r", 2 * MB, 32000),
    residualScale: 0.5, output: arena.slice("y", 3 * MB, 32000),
    next: { gamma: tensor(affine), beta: tensor(affine), output: arena.slice("z", 4 * MB, 32000) },
  });
  check(await host.BlockNormKernel.create({}, arena), norm, [
    [{ kind: "batch" }, Error, "block has an unsupported norm kind batch"],
    [{ rows: -1 }, RangeError, "block rows must be a non-negative 32-bit integer"],
    [{ rows: 17 }, RangeError, "block input needs 34000 bytes; arena slice has 32000"],
    [{ gamma: tensor(host.channelTensorRecords(500)) }, Error, "block gamma must be float32 channel logical/storage [1000], 4000 bytes"],
    [{ gateRows: 4 }, RangeError, "block gate needs 8000 bytes; arena slice has 2000"],
    [{ output: arena.slice("y", 2048, 32000) }, Error, "block outputs must be the input or the residual"],
    [{ next: { gamma: tensor(affine) } }, Error, "block needs next gamma and next output together"],
    [{ epsilon: -1 }, Error, "block epsilon must be a finite number of at least 0"],
  ]);

  const records = host.q4TensorRecords({ inner: 640, columns: 1032, groupSize: 64 });
  assert.deepStrictEqual(records.scales.runtimeRecord.logicalShape, [10, 1032]);
  assert.strictEqual(records.packed.runtimeRecord.byteLength, 640 * 1032 / 2);
  const q4 = () => ({
    label: "head", rows: 4, inner: 640, columns: 1032, groupSize: 64, a: arena.slice("a", 0, 4 * 640 * 2),
    packed: tensor(records.packed), scales: tensor(records.scales), offsets: tensor(records.offsets),
    bias: tensor(host.channelTensorRecords(1032)), output: arena.slice("logits", MB, 4 * 1032 * 2), activation: "silu",
  });
  check(await host.Q4GemmKernel.create({}, arena), q4, [
    [{ activation: "tanh" }, Error, "head has an unsupported activation tanh"],
    [{ groupSize: 48 }, RangeError, "head group size must be a power of two from 32 on, or 0"],
    [{ groupSize: 32 }, Error, "head scales and offsets must be [20, 1032]"],
    [{ inner: 641 }, RangeError, "head a needs 5128 bytes; arena slice has 5120"],
    [{ packed: undefined }, Error, "head needs a, packed, scales and output"],
    [{ output: arena.slice("a", 256, 4 * 1032 * 2) }, Error, "head output must not overlap a"],
    [{ residualScale: 2 }, Error, "head has a residual scale without a residual"],
  ]);

  const score = () => ({
    label: "confidence", rows: 4, columns: 1025, rowStride: 1032, logits: arena.slice("logits", MB, 4 * 1032 * 2),
    tokens: arena.slice("tokens", 0, 16), logProbs: arena.slice("p", 256, 16), entropies: arena.slice("h", 512, 16),
    alternatives: 3, topTokens: arena.slice("top", 1024, 48), topLogProbs: arena.slice("topP", 2048, 48), temperature: 0.7,
  });
  check(await host.TokenScoreKernel.create({}, arena), score, [
    [{ alternatives: 33 }, RangeError, "confidence alternatives must be in [0, 32]"],
    [{ temperature: 0 }, RangeError, "confidence temperature must be in [2^-20, 2^20]"],
    [{ logProbs: undefined }, Error, "confidence needs tokens and log probs together"],
    [{ entropies: arena.slice("h", 256, 16) }, Error, "confidence outputs must not overlap"],
    [{ rows: 5 }, RangeError, "confidence logits needs 10306 bytes; arena slice has 8256"],
  ]);
  assert.strictEqual(host.SCORE_NO_TOKEN, 0xffffffff);
  console.log("host_cpu_operators ok");
}
main().catch((e) => { console.error(e); process.exit(1); });
