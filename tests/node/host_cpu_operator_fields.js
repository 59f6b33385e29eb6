// Fields of BlockNormKernel, Q4GemmKernel and TokenScoreKernel descriptors
// with values that are none of theirs: refused, by the host and by the addon
// under it, never left out. Run by tests/test_node_operator_fields.py.
"use strict";
const assert = require("assert");
const path = require("path");
const root = path.join(__dirname, "..", "..", "parakeet.wgsl_amd");
const host = require(path.join(root, "host"));
const addon = require(process.env.PK_NAPI_ADDON || path.join(root, "lib", "pk_napi.node"));

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
function refused(fn, type, message) {
  assert.throws(fn, (e) => (e instanceof type && e.message.includes(message)) || assert.fail(`${e.name}: ${e.message}`));
}
const STRIDES = [-1, 1000.5, 2 ** 32 + 1500, "1000", null, NaN];
const NUMBERS = ["0.5", "0", null, true, BigInt(1), {}];

async function main() {
  const affine = host.channelTensorRecords(1000), beside = { gamma: tensor(affine), output: arena.slice("z", 4 * MB, 64000) };
  const norm = () => ({
    label: "block", rows: 16, channels: 1000, input: arena.slice("x", 0, 64000), gate: arena.slice("g", MB, 64000),
    residual: arena.slice("r", 2 * MB, 64000), output: arena.slice("y", 3 * MB, 64000), next: beside,
  });
  const records = host.q4TensorRecords({ inner: 640, columns: 1032, groupSize: 64 });
  const q4 = () => ({
    label: "head", rows: 4, inner: 640, columns: 1032, groupSize: 64, a: arena.slice("a", 0, 16384),
    packed: tensor(records.packed), scales: tensor(records.scales), output: arena.slice("l", MB, 16384),
    residual: arena.slice("m", 2 * MB, 16384),
  });
  const score = () => ({
    label: "confidence", rows: 4, columns: 1025, logits: arena.slice("l", MB, 16384), entropies: arena.slice("h", 512, 16),
  });
  const kinds = [
    [await host.BlockNormKernel.create({}, arena), norm, "blockNorm",
     ["inputStride", "gateStride", "gateRows", "residualStride", "outputStride"], ["residualScale", "epsilon"]],
    [await host.Q4GemmKernel.create({}, arena), q4, "q4", ["aStride", "outputStride", "residualStride"], ["residualScale"]],
    [await host.TokenScoreKernel.create({}, arena), score, "score", ["rowStride", "alternatives"], ["temperature"]],
  ];
  for (const [kernel, make, prefix, sizes, numbers] of kinds) {
    const { label } = make();
    kernel.validateDescriptor(make());
    for (const [names, values, type, what] of [[sizes, STRIDES, RangeError, "a non-negative 32-bit integer"],
                                               [numbers, NUMBERS, Error, "a number"]])
      for (const name of names) {
        for (const value of values)
          refused(() => kernel.validateDescriptor(Object.assign(make(), { [name]: value })), type, `${label} ${name} must be ${what}`);
        // undefined is absent
        kernel.validateDescriptor(Object.assign(make(), { [name]: undefined }));
      }
    // the addon by itself: null and undefined are absent, anything else is the field's or an error
    const validate = addon[`${prefix}Validate`], plain = () => kernel.nativeDescriptor(make());
    validate(plain());
    for (const name of sizes)
      for (const value of STRIDES.concat([true, {}])) {
        const change = () => validate(Object.assign(plain(), { [name]: value }));
        if (value === null) change();
        else refused(change, Error, `${name} must be a non-negative 32-bit integer`);
      }
    for (const name of numbers)
      for (const value of NUMBERS) {
        const change = () => validate(Object.assign(plain(), { [name]: value }));
        if (value === null) change();
        else refused(change, Error, `${name} must be a number`);
      }
    for (const name of Object.keys(plain()).filter((n) => n.endsWith("Bytes"))) {
      const binding = name.slice(0, -5);
      refused(() => validate(Object.assign(plain(), { [binding]: "buffer" })), Error, `${binding} must be a device pointer`);
      refused(() => validate(Object.assign(plain(), { [name]: -4 })), Error, `${name} must be a byte count`);
      refused(() => validate(Object.assign(plain(), { [name]: undefined })), Error, `${name} must be a byte count`);
    }
  }

  // the stride of the next output is one of them
  const [kernel] = kinds[0];
  for (const outputStride of STRIDES)
    refused(() => kernel.validateDescriptor(Object.assign(norm(), { next: Object.assign({}, beside, { outputStride }) })),
            RangeError, "block nextOutputStride must be a non-negative 32-bit integer");
  refused(() => kernel.validateDescriptor(Object.assign(norm(), { next: Object.assign({}, beside, { outputStride: 999 }) })),
          RangeError, "block next output stride must be at least the channels");
  kernel.validateDescriptor(Object.assign(norm(), { next: Object.assign({}, beside, { outputStride: 1500 }) }));
  assert.strictEqual(kernel.nativeDescriptor(Object.assign(norm(), { next: Object.assign({}, beside, { outputStride: 1500 }) }))
                       .nextOutputStride, 1500);
  console.log("host_cpu_operator_fields ok");
}
main().catch((e) => { console.error(e); process.exit(1); });
